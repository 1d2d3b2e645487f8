"""Measured cases of the paged-serving operators and of the token scores.

Four operators that a serving step runs one after another:

  slots   block tables and slot maps built on the GPU from request lengths and
          a list of free pages;
  rope    the split of a q/k/v projection's rows, an optional RMS norm of each
          query and key head, the rotary positions (half or interleaved, whole
          head or part of it, positions of long contexts), K and V stored into
          their pages;
  attn    attention of one new token per sequence over the paged cache;
  score   log probability of given tokens, entropy of the distribution and its
          best alternatives, from a row of logits.

``own`` False computes them in elementary torch operations, True calls the
framework.  Sizes are those of the 7B (28/4 heads of 128, vocabulary 152064)
and 1.5B (12/2 heads) geometries of this framework, and generic ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def listed():
    return [
        # One decode step of a batch of 64: every request gets one token, some
        # of them a new page.  The call is all latency.
        {"name": "slots decode 64", "op": "slots", "batch": 64, "new": 1, "max_len": 8192, "page": 16, "pad": 0},
        # Chunked prefill next to decoding: 256 requests with 0 to 500 new
        # tokens each, in a buffer padded for a captured graph.
        {"name": "slots prefill 256", "op": "slots", "batch": 256, "new": 500, "max_len": 4096, "page": 32,
         "pad": 1000},
        # One decode step of 16 requests, 7B heads, head norms.
        {"name": "rope decode 16", "op": "rope", "rows": 16, "hq": 28, "hkv": 4, "dim": 128, "rot": 128,
         "interleaved": False, "norm": True, "page": 16, "far": 32768, "type": "bf16"},
        # One block step: 64 sequences of 32 tokens, 7B heads.
        {"name": "rope block 2048", "op": "rope", "rows": 2048, "hq": 28, "hkv": 4, "dim": 128, "rot": 128,
         "interleaved": False, "norm": True, "page": 32, "far": 8192, "type": "bf16"},
        # A long prefill chunk, interleaved pairs in half of each head, far
        # positions, no head norm.
        {"name": "rope prefill 16001", "op": "rope", "rows": 16001, "hq": 12, "hkv": 2, "dim": 128, "rot": 64,
         "interleaved": True, "norm": False, "page": 64, "far": 1000000, "type": "fp16"},
        # One request with a short prompt: latency.
        {"name": "attn one short", "op": "attn", "batch": 1, "hq": 28, "hkv": 4, "dim": 128, "page": 16,
         "min_len": 200, "max_len": 400, "type": "bf16"},
        # One request with a long context: the work has to be split.
        {"name": "attn one long", "op": "attn", "batch": 1, "hq": 28, "hkv": 4, "dim": 128, "page": 64,
         "min_len": 65000, "max_len": 66000, "type": "bf16"},
        # A ragged batch of 64 up to the 8192 tokens of the block attention
        # benchmark, with empty rows as in a padded batch.
        {"name": "attn batch 64", "op": "attn", "batch": 64, "hq": 28, "hkv": 4, "dim": 128, "page": 32,
         "min_len": 1, "max_len": 8192, "type": "bf16"},
        # Many short requests, 1.5B heads, fp16.
        {"name": "attn many short", "op": "attn", "batch": 200, "hq": 12, "hkv": 2, "dim": 128, "page": 16,
         "min_len": 1, "max_len": 1000, "type": "fp16"},
        # The logits of a few decoded tokens with 20 alternatives each.
        {"name": "score 8", "op": "score", "rows": 8, "vocab": 152064, "top": 20, "type": "bf16"},
        # The sampler's rows: 64 sequences, sub-blocks of 8 tokens.
        {"name": "score 512", "op": "score", "rows": 512, "vocab": 152064, "top": 20, "type": "bf16"},
        # The tokens of an evaluation's answers, odd vocabulary, fp32 logits
        # (rows that start off a 16-byte boundary).
        {"name": "score 1500 odd", "op": "score", "rows": 1500, "vocab": 50257, "top": 5, "type": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


HEADS = [(28, 4, 128), (12, 2, 128), (32, 8, 128), (16, 16, 64), (8, 1, 128), (14, 2, 64), (20, 1, 64), (64, 4, 128),
         (16, 2, 256), (6, 6, 128)]
MOST_TOKENS = 60000         # slots: batch * new
MOST_ROPE_BYTES = 120e6     # rope: rows * (hq + 2 hkv) * dim * 2 * 2
MOST_KV_BYTES = 500e6       # attn: batch * (longest) * hkv * dim * 2 * 2
MOST_LOGIT_BYTES = 140e6    # score: rows * vocab * element


def draw(rng: random.Random):
    op = rng.choice(["slots", "rope", "attn", "attn", "score"])
    page = rng.choice([8, 16, 16, 32, 64, 128, 20])
    if op == "slots":
        batch = _log_int(rng, 1, 1000)
        new = 1 if rng.random() < 0.3 else _log_int(rng, 2, max(2, min(4000, MOST_TOKENS // batch)))
        return {"op": op, "batch": batch, "new": new, "max_len": _log_int(rng, 1, 20000), "page": page,
                "pad": rng.choice([0, 0, 1, 300])}
    hq, hkv, dim = rng.choice(HEADS)
    if op == "rope":
        most = int(MOST_ROPE_BYTES / ((hq + 2 * hkv) * dim * 4))
        return {"op": op, "rows": _log_int(rng, 1, most), "hq": hq, "hkv": hkv, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.5,
                "norm": rng.random() < 0.5, "page": page, "far": rng.choice([4096, 131072, 1000000]),
                "type": rng.choice(["bf16", "fp16"])}
    if op == "attn":
        batch = _log_int(rng, 1, 256)
        most = int(MOST_KV_BYTES / (batch * hkv * dim * 4))
        hi = _log_int(rng, 1, min(131072, most))
        lo = rng.choice([1, max(1, hi // 2), hi])
        return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "min_len": lo,
                "max_len": hi, "type": rng.choice(["bf16", "bf16", "fp16"])}
    kind = rng.choice(["bf16", "fp16", "fp32"])
    vocab = _log_int(rng, 1000, 160000)
    most = int(MOST_LOGIT_BYTES / (vocab * (4 if kind == "fp32" else 2)))
    return {"op": op, "rows": _log_int(rng, 1, max(1, most)), "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]),
            "type": kind}


def _pages(count, page):
    return (count + page - 1) // page


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"slots": _prepare_slots, "rope": _prepare_rope, "attn": _prepare_attn, "score": _prepare_score}[
        case["op"]](case, g)


def _ints(g, lo, hi, shape, dtype=torch.int32):
    """Uniform integers in [lo, hi]."""
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV).to(dtype)


def _table(g, lens, page, width, spare):
    """A block table of distinct pages in random order, -1 behind them, and the pages left over."""
    used = torch.arange(width, device=DEV)[None, :] < _pages(lens.long(), page)[:, None]
    n = int(used.sum())
    perm = torch.randperm(n + spare, generator=g, device=DEV).int()
    table = torch.full(used.shape, -1, dtype=torch.int32, device=DEV)
    table[used] = perm[:n]
    return table, perm[n:].contiguous(), n + spare


def _tokens(c, i):
    return 1 if c["new"] == 1 else c["new"] * (i if c["batch"] > 1 else 1) // max(1, c["batch"] - 1)


def _prepare_slots(c, g):
    B, page = c["batch"], c["page"]
    lens = _ints(g, 0, c["max_len"], (B,))
    # one new token each in a decode step; otherwise from none to all of them, dealt out by the seed
    ramp = [_tokens(c, i) for i in range(B)]
    n_new = torch.tensor(ramp, dtype=torch.int32, device=DEV)[torch.randperm(B, generator=g, device=DEV)]
    width = _pages(c["max_len"] + c["new"], page)
    need = int((_pages(lens.long() + n_new, page) - _pages(lens.long(), page)).sum())
    table, free, _ = _table(g, lens, page, width, need + 7)
    total = sum(ramp) + c["pad"]
    i64 = lambda n: torch.empty(n, dtype=torch.int64, device=DEV)  # noqa: E731
    return {"case": c, "lens": lens, "n_new": n_new, "table": table, "free": free,
            "count": torch.tensor([free.numel(), 0], dtype=torch.int32, device=DEV),
            "slots": i64(total), "positions": i64(total),
            "cu": torch.empty(B + 1, dtype=torch.int32, device=DEV),
            "new_lens": torch.empty_like(lens), "new_count": torch.zeros(2, dtype=torch.int32, device=DEV)}


def _prepare_rope(c, g):
    rows, hq, hkv, D, page, dt = c["rows"], c["hq"], c["hkv"], c["dim"], c["page"], TYPES[c["type"]]
    pages = _pages(rows, page) + 3
    y = torch.randn(rows, (hq + 2 * hkv) * D, generator=g, device=DEV).to(dt)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:rows].contiguous()
    slots[rows - rows // 16:] = -1  # the padding rows of a captured graph store nothing
    base = 1e6
    inv_freq = base ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"])
    weight = lambda: (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dt)  # noqa: E731
    return {"case": c, "y": y, "slots": slots, "positions": _ints(g, 0, c["far"], (rows,), torch.int64),
            "inv_freq": inv_freq.float(), "qw": weight() if c["norm"] else None, "kw": weight() if c["norm"] else None,
            "k": torch.zeros(pages, page, hkv, D, dtype=dt, device=DEV),
            "v": torch.zeros(pages, page, hkv, D, dtype=dt, device=DEV),
            # the factor that long-context scaling puts on cos and sin
            "factor": 1.0 if c["far"] <= 131072 else 1.25,
            "q": torch.empty(rows, hq, D, dtype=dt, device=DEV)}


def _prepare_attn(c, g):
    B, hq, hkv, D, page, dt = c["batch"], c["hq"], c["hkv"], c["dim"], c["page"], TYPES[c["type"]]
    lens = _ints(g, c["min_len"], c["max_len"], (B,))
    lens[15::16] = 0  # rows of a padded batch
    table, _, pages = _table(g, lens, page, _pages(c["max_len"], page), 2)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.bfloat16).to(dt)  # noqa: E731
    return {"case": c, "lens": lens, "table": table, "q": (2 * torch.randn(B, hq, D, generator=g, device=DEV)).to(dt),
            "k": rnd(pages, page, hkv, D), "v": rnd(pages, page, hkv, D),
            "out": torch.empty(B, hq, D, dtype=dt, device=DEV)}


def _prepare_score(c, g):
    rows, V = c["rows"], c["vocab"]
    x = torch.randn(rows, V, generator=g, device=DEV).mul_(2.5)
    at = _ints(g, 0, V - 1, (rows,), torch.int64)
    x.scatter_add_(1, at[:, None], 15 * torch.rand(rows, 1, generator=g, device=DEV))  # how sure the model is
    x[:, torch.randperm(V, generator=g, device=DEV)[: V // 200]] = -math.inf            # tokens that may not come
    x[torch.arange(rows, device=DEV), at] = x[torch.arange(rows, device=DEV), at].clamp_min(-20.0)
    x = x.to(TYPES[c["type"]])
    targets = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.5, at, _ints(g, 0, V - 1, (rows,), torch.int64))
    targets[x[torch.arange(rows, device=DEV), targets] == -math.inf] = -1  # no target in this row
    return {"case": c, "x": x, "targets": targets}


def run(s):
    return {"slots": _run_slots, "rope": _run_rope, "attn": _run_attn, "score": _run_score}[s["case"]["op"]](s)


def _run_slots(s):
    page = s["case"]["page"]
    if own:
        from fast_v2_b200 import paged

        paged.build_slots(s["lens"], s["n_new"], s["table"], s["free"], s["count"], page, s["slots"], s["positions"],
                          s["cu"], s["new_lens"], s["new_count"])
        return [s["slots"], s["positions"], s["cu"], s["table"], s["new_lens"], s["new_count"][:1]]
    lens, n_new, free = s["lens"].long(), s["n_new"].long(), s["free"].long()
    total = s["slots"].numel()
    new_lens = lens + n_new
    old, now = _pages(lens, page), _pages(new_lens, page)
    cu = torch.cat([n_new.new_zeros(1), n_new.cumsum(0)])
    at = torch.cat([n_new.new_zeros(1), (now - old).cumsum(0)])
    # new pages come off the end of the free list, in the order of the requests
    col = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    take = s["count"][0].long() - 1 - (at[:-1, None] + col - old[:, None])
    fresh = (col >= old[:, None]) & (col < now[:, None])
    table = torch.where(fresh, free[take.clamp(0, free.numel() - 1)], s["table"].long())
    t = torch.arange(total, device=DEV)
    b = torch.searchsorted(cu[1:], t, right=True).clamp_max(lens.numel() - 1)
    real = t < cu[-1]
    pos = lens[b] + t - cu[b]
    slots = table[b, (pos // page).clamp_max(table.shape[1] - 1)] * page + pos % page
    return [torch.where(real, slots, -1), torch.where(real, pos, 0), cu.int(), table.int(), new_lens.int(),
            s["count"][:1] - at[-1:].int()]


def _run_rope(s):
    c = s["case"]
    hq, hkv, D, rot = c["hq"], c["hkv"], c["dim"], c["rot"]
    if own:
        from fast_v2_b200 import paged

        paged.norm_rope_store(s["y"], s["positions"], s["inv_freq"], s["q"], s["k"], s["v"], s["slots"],
                              q_weight=s["qw"], k_weight=s["kw"], eps=1e-6, interleaved=c["interleaved"],
                              rope_scale=s["factor"])
        return [s["q"], s["k"], s["v"]]
    y = s["y"].float().view(-1, hq + 2 * hkv, D)
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float() * s["factor"], angle.sin().float() * s["factor"]

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        r = x[..., :rot]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = r[..., : rot // 2], r[..., rot // 2:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, x[..., rot:]], -1).to(s["y"].dtype)

    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["k"].view(-1, hkv, D)[at] = turned(y[:, hq:hq + hkv], s["kw"])[keep]
    s["v"].view(-1, hkv, D)[at] = y[:, hq + hkv:].to(s["y"].dtype)[keep]
    return [turned(y[:, :hq], s["qw"]), s["k"], s["v"]]


def _run_attn(s):
    c = s["case"]
    B, hq, hkv, D, page = c["batch"], c["hq"], c["hkv"], c["dim"], c["page"]
    scale = D ** -0.5
    if own:
        from fast_v2_b200 import paged

        return paged.decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], scale, out=s["out"])
    at = s["table"].long().clamp_min(0)
    n = at.shape[1] * page
    seen = (torch.arange(n, device=DEV)[None, :] < s["lens"][:, None])[:, None, None, :]
    k = s["k"][at].view(B, n, hkv, D).float()
    scores = torch.einsum("bhgd,bnhd->bhgn", s["q"].float().view(B, hkv, hq // hkv, D), k) * scale
    del k
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)  # a row that sees no key comes out as zeros
    v = s["v"][at].view(B, n, hkv, D).float()
    return torch.einsum("bhgn,bnhd->bhgd", p, v).reshape(B, hq, D).to(s["q"].dtype)


def _run_score(s):
    top = s["case"]["top"]
    if own:
        from fast_v2_b200 import scoring

        r = scoring.token_logprobs(s["x"], s["targets"], top)
        return [r.logprob, r.entropy] + ([r.top_logprob, r.top_token] if top else [])
    x = s["x"].float()
    V = x.shape[1]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    logprob = x.gather(1, s["targets"].clamp_min(0)[:, None]) - lse
    logprob = torch.where(s["targets"] >= 0, logprob[:, 0], 0.0)
    entropy = z.log()[:, 0] - (e * (x - m).clamp_min(torch.finfo(torch.float32).min)).sum(-1) / z[:, 0]
    if not top:
        return [logprob, entropy]
    # whole numbers in the order of the values, the lower index first among equals
    bits = x.view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 20) + (V - 1 - torch.arange(V, device=DEV))
    token = (V - 1) - (key.topk(top, -1).values & ((1 << 20) - 1))
    return [logprob, entropy, x.gather(1, token) - lse, token]


def work(case):
    c = case
    if c["op"] == "slots":
        tokens = sum(_tokens(c, i) for i in range(c["batch"])) + c["pad"]
        pages = c["batch"] + tokens / c["page"]
        # lengths, counts and last pages in, lengths and offsets out; free pages in, table entries out; slot and position
        return {"bytes": c["batch"] * 20 + pages * 8 + tokens * 16, "flops": 0}
    if c["op"] == "rope":
        n = c["rows"] * (c["hq"] + 2 * c["hkv"]) * c["dim"]
        return {"bytes": n * 4 + c["rows"] * 16, "flops": 10 * n}
    if c["op"] == "attn":
        keys = c["batch"] * (c["min_len"] + c["max_len"]) / 2 * (1 - c["batch"] // 16 / c["batch"])
        return {"bytes": keys * c["hkv"] * c["dim"] * 4 + c["batch"] * c["hq"] * c["dim"] * 4 + keys / c["page"] * 4,
                "flops": 4 * keys * c["hq"] * c["dim"]}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * (4 if c["type"] == "fp32" else 2) + c["rows"] * (16 + 12 * c["top"]), "flops": 5 * n}


def exact(case, seed):
    s = prepare(case, seed)
    return {"slots": _exact_slots, "rope": _exact_rope, "attn": _exact_attn, "score": _exact_score}[case["op"]](case, s)


def _exact_slots(c, s):
    """Request by request on the host, as a scheduler would."""
    page = c["page"]
    lens, n_new, free, table = s["lens"].tolist(), s["n_new"].tolist(), s["free"].tolist(), s["table"].tolist()
    slots, positions, cu, new_lens = [], [], [0], []
    for b, (have, n) in enumerate(zip(lens, n_new)):
        for p in range(have, have + n):
            if p == -(-have // page) * page or (p % page == 0 and p > have):
                table[b][p // page] = free.pop()
            slots.append(table[b][p // page] * page + p % page)
            positions.append(p)
        cu.append(cu[-1] + n)
        new_lens.append(have + n)
    slots += [-1] * c["pad"]
    positions += [0] * c["pad"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return [torch.tensor(slots), torch.tensor(positions), i32(cu), i32(table), i32(new_lens), i32([len(free)])]


def _exact_rope(c, s):
    """Each pair of a head as a complex number, turned by exp(i angle)."""
    hq, hkv, D, rot, rows = c["hq"], c["hkv"], c["dim"], c["rot"], c["rows"]
    y = s["y"].double().reshape(rows, hq + 2 * hkv, D)
    turn = torch.polar(torch.full((rows, 1, rot // 2), s["factor"], dtype=torch.float64, device=DEV),
                       s["positions"].double().view(-1, 1, 1) * s["inv_freq"].double().view(1, 1, -1))

    def head(x, w):
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
        out = x.clone()
        if c["interleaved"]:
            z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
            out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., : rot // 2], x[..., rot // 2: rot]) * turn
            out[..., : rot // 2], out[..., rot // 2: rot] = z.real, z.imag
        return out

    k, v = s["k"].double().view(-1, hkv, D), s["v"].double().view(-1, hkv, D)
    n = int((s["slots"] >= 0).sum())  # the rows behind them are padding
    k[s["slots"][:n]] = head(y[:, hq:hq + hkv], s["kw"])[:n]
    v[s["slots"][:n]] = y[:n, hq + hkv:]
    return [head(y[:, :hq], s["qw"]), k.view(s["k"].shape), v.view(s["v"].shape)]


def _exact_attn(c, s):
    """Sequence by sequence, in 64 bits."""
    hq, hkv, D, page = c["hq"], c["hkv"], c["dim"], c["page"]
    out = torch.zeros(c["batch"], hkv, hq // hkv, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        if n:
            at = s["table"][b, : _pages(n, page)].long()
            k, v = (s[x][at].reshape(-1, hkv, D)[:n].transpose(0, 1).double() for x in "kv")
            q = s["q"][b].double().view(hkv, hq // hkv, D)
            out[b] = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(D), -1) @ v
    return out.view(c["batch"], hq, D)


def _exact_score(c, s):
    top, got = c["top"], []
    for x, t in zip(s["x"].split(128), s["targets"].split(128)):
        logp = torch.log_softmax(x.double(), -1)
        p = logp.exp()
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
        target = torch.where(t >= 0, logp.gather(1, t.clamp_min(0)[:, None])[:, 0], 0.0)
        order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
        got.append([target, entropy] + ([logp.gather(1, order), order] if top else []))
    return [torch.cat(v) for v in zip(*got)]
