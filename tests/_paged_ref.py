"""Plain 64-bit implementations of the paged-cache operators and of the token
scores, with the error bounds that the tests hold the kernels to."""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def pages_of(n: int, page: int) -> int:
    return -(-n // page)


def slots_plain(lens, n_new, table, free, count, page, rows):
    """Request by request; refuses what the operator refuses.  Lists in, lists
    out: (slots, positions, cu, table, new_lens, count, refused)."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    slots, positions = [-1] * rows, [0] * rows
    cu, new_lens, refused = [0], [], []
    asked = 0    # pages asked for so far, refused ones of valid requests included
    taken = 0
    for b, (have, n) in enumerate(zip(lens, n_new)):
        m = max(n, 0)
        ok = have >= 0 and n >= 0 and have + n <= width * page
        need = pages_of(have + n, page) - pages_of(have, page) if ok else 0
        served = ok and (need == 0 or asked + need <= count) and cu[-1] + m <= rows
        if served:
            for j in range(need):
                table[b][pages_of(have, page) + j] = free[count - 1 - asked - j]
            if need:
                taken = asked + need
        else:
            refused.append(b)
        for i in range(m):
            t = cu[-1] + i
            if t < rows:
                p = have + i
                positions[t] = p
                if served and table[b][p // page] >= 0:
                    slots[t] = table[b][p // page] * page + p % page
        asked += need
        cu.append(cu[-1] + m)
        new_lens.append(have + n if served else have)
    return slots, positions, cu, table, new_lens, count - taken, refused


def rope_plain(x, pos, inv_freq, interleaved, scale, weight=None, eps=1e-6):
    """x [rows, heads, D] -> (out, slack) in 64 bits; slack bounds the fp32
    arithmetic: D/2 additions of the mean of squares (half of their relative
    error reaches the root), 16 operations more, on |a| + |b| of a pair."""
    x = x.double()
    D, rot = x.shape[-1], 2 * inv_freq.numel()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    ang = pos.double()[:, None, None] * inv_freq.double()
    c, s = ang.cos() * scale, ang.sin() * scale
    out, mag = x.clone(), x.abs()
    if rot:
        ia = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
        ib = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
        a, b = x[..., ia], x[..., ib]
        out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
        mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * scale
    return out, mag * (D / 2 + 16) * U32


def attn_plain(q, k_pages, v_pages, table, lens, scale):
    """(out, bound) in 64 bits.  bound: half a step of the output, half a step
    of each weight p (rounded to the type of V before the product), and the
    fp32 products: D + 2 roundings of a score of magnitude sum |q k| move p by
    that much relative, a sum over the keys by 2^-24 a key of a tile (64) and
    a few joins."""
    B, hq, D = q.shape
    page, hkv = k_pages.shape[1], k_pages.shape[2]
    out = torch.zeros(B, hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    h = half_step(q.dtype)
    for b, n in enumerate(lens.tolist()):
        at = table[b, : pages_of(n, page)].long()
        good = (at >= 0) & (at < k_pages.shape[0])
        see = good.repeat_interleave(page)[:n]
        if not bool(see.any()):
            continue
        at = at.clamp(0, k_pages.shape[0] - 1)
        k = k_pages[at].reshape(-1, hkv, D)[:n][see].double()
        v = v_pages[at].reshape(-1, hkv, D)[:n][see].double()
        k, v = (t.repeat_interleave(hq // hkv, 1).transpose(0, 1) for t in (k, v))
        qq = q[b].double()[:, None]
        s = (qq @ k.transpose(1, 2))[:, 0] * scale
        p = torch.softmax(s, -1)
        out[b] = (p[:, None] @ v)[:, 0]
        mass = (p[:, None] @ v.abs())[:, 0]
        ds = (qq.abs() @ k.abs().transpose(1, 2)).amax((1, 2)) * abs(scale) * (D + 4) * U32
        bound[b] = h * out[b].abs() + (h + 2 * ds[:, None] + 200 * U32) * mass * (1 + h)
    # fp16 has no normal numbers below 2^-14: half a step there is 2^-25
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    return out, bound + 2 * tiny


def scores_plain(x, targets, top):
    """(logprob, entropy, top_logprob, top_token, bound of lse, bound of entropy)."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    p = e / z
    d = torch.where(p > 0, x - m, 0.0)
    entropy = (z.log() - (p * d).sum(-1, keepdim=True))[:, 0]
    lp = torch.where(targets >= 0, (x.gather(1, targets.clamp_min(0)[:, None]) - lse)[:, 0], 0.0)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    top_lp = x.gather(1, order) - lse
    # sums of V / 512 terms a thread and 40 joins; an exponential is off by two
    # steps and by |x - m| steps of its argument, which weighs in with p |x - m|
    n = x.shape[-1] / 512 + 44
    spread = (p * d.abs()).sum(-1)
    rel = (n + 4 * spread) * U32
    b_lse = rel + 4 * U32 * (lse[:, 0].abs() + m[:, 0].abs())
    far = (p * d * d).sum(-1)
    b_ent = rel * (1 + spread) + 4 * U32 * (1 + spread + far + entropy.abs())
    return lp, entropy, top_lp, order, b_lse, b_ent


def make_table(g, lens, page, width, spare, device):
    """Distinct pages in random order for sequences of these lengths; -1
    behind them.  (table, free pages, number of pages)."""
    need = [pages_of(n, page) for n in lens]
    perm = torch.randperm(sum(need) + spare, generator=g).tolist()
    table = [[-1] * width for _ in lens]
    for b, n in enumerate(need):
        for i in range(n):
            table[b][i] = perm.pop()
    t = torch.tensor(table, dtype=torch.int32).reshape(len(lens), width)
    return t.to(device), torch.tensor(perm, dtype=torch.int32, device=device), sum(need) + spare


def assert_within(name, got, ref, bound):
    kind, got, ref = got.dtype, got.double(), ref.double()
    # what lies past the type's largest number (fp32: 2^128 (1 - 2^-24) = 3.4e38) by half a step rounds to infinity
    top = torch.finfo(kind).max
    ref = torch.where(ref.abs() > top * (1 + half_step(kind)), ref.sign() * math.inf, ref)
    same = (got == ref) | (got.isnan() & ref.isnan())
    bad = ~same & ~((got - ref).abs() <= bound)
    if bool(bad.any()):
        i = int(bad.flatten().nonzero()[0])
        worst = float(((got - ref).abs() / bound.clamp_min(1e-300)).flatten()[bad.flatten()].max())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound, worst {worst:.3g} times; "
                             f"first at {i}: {float(got.flatten()[i])!r} for {float(ref.flatten()[i])!r} "
                             f"(bound {float(bound.expand_as(got).flatten()[i]):.3g})")
