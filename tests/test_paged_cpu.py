"""CPU checks of the paged-cache operators and the token scores: the C ABI
refuses bad arguments before anything is launched, the plain implementations
that the GPU tests compare with agree with independent statements, and the
rotary frequencies follow their formulas."""
import ctypes
import math

import pytest
import torch

from fast_v2_b200 import _lib, paged, scoring
from tests import _paged_ref as R

OK, NULL, SHAPE, ALIGN, DTYPE, WORKSPACE, UNSUPPORTED = range(7)
i32, i64, f32, vp = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
P = 1 << 20  # an aligned address that is never read: every call here is refused or empty
BF16, F16, F32 = 0, 1, 2


def _fn(name, argtypes):
    f = getattr(_lib.abi(), name)
    f.argtypes, f.restype = argtypes, i32
    return f


def _call(name, types, base, change):
    args = dict(base)
    for k, v in change.items():
        assert k in args
        args[k] = v
    return _fn(name, types)(*args.values())


SLOTS = dict(lens=P, n_new=P, batch=2, table=P, table_sb=4, max_pages=4, free_pages=P, n_free=8, count=P, page=16,
             slots=P, positions=P, n_rows=4, cu=P, new_lens=P, new_count=P, stream=None)
SLOTS_T = [vp, vp, i32, vp, i64, i32, vp, i32, vp, i32, vp, vp, i64, vp, vp, vp, vp]


@pytest.mark.parametrize("change,rc", [
    (dict(batch=0), SHAPE), (dict(batch=4097), SHAPE), (dict(page=0), SHAPE), (dict(max_pages=-1), SHAPE),
    (dict(table_sb=3), SHAPE), (dict(n_free=-1), SHAPE), (dict(n_rows=-1), SHAPE), (dict(n_rows=1 << 31), SHAPE),
    (dict(max_pages=1 << 20, table_sb=1 << 20, page=1 << 12), SHAPE),
    (dict(max_pages=1, table_sb=1, page=1 << 30), SHAPE), (dict(lens=None), NULL),
    (dict(n_new=None), NULL), (dict(table=None), NULL), (dict(free_pages=None), NULL), (dict(count=None), NULL),
    (dict(slots=None), NULL), (dict(positions=None), NULL), (dict(cu=None), NULL), (dict(new_lens=None), NULL),
    (dict(new_count=None), NULL)])
def test_page_slots_refusals(change, rc):
    assert _call("fdl_page_slots", SLOTS_T, SLOTS, change) == rc


RELEASE = dict(done=P, lens=P, batch=2, table=P, table_sb=4, max_pages=4, free_pages=P, n_free=8, count=P, page=16,
               stream=None)
RELEASE_T = [vp, vp, i32, vp, i64, i32, vp, i32, vp, i32, vp]


@pytest.mark.parametrize("change,rc", [
    (dict(batch=0), SHAPE), (dict(batch=4097), SHAPE), (dict(page=0), SHAPE), (dict(table_sb=3), SHAPE),
    (dict(max_pages=1, table_sb=1, page=1 << 30), SHAPE), (dict(done=None), NULL), (dict(lens=None), NULL), (dict(table=None), NULL), (dict(free_pages=None), NULL),
    (dict(count=None), NULL)])
def test_page_release_refusals(change, rc):
    assert _call("fdl_page_release", RELEASE_T, RELEASE, change) == rc


ROPE = dict(y=P, y_rs=1536, pos=P, inv_freq=P, n_freq=64, qw=P, kw=P, eps=1e-6, inter=0, scale=1.0, q=P, k=P, v=2 * P,
            sp=4096, ss=256, sh=128, num_pages=8, page=16, slots=P, rows=4, hq=8, hkv=2, dim=128, dtype=BF16,
            stream=None)
ROPE_T = [vp, i64, vp, vp, i32, vp, vp, f32, i32, f32, vp, vp, vp, i64, i64, i64, i32, i32, vp, i64, i32, i32, i32,
          i32, vp]


@pytest.mark.parametrize("change,rc", [
    (dict(rows=0), OK), (dict(rows=0, y=None), OK), (dict(dtype=F32), DTYPE), (dict(dtype=7), DTYPE),
    (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(hq=0), SHAPE), (dict(hkv=0), SHAPE),
    (dict(dim=120), SHAPE), (dict(dim=8), SHAPE), (dict(dim=272), SHAPE), (dict(n_freq=65), SHAPE),
    (dict(n_freq=12), SHAPE), (dict(n_freq=72), SHAPE), (dict(n_freq=-8), SHAPE), (dict(num_pages=0), SHAPE),
    (dict(page=0), SHAPE), (dict(num_pages=1 << 20, page=1 << 12), SHAPE), (dict(y_rs=1528), SHAPE),
    (dict(hq=1 << 30, hkv=1 << 29, y_rs=1 << 60), SHAPE), (dict(v=P), SHAPE), (dict(sh=0), SHAPE), (dict(ss=0), SHAPE),
    (dict(sp=0), SHAPE), (dict(y=None), NULL), (dict(pos=None), NULL),
    (dict(inv_freq=None), NULL), (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL),
    (dict(slots=None), NULL), (dict(y=P + 2), ALIGN), (dict(q=P + 8), ALIGN), (dict(k=P + 2), ALIGN),
    (dict(v=P + 4), ALIGN), (dict(qw=P + 2), ALIGN), (dict(kw=P + 2), ALIGN), (dict(y_rs=1540), ALIGN),
    (dict(sp=4100), ALIGN), (dict(ss=257), ALIGN), (dict(sh=132), ALIGN)])
def test_norm_rope_store_refusals(change, rc):
    assert _call("fdl_norm_rope_store", ROPE_T, ROPE, change) == rc


ATTN = dict(q=P, q_sb=1024, q_sh=128, k=P, v=P, sp=4096, ss=256, sh=128, num_pages=8, page=16, table=P, table_sb=4,
            max_pages=4, lens=P, batch=2, hq=8, hkv=2, dim=128, dtype=BF16, scale=0.1, out=P, o_sb=1024, o_sh=128,
            ws=P, ws_bytes=1 << 40, stream=None)
ATTN_T = [vp, i64, i64, vp, vp, i64, i64, i64, i32, i32, vp, i64, i32, vp, i32, i32, i32, i32, i32, f32, vp, i64, i64,
          vp, i64, vp]


@pytest.mark.parametrize("change,rc", [
    (dict(batch=0), OK), (dict(dtype=F32), DTYPE), (dict(batch=-1), SHAPE), (dict(batch=65536), SHAPE),
    (dict(hq=0), SHAPE), (dict(hkv=0), SHAPE), (dict(hq=9), SHAPE), (dict(page=0), SHAPE), (dict(num_pages=-1), SHAPE),
    (dict(max_pages=-1), SHAPE), (dict(table_sb=3), SHAPE), (dict(num_pages=0), SHAPE), (dict(hq=8192), SHAPE),
    (dict(max_pages=1 << 20, table_sb=1 << 20, page=1 << 12), SHAPE), (dict(dim=96), UNSUPPORTED),
    (dict(dim=512), UNSUPPORTED), (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL),
    (dict(table=None), NULL), (dict(lens=None), NULL), (dict(out=None), NULL), (dict(q=P + 2), ALIGN),
    (dict(k=P + 8), ALIGN), (dict(v=P + 2), ALIGN), (dict(out=P + 2), ALIGN), (dict(q_sh=132), ALIGN),
    (dict(q_sb=1028), ALIGN), (dict(sp=4097), ALIGN), (dict(ss=260), ALIGN), (dict(sh=129), ALIGN),
    (dict(o_sb=1026), ALIGN), (dict(o_sh=130), ALIGN)])
def test_paged_attn_refusals(change, rc):
    assert _call("fdl_paged_attn", ATTN_T, ATTN, change) == rc


SCORE = dict(x=P, rs=1000, rows=2, vocab=1000, dtype=BF16, targets=P, lp=P, ent=P, top=5, top_lp=P, top_tok=P,
             stream=None)
SCORE_T = [vp, i64, i32, i32, i32, vp, vp, vp, i32, vp, vp, vp]


@pytest.mark.parametrize("change,rc", [
    (dict(rows=0), OK), (dict(rows=0, x=None), OK), (dict(dtype=3), DTYPE), (dict(rows=-1), SHAPE),
    (dict(vocab=0, rs=0), SHAPE), (dict(rs=-1), SHAPE), (dict(top=-1), SHAPE), (dict(top=33), SHAPE),
    (dict(vocab=4, top=5), SHAPE), (dict(x=None), NULL), (dict(targets=None), NULL), (dict(lp=None), NULL),
    (dict(ent=None), NULL), (dict(top_lp=None), NULL), (dict(top_tok=None), NULL), (dict(x=P + 1), ALIGN),
    (dict(dtype=F32, x=P + 2), ALIGN)])
def test_token_logprobs_refusals(change, rc):
    assert _call("fdl_token_logprobs", SCORE_T, SCORE, change) == rc


def test_wrappers_refuse_before_the_kernel():
    x = torch.zeros(2, 10)
    t = torch.zeros(2, dtype=torch.int64)
    for top in (-1, 11, 33):
        with pytest.raises(ValueError):
            scoring.token_logprobs(x, t, top)
    with pytest.raises(ValueError):
        scoring.token_logprobs(x[0], t)
    with pytest.raises((RuntimeError, NotImplementedError)):  # no CPU kernel
        scoring.token_logprobs(x, t)
    for kw in (dict(batch=0), dict(batch=5000), dict(page_size=0), dict(num_pages=0), dict(num_layers=0)):
        args = dict(num_layers=1, num_pages=4, page_size=4, batch=2, max_seq_len=8, num_kv_heads=1, head_dim=64,
                    dtype=torch.bfloat16, device="cpu") | kw
        with pytest.raises(ValueError):
            paged.PagedKVCache(**args)
    for args in ((7, 1e4), (0, 1e4)):
        with pytest.raises(ValueError):
            paged.rope_frequencies(*args)
    with pytest.raises(ValueError):
        paged.rope_frequencies(64, 1e4, factor=0.5)


def test_rope_frequencies():
    f, s = paged.rope_frequencies(64, 1e4)
    ref = torch.tensor([1e4 ** (-2 * j / 64) for j in range(32)], dtype=torch.float64).float()
    assert torch.equal(f, ref) and s == 1.0
    f4, s4 = paged.rope_frequencies(64, 1e4, factor=4.0)
    assert torch.equal(f4, (ref.double() / 4).float()) or (f4 - ref / 4).abs().max() <= ref.max() * 2 ** -24
    assert s4 == 1.0
    L = 4096
    fy, sy = paged.rope_frequencies(128, 1e6, factor=8.0, original_len=L)
    base, _ = paged.rope_frequencies(128, 1e6)
    turns = base.double() * L / (2 * math.pi)
    ratio = (fy / base).double()
    assert sy == pytest.approx(0.1 * math.log(8) + 1)
    assert bool((ratio[turns > 33] == 1).all())                        # fast pairs stay
    assert torch.allclose(ratio[turns < 0.9], torch.full((1,), 1 / 8, dtype=torch.float64), rtol=1e-6)
    assert bool((ratio[1:] <= ratio[:-1] + 1e-7).all())                # a ramp in between


def test_plain_slots_on_a_known_case():
    # page 4; sequence 0 has 3 tokens (page 9) and gets 3, sequence 1 is new and gets 5
    slots, pos, cu, table, lens, count, refused = R.slots_plain(
        [3, 0], [3, 5], [[9, -1, -1], [-1, -1, -1]], [0, 1, 2, 3, 4], 5, 4, 10)
    assert slots == [39, 16, 17, 12, 13, 14, 15, 8, -1, -1]
    assert pos == [3, 4, 5, 0, 1, 2, 3, 4, 0, 0]
    assert cu == [0, 3, 8] and table == [[9, 4, -1], [3, 2, -1]] and lens == [6, 5] and count == 2 and not refused
    # the pool runs out at sequence 1: it is refused whole, a sequence that needs no page goes on
    got = R.slots_plain([3, 0, 1], [3, 5, 2], [[9, -1], [-1, -1], [8, -1]], [0, 1], 2, 4, 10)
    assert got[0] == [39, 4, 5, -1, -1, -1, -1, -1, 33, 34] and got[6] == [1] and got[4] == [6, 0, 3] and got[5] == 1


def test_plain_attention_against_torch_sdpa():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(3, 6, 64, generator=g).to(torch.bfloat16)
    lens = [5, 0, 33]
    table, _, n = R.make_table(g, lens, 8, 5, 2, "cpu")
    k, v = (torch.randn(n, 8, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    out, bound = R.attn_plain(q, k, v, table, torch.tensor(lens), 0.2)
    assert bool((out[1] == 0).all())
    for b in (0, 2):
        at = table[b][: R.pages_of(lens[b], 8)].long()
        kk, vv = (t[at].reshape(-1, 2, 64)[: lens[b]].double().repeat_interleave(3, 1).transpose(0, 1) for t in (k, v))
        ref = torch.nn.functional.scaled_dot_product_attention(q[b].double()[:, None], kk, vv, scale=0.2)[:, 0]
        assert torch.allclose(out[b], ref, atol=1e-12)
