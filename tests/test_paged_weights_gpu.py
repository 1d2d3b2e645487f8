"""GPU tests of the accuracy of one-token attention's softmax weights: what a
16-bit product could lose of them, and what one strong key could hide."""
import math

import pytest
import torch

from fast_v2_b200 import _lib, paged
from tests import _paged_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _ops():
    _lib.ensure_ops()
    _lib.last_device_error()
    yield
    code, info = _lib.last_device_error()
    assert code == 0, f"device error {code} (info {info}) left by the test"


def _dense(q, k, v, lens, scale):
    """(out, bound) in 64 bits over K and V [B, n, hkv, D].  bound: half a step
    of the output; a weight goes into the product as two numbers of V's type,
    which leaves h^2 of it; D + 4 roundings of a score of magnitude sum |q k|
    move a weight by that much relative, in the numerator and in the sum; 200
    fp32 roundings of sums and joins.  fp16 alone: what is below 2^-14 is a
    multiple of 2^-24, next to a largest weight of 2^-5 in each 16 keys: 2^-20
    a key, 2^-16 of the largest value."""
    B, hq, D = q.shape
    h, u = R.half_step(q.dtype), R.U32
    out = torch.zeros(B, hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        kk, vv = (t[b, :n].double().repeat_interleave(hq // t.shape[2], 1).transpose(0, 1) for t in (k, v))
        qq = q[b].double()[:, None]
        p = torch.softmax((qq @ kk.transpose(1, 2))[:, 0] * scale, -1)
        out[b] = (p[:, None] @ vv)[:, 0]
        mass = (p[:, None] @ vv.abs())[:, 0]
        ds = (qq.abs() @ kk.abs().transpose(1, 2)).amax((1, 2)) * abs(scale) * (D + 4) * u
        bound[b] = h * out[b].abs() + (h * h + 2 * ds[:, None] + 200 * u) * mass * (1 + h)
        if q.dtype == HF:
            bound[b] += 2.0 ** -16 * vv.abs().amax((0, 1)) + 2.0 ** -24
    return out, bound


def _paged(k, v, page):
    """Dense K and V [B, n, hkv, D] as pages in reverse order and their table."""
    B, n, hkv, D = k.shape
    each = R.pages_of(n, page)
    pool = []
    for t in (k, v):
        full = torch.zeros(B, each * page, hkv, D, dtype=t.dtype, device=DEV)
        full[:, :n] = t
        pool.append(full.view(B * each, page, hkv, D).flip(0).contiguous())
    table = torch.arange(B * each - 1, -1, -1, device=DEV, dtype=torch.int32).view(B, each)
    return pool[0], pool[1], table


def _check(q, k, v, lens, scale, page=16):
    kp, vp, table = _paged(k, v, page)
    out = paged.decode_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), scale)
    ref, bound = _dense(q, k, v, lens, scale)
    R.assert_within("attention", out, ref, bound)


@pytest.mark.parametrize("hq,hkv,D", [(28, 4, 128), (64, 4, 128), (16, 16, 64), (6, 2, 256)])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("most", [40, 900, 9000])
def test_weights_are_not_cut_to_16_bits(most, dt, hq, hkv, D):
    """Values that nearly cancel show a weight's rounding; few keys do not
    average it out."""
    g = torch.Generator(device=DEV).manual_seed(most + D)
    lens = [2, 3, 5, 0, 17, 33, most]
    B = len(lens)
    k, v = (torch.randn(B, most, hkv, D, generator=g, device=DEV).to(dt) for _ in range(2))
    sign = torch.where(torch.arange(most, device=DEV) % 2 == 0, 1.0, -1.0)[None, :, None, None]
    v = (sign * (1 + v.abs().float() / 8)).to(dt)
    q = (2 * torch.randn(B, hq, D, generator=g, device=DEV)).to(dt)
    _check(q, k, v, lens, D ** -0.5)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("lead", [8.0, 11.0, 16.0, 17.4, 25.0])
@pytest.mark.parametrize("B,n,where", [(1, 131072, "first"), (1, 131072, "last"), (6, 40000, "middle"), (8, 3000, "first"),
                                       (2, 250, "last"), (200, 400, "first")])
def test_weak_keys_behind_a_strong_one_keep_their_share(B, n, where, lead, dt):
    """One key leads all others, which are equal, by `lead` nats: their share
    is (n - 1) / (n - 1 + e^lead) whatever their place, on the line and in the
    forms for short caches."""
    D, hq, hkv = 64, 4, 2
    at = {"first": 0, "middle": n // 2 + 5, "last": n - 1}[where]
    k = torch.zeros(B, n, hkv, D, dtype=dt, device=DEV)
    k[:, at, :, 0] = 8.0
    v = torch.zeros(B, n, hkv, D, dtype=dt, device=DEV)
    v[:] = torch.linspace(0.5, 8, D, device=DEV).to(dt)
    v[:, at] = 0
    q = torch.zeros(B, hq, D, dtype=dt, device=DEV)
    q[:, :, 0] = 1.0
    scale = lead / 8.0
    _check(q, k, v, [n] * B, scale)
    v[:, at] = -2.0
    _check(q, k, v, [n - 1 if where == "middle" else n] * B, scale)


@pytest.mark.parametrize("lead", [14.0, 17.0, 17.4, 22.0])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (24, 2)])
def test_many_weak_keys_of_one_warp_keep_their_share(hq, hkv, dt, lead):
    """With many sequences a warp walks tens of thousands of keys behind the
    strong one (the sequences share their pages)."""
    B, n, D = 150, 131072, 64
    k = torch.zeros(1, n, hkv, D, dtype=dt, device=DEV)
    k[:, 0, :, 0] = 8.0
    k[:, 60000, :, 0] = 4.0  # and another one on the way
    v = torch.zeros(1, n, hkv, D, dtype=dt, device=DEV)
    v[:] = torch.linspace(0.5, 8, D, device=DEV).to(dt)
    v[:, 0] = 0
    q = torch.zeros(B, hq, D, dtype=dt, device=DEV)
    q[:, :, 0] = 1.0
    q[:, 1::2, 0] = 0.0  # every second head weighs all keys alike
    kp, vp, table = _paged(k, v, 16)
    out = paged.decode_attention(q, kp, vp, table.repeat(B, 1), torch.full((B,), n, dtype=torch.int32, device=DEV),
                                 lead / 8.0)
    ref, bound = _dense(q[:1], k, v, [n], lead / 8.0)
    R.assert_within("attention", out, ref.expand(B, hq, D), bound.expand(B, hq, D))


def test_tiles_far_below_the_reference_with_infinite_scores_and_masked_pages():
    D = 64
    k = torch.zeros(1, 400, 1, D, dtype=HF, device=DEV)
    v = torch.ones(1, 400, 1, D, dtype=HF, device=DEV)
    k[0, 3, 0, 0] = 40.0
    k[0, 64:192, 0, 1] = -math.inf  # tiles without a finite score
    q = torch.zeros(1, 8, D, dtype=HF, device=DEV)
    q[:, :, 0] = 1.0
    q[:, :, 1] = 1.0
    kp, vp, table = _paged(k, v, 16)
    lens = torch.tensor([400], dtype=torch.int32, device=DEV)
    out = paged.decode_attention(q, kp, vp, table, lens, 1.0)
    assert bool((out == 1).all())
    table[0, 13] = -1  # and a tile without a page
    out = paged.decode_attention(q, kp, vp, table, lens, 1.0)
    assert _lib.last_device_error() == (1, -1)
    assert bool((out == 1).all())


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("gap", [9.3, 12.7, 20.1])
def test_a_reference_that_moves_at_every_tile_does_not_drift(gap, dt):
    """Every second run of 64 keys lies `gap` nats below the others: old and
    new keys keep their weights through thousands of moves."""
    B, n, D, hq, hkv = 150, 131072, 64, 4, 2
    k = torch.zeros(1, n, hkv, D, dtype=dt, device=DEV)
    low = (torch.arange(n, device=DEV) // 64) % 2 == 1
    k[:, low, :, 0] = -4.0
    k[:, 64000:64064, :, 0] = 1.0
    v = torch.ones(1, n, hkv, D, dtype=dt, device=DEV)
    v[:, : n // 2] = -1.0
    v[:, :, :, D // 2:] *= torch.where(low, 16.0, 1 / 16).to(dt)[None, :, None, None]
    q = torch.zeros(B, hq, D, dtype=dt, device=DEV)
    q[:, :, 0] = 1.0
    kp, vp, table = _paged(k, v, 16)
    out = paged.decode_attention(q, kp, vp, table.repeat(B, 1), torch.full((B,), n, dtype=torch.int32, device=DEV),
                                 gap / 4.0)
    ref, bound = _dense(q[:1], k, v, [n], gap / 4.0)
    ratio = ((out.double() - ref).abs() / bound).max()
    print(f"worst share of the bound {float(ratio):.3f}, worst error {float((out.double() - ref).abs().max()):.3g}")
    R.assert_within("attention", out, ref.expand(B, hq, D), bound.expand(B, hq, D))
