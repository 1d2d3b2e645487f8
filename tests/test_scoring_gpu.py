"""GPU tests of the token scores against a plain 64-bit implementation."""
import math

import pytest
import torch

from fast_v2_b200 import _lib, scoring
from tests import _paged_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _ops():
    _lib.ensure_ops()
    _lib.last_device_error()
    yield
    code, info = _lib.last_device_error()
    assert code == 0, f"device error {code} (info {info}) left by the test"


def _check(x, targets, top):
    got = scoring.token_logprobs(x, targets, top)
    lp, ent, tlp, tok, bl, be = R.scores_plain(x, targets, top)
    R.assert_within("logprob", got.logprob, lp, bl + lp.abs() * R.U32)
    R.assert_within("entropy", got.entropy, ent, be)
    if top:
        assert torch.equal(got.top_token, tok)
        R.assert_within("top", got.top_logprob, tlp, bl[:, None] + tlp.abs() * R.U32)
    else:
        assert got.top_logprob is None and got.top_token is None
    return got


def _logits(seed, rows, V, dt, scale=2.5, pad=0, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    base = torch.full((rows * (V + pad) + offset + 8,), float("nan"), dtype=dt, device=DEV)
    x = base[offset: offset + rows * (V + pad)].view(rows, V + pad)[:, :V]
    x.copy_(torch.randn(rows, V, generator=g, device=DEV) * scale)
    t = torch.randint(0, V, (rows,), generator=g, device=DEV)
    return x, t


@pytest.mark.parametrize("dt", [BF, HF, F])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 0), (1, 1, 1), (3, 2, 2), (5, 7, 5), (2, 8, 8), (4, 33, 32), (9, 100, 32),
                                        (2, 511, 20), (3, 4097, 32), (1, 152064, 20), (8, 151936, 20),
                                        (64, 50257, 5), (150, 8193, 1), (400, 32000, 0), (700, 1001, 20)])
def test_scores(rows, V, top, dt):
    x, t = _logits(rows + V, rows, V, dt)
    t[::5] = -1
    _check(x, t, top)


@pytest.mark.parametrize("dt", [BF, F])
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (3, 5), (8, 0), (7, 3)])
@pytest.mark.parametrize("rows,V", [(3, 1000), (40, 6001), (2, 5)])
def test_scores_of_rows_off_the_alignment(rows, V, pad, offset, dt):
    x, t = _logits(1, rows, V, dt, pad=pad, offset=offset)
    _check(x, t, min(V, 20))


@pytest.mark.parametrize("rows", [1, 30, 400])
@pytest.mark.parametrize("V", [300, 20011, 152064])
def test_scores_of_tied_rows(rows, V):
    if rows * V > 2e7:
        rows = 130
    x = torch.zeros(rows, V, dtype=BF, device=DEV)
    t = torch.zeros(rows, dtype=torch.int64, device=DEV)
    _check(x, t, 32)                                    # all equal: the lowest indices
    x[:, V - 40:] = 1.0
    _check(x, t, 20)                                    # equal at the end
    x.fill_(-math.inf)
    x[:, 7::97] = 2.0
    t.fill_(7)
    _check(x, t, 2)
    x.fill_(-math.inf)
    x[:, [3, 200, V - 1]] = torch.tensor([1.0, 3.0, 3.0], device=DEV).to(BF)
    t.fill_(3)
    got = _check(x, t, 32)                              # fewer possible tokens than asked for
    assert got.top_token[0, :4].tolist() == [200, V - 1, 3, 0] and got.top_logprob[0, 3] == -math.inf
    x[:, 1] = -0.0
    x[:, 0] = 0.0
    _check(x, t, 5)                                     # -0 and 0 are equal


@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("dt", [BF, F])
def test_scores_of_rows_with_their_best_in_few_places(rows, dt):
    """The largest logits crowd in one stretch, in one residue class, or rise
    or fall along the row."""
    V = 40000
    x, t = _logits(3, rows, V, dt, scale=1.0)
    y = x.clone()
    y[:, 8000:9000] += 20
    _check(y, t, 32)
    for step in (8, 4096, 16384):
        y = x.clone()
        y[:, 5::step] += 20
        _check(y, t, 32)
        y = x.clone()
        for o in range(8):
            y[:, o::step] += 20
        _check(y, t, 32)
    ramp = torch.linspace(0, 50, V, device=DEV).to(dt)
    _check(ramp.expand(rows, V).contiguous(), t, 32)
    _check(ramp.flip(0).expand(rows, V).contiguous(), t, 32)


def test_scores_of_sure_and_unsure_rows():
    x, t = _logits(4, 4, 30000, F, scale=0.01)
    x[1, 77] = 200.0
    x[2] *= 3000
    x[3] = x[3] - 1e4
    t[1] = 77
    _check(x, t, 20)
    big = torch.full((2, 5000), -3e38, dtype=F, device=DEV)
    big[0, 9] = 3e38
    _check(big, torch.tensor([9, 1], device=DEV), 3)


def test_rows_that_are_no_distribution():
    x, t = _logits(5, 6, 3001, F)
    x[1, 3000] = float("nan")
    x[2, 17] = float("inf")
    x[3] = -math.inf
    x[4, :] = float("nan")
    got = scoring.token_logprobs(x, t, 4)
    code, info = _lib.last_device_error()
    assert code == 1 and info in (1, 2, 3, 4)
    for r in (1, 2, 3, 4):
        assert bool(got.logprob[r].isnan()) and bool(got.entropy[r].isnan())
        assert got.top_token[r].tolist() == [-1] * 4 and bool(got.top_logprob[r].isnan().all())
    keep = torch.tensor([0, 5], device=DEV)
    good = scoring.token_logprobs(x[keep], t[keep], 4)
    assert torch.equal(got.top_token[keep], good.top_token)
    lp, _, _, tok, bl, _ = R.scores_plain(x[keep], t[keep], 4)
    R.assert_within("logprob", got.logprob[keep], lp, bl + lp.abs() * R.U32)
    assert torch.equal(good.top_token, tok)


def test_targets_past_the_vocabulary_are_reported():
    x, t = _logits(6, 3, 100, BF)
    t[1] = 100
    got = scoring.token_logprobs(x, t, 1)
    assert _lib.last_device_error() == (1, 100)
    assert bool(got.logprob[1].isnan()) and bool(got.logprob[[0, 2]].isfinite().all())


def test_scores_on_streams_and_in_a_graph():
    x, t = _logits(7, 200, 9001, BF)
    want = scoring.token_logprobs(x, t, 20)
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(10):
        with torch.cuda.stream(s[i % 2]):
            got.append(scoring.token_logprobs(x, t, 20))
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)  # the same bits on every run
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = scoring.token_logprobs(x, t, 20)
    x.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(r.top_token, scoring.token_logprobs(x, t, 20).top_token)


def test_refusals_and_empty_rows():
    x, t = _logits(8, 4, 64, BF)
    for args in ((x, t.int()), (x, t[:3]), (x, t.cpu()), (x.t(), t), (x.double(), t)):
        with pytest.raises(RuntimeError):
            scoring.token_logprobs(*args)
    r = scoring.token_logprobs(x[:0], t[:0], 3)
    assert r.logprob.shape == (0,) and r.top_token.shape == (0, 3)


def test_one_row_expanded_for_several_targets():
    x, _ = _logits(9, 1, 3001, BF)
    t = torch.arange(0, 3001, 300, device=DEV)
    got = _check(x.expand(t.numel(), 3001), t, 2)
    # one row at one address: the same sums for every target
    assert bool((got.entropy == got.entropy[0]).all()) and bool((got.top_token == got.top_token[0]).all())


@pytest.mark.parametrize("dt,V,top", [(BF, 1000, 20), (HF, 3500, 32), (F, 5119, 5), (BF, 250, 8), (BF, 48001, 20),
                                      (F, 20001, 32)])
def test_scores_of_many_rows(dt, V, top):
    """The forms for many rows: a warp a row, half a CTA a row."""
    x, t = _logits(V, 1300, V, dt)
    t[::7] = -1
    x[3] = -math.inf
    x[3, V // 2] = 1.0
    t[3] = V // 2
    x[4] = 0.25                          # all equal
    x[5, : V // 2] = torch.finfo(dt).min  # a mask of the lowest value
    x[6] = torch.finfo(dt).min
    t[5] = V - 1
    _check(x, t, top)
    x[7, V - 1] = float("nan")
    got = scoring.token_logprobs(x, t, top)
    assert _lib.last_device_error() == (1, 7)
    assert bool(got.logprob[7].isnan()) and got.top_token[7].tolist() == [-1] * top


@pytest.mark.parametrize("rows", [2, 700])
@pytest.mark.parametrize("dt", [BF, HF, F])
def test_scores_under_masks_of_the_lowest_value(rows, dt):
    V = 9000
    x, t = _logits(rows, rows, V, dt)
    low = torch.finfo(dt).min
    x[:, 100:8900] = low
    t.fill_(8950)
    _check(x, t, 32)
    x[0] = low                            # nothing but the mask: every token alike
    t[0] = 5
    _check(x, t, 7)
    x[1, :] = -math.inf
    x[1, 17] = low
    t[1] = 17
    _check(x, t, 3)
