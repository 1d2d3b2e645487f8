"""GPU tests of dimensions with one entry: their stride says nothing and may be
any number."""
import pytest
import torch

from fast_v2_b200 import _lib, paged, scoring
from tests import _paged_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _ops():
    _lib.ensure_ops()
    _lib.last_device_error()
    yield
    code, info = _lib.last_device_error()
    assert code == 0, f"device error {code} (info {info}) left by the test"


def odd(t, *dims):
    """t's memory with an odd stride in these dimensions of one entry."""
    assert all(t.size(d) == 1 for d in dims)
    return t.as_strided(t.shape, [7 if d in dims else s for d, s in enumerate(t.stride())])


@pytest.mark.parametrize("lens", [[50], [9000]])
def test_attention_of_one_sequence_one_head_one_page(lens):
    g = torch.Generator(device=DEV).manual_seed(1)
    n = lens[0]
    k, v = (torch.randn(1, n, 1, 64, generator=g, device=DEV).to(BF) for _ in range(2))
    q = torch.randn(1, 1, 64, generator=g, device=DEV).to(BF)
    table, length = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = odd(torch.empty(1, 1, 64, dtype=BF, device=DEV), 0, 1)
    paged.decode_attention(odd(q, 0, 1), odd(k, 0, 2), odd(v, 2), odd(table, 1), length, out=out)
    ref, bound = R.attn_plain(q, k, v, table, length, 64 ** -0.5)
    R.assert_within("attention", out, ref, bound)


def test_store_into_a_page_of_one_slot_and_one_head():
    y = torch.randn(1, 3 * 64, device=DEV).to(BF)
    k, v = (torch.zeros(1, 1, 1, 64, dtype=BF, device=DEV) for _ in range(2))
    q, one = torch.empty(1, 1, 64, dtype=BF, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    inv = torch.empty(0, device=DEV)
    paged.norm_rope_store(odd(y, 0), one, inv, q, odd(k, 0, 1, 2), odd(v, 0), one)
    assert torch.equal(torch.cat([q.flatten(), k.flatten(), v.flatten()]), y[0])


def test_scores_of_a_vocabulary_of_one():
    x = torch.randn(4, 6, device=DEV)
    got = scoring.token_logprobs(x[:, ::2][:, :1], torch.zeros(4, dtype=torch.int64, device=DEV), 1)
    assert got.logprob.tolist() == [0.0] * 4 and got.top_token.tolist() == [[0]] * 4
