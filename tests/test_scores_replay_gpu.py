"""GPU test of captured token scores over new values."""
import pytest
import torch

from fast_v2_b200 import _lib, scoring
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


@pytest.mark.parametrize("rows,V", [(8, 152064), (200, 9001), (700, 20000), (1300, 1000)])
def test_scores_replayed_over_new_logits(rows, V):
    """In each form of the kernel: every output of a replay is that of a call
    on the new values."""
    g = torch.Generator(device=DEV).manual_seed(V)
    fresh = lambda: 3 * torch.randn(rows, V, generator=g, device=DEV)  # noqa: E731
    x, t = fresh().to(BF), torch.randint(0, V, (rows,), generator=g, device=DEV)
    scoring.token_logprobs(x, t, 20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = scoring.token_logprobs(x, t, 20)
    for _ in range(2):
        x.copy_(fresh())
        t.copy_(torch.randint(0, V, (rows,), generator=g, device=DEV))
        graph.replay()
        for a, b in zip(r, scoring.token_logprobs(x, t, 20)):
            assert torch.equal(a, b)
        lp, ent, tlp, tok, bl, be = R.scores_plain(x, t, 20)
        R.assert_within("logprob", r.logprob, lp, bl + lp.abs() * R.U32)
        R.assert_within("entropy", r.entropy, ent, be)
        assert torch.equal(r.top_token, tok)
