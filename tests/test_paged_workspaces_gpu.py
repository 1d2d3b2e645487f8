"""GPU tests of calls in flight at once that need a workspace each."""
import threading

import pytest
import torch

from fast_v2_b200 import _lib, paged
from tests import _paged_ref as R
from tests.test_paged_gpu import _attn_case

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


def _line_case(seed, lens=(9000, 20, 500)):
    """A call on the line, with its checked result."""
    case = _attn_case(seed, list(lens), 28, 4, 128, 16, BF)
    q, k, v, table, n = case
    width = table.shape[1] * k.shape[1]
    assert _lib.abi().fdl_paged_attn_workspace_bytes(q.shape[0], 28, 4, 128, width) > 0
    want = paged.decode_attention(*case)
    ref, bound = R.attn_plain(q, k, v, table, n, 128 ** -0.5)
    R.assert_within("attention", want, ref, bound)
    return case, want


def test_calls_on_streams_have_a_workspace_each():
    cases = [_line_case(s, lens) for s, lens in ((1, (9000, 20, 500)), (2, (100, 9000)), (3, (9500, 9000, 1)))]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for st, (case, want) in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append((paged.decode_attention(*case), want))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, b)


def test_graphs_replayed_at_once_have_a_workspace_each():
    cases = [_line_case(s, lens) for s, lens in ((4, (9000, 20, 500)), (5, (100, 9000)), (6, (9100, 9100, 64)))]
    graphs = []
    for case, want in cases:
        out, st, g = torch.empty_like(want), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=st):
            for _ in range(4):
                paged.decode_attention(*case, out=out)
        graphs.append((g, st, out))
    for _, _, out in graphs:
        out.fill_(3)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, st, _ in graphs:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, _, out), (_, want) in zip(graphs, cases):
        assert torch.equal(out, want)


def test_calls_from_threads_have_a_workspace_each():
    cases = [_line_case(10 + s, (9000 + 100 * s, 30 * s, 500)) for s in range(4)]
    torch.cuda.synchronize()
    bad = []

    def work(case, want):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            outs = [paged.decode_attention(*case) for _ in range(30)]
            st.synchronize()
            bad.extend(1 for o in outs if not torch.equal(o, want))

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
