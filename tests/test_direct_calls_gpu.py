"""GPU tests of calls that torch watches: traces, function modes, the profiler,
derivatives.  The entries for plain tensors may not pass them by."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.overrides import TorchFunctionMode

from fast_v2_b200 import _lib, paged, scoring

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


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _calls(seed=0):
    """name -> (function of one tensor, that tensor)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)  # noqa: E731
    k, v, table, lens = r(8, 16, 2, 64), r(8, 16, 2, 64), i32([[1, 5], [7, 0]]), i32([20, 9])
    targets = torch.tensor([3, 5, -1], device=DEV)
    pos, slots = torch.tensor([4, 9], device=DEV), torch.tensor([17, 70], device=DEV)
    inv, _ = paged.rope_frequencies(64, device=DEV)

    def rope(y):
        q, kp, vp = torch.zeros(2, 4, 64, dtype=BF, device=DEV), torch.zeros_like(k), torch.zeros_like(k)
        paged.norm_rope_store(y, pos, inv, q, kp, vp, slots)
        return torch.cat([q.flatten(), kp.flatten(), vp.flatten()])

    def slots_of(n_new):
        t, s, p = table.clone(), torch.zeros(6, dtype=torch.int64, device=DEV), torch.zeros(6, dtype=torch.int64, device=DEV)
        paged.build_slots(lens.clone(), n_new, t, i32([2, 3]), i32([2, 0]), 16, s, p, i32([0] * 3))
        return torch.cat([s, p])

    return {"paged_decode_attn": (lambda q: paged.decode_attention(q, k, v, table, lens, 0.125), r(2, 4, 64)),
            "token_logprobs": (lambda x: torch.cat(scoring.token_logprobs(x, targets, 4)[:2]), r(3, 999)),
            "norm_rope_store": (rope, r(2, 8 * 64)),
            "page_slots": (slots_of, i32([2, 3]))}


NAMES = ["paged_decode_attn", "token_logprobs", "norm_rope_store", "page_slots"]


@pytest.mark.parametrize("name", NAMES)
def test_a_trace_records_the_call(name):
    f, x = _calls()[name]
    traced = torch.jit.trace(f, (x,), check_trace=False)
    assert f"fdl::{name}" in str(traced.graph)
    other = _calls(1)[name][1] if name != "page_slots" else i32([1, 4])
    assert torch.equal(traced(other), f(other))


@pytest.mark.parametrize("name", NAMES)
def test_a_function_mode_sees_the_call(name):
    f, x = _calls()[name]
    want, seen = f(x), []

    class Mode(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Mode():
        got = f(x)
    assert torch.equal(got, want) and any(name in s for s in seen)


@pytest.mark.parametrize("name", NAMES)
def test_the_profiler_names_the_call(name):
    f, x = _calls()[name]
    f(x)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        f(x)
    assert f"fdl::{name}" in {e.key for e in prof.key_averages()}


@pytest.mark.parametrize("name", NAMES[:3])
def test_forward_mode_derivatives_are_refused(name):
    f, x = _calls()[name]
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="derivative"):
            f(fwd.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="derivative"):
        torch.func.jvp(f, (x,), (x,))
    f(x)


def test_the_plain_entry_is_taken_without_any_of_them():
    logits, targets = torch.randn(3, 99, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    assert _lib.direct().token_logprobs(logits, targets, 2) is not NotImplemented
    with torch.no_grad():
        assert _lib.direct().token_logprobs(logits, targets, 2) is not NotImplemented
    with torch.inference_mode():
        assert _lib.direct().token_logprobs(logits, targets, 2) is not NotImplemented
    with torch.autocast("cuda"):
        assert _lib.direct().token_logprobs(logits, targets, 2) is not NotImplemented


@pytest.mark.parametrize("name", NAMES[:3])
def test_inputs_that_want_gradients_get_none_in_any_way_of_calling(name):
    f, x = _calls()[name]
    want, x = f(x), x.requires_grad_()
    assert torch.equal(f(x), want) and not f(x).requires_grad
    got = torch.compile(f, backend="aot_eager")(x)
    assert torch.equal(got, want) and not got.requires_grad
    y = x * 1.0
    assert torch.equal(f(y), want) and not f(y).requires_grad
