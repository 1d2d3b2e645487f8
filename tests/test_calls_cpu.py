"""CPU checks of the ways into the operators: compiled calls, hosts without
Python, calls under modes and traces."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from fast_v2_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]


def _fresh(program: str) -> str:
    r = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    return r.stdout


COMPILED = {
    "scores": "scoring.token_logprobs(torch.empty(9, 1000, device='meta'), e(9, torch.int64), 3).top_token",
    "attention": "paged.decode_attention(h(2, 8, 64), h(4, 16, 2, 64), h(4, 16, 2, 64), e((2, 3)), e(2))",
    "slots": "paged.build_slots(e(2), e(2), e((2, 3)), e(9), e(2), 16, e(5, torch.int64), e(5, torch.int64), e(3))",
    "rope": "paged.norm_rope_store(h(5, 12 * 64), e(5, torch.int64), e(16, torch.float32), h(5, 8, 64), "
            "h(4, 16, 2, 64), h(4, 16, 2, 64), e(5, torch.int64))",
    "release": "paged.release_pages(e(2, torch.bool), e(2), e((2, 3)), e(9), e(2), 16)",
}


def test_the_first_call_of_a_process_may_be_compiled():
    calls = ", ".join(f"lambda: {c}" for c in COMPILED.values())
    out = _fresh(f"""
import torch
from fast_v2_b200 import paged, scoring
def e(n, t=torch.int32): return torch.empty(n, dtype=t, device='meta')
def h(*n): return torch.empty(n, dtype=torch.bfloat16, device='meta')
for call in ({calls}):
    def f(x):
        r = call()
        return (r if r is not None else x) + 1
    print(tuple(torch.compile(f, fullgraph=True, backend='eager')(torch.empty(7, device='meta')).shape))
    torch._dynamo.reset()
""")
    assert out.split("\n")[-6:-1] == ["(9, 3)", "(2, 8, 64)", "(7,)", "(7,)", "(7,)"]


HOST = r"""
#include <dlfcn.h>
#include <stdio.h>
int main(int argc, char** argv) {
  for (int i = 1; i < argc; ++i)
    if (!dlopen(argv[i], RTLD_NOW | RTLD_GLOBAL)) {
      puts(dlerror());
      return i;
    }
  return dlsym(RTLD_DEFAULT, "Py_IsInitialized") ? 100 : 0;
}
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not installed")
def test_a_host_without_python_loads_the_torch_operators(tmp_path):
    """libfdl_torch.so registers torch.ops.fdl in a libtorch process that has
    no interpreter."""
    src, exe = tmp_path / "host.c", tmp_path / "host"
    src.write_text(HOST)
    subprocess.run(["gcc", "-std=gnu99", "-Wall", "-Werror", str(src), "-ldl", "-o", str(exe)], check=True)
    torch_lib = Path(torch.__file__).parent / "lib"
    r = subprocess.run([str(exe), str(_lib.LIB_ABI), str(_lib.LIB_TORCH)], capture_output=True, text=True, timeout=600,
                       env=os.environ | {"LD_LIBRARY_PATH": f"{torch_lib}:{os.environ.get('LD_LIBRARY_PATH', '')}"})
    assert r.returncode == 0, r.stdout + r.stderr


def test_derivatives_are_refused_or_not_recorded():
    import torch.autograd.forward_ad as fwd

    _lib.ensure_ops()
    x = torch.randn(3, 10, device="meta")
    t = torch.zeros(3, dtype=torch.int64, device="meta")
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="derivative"):
            torch.ops.fdl.token_logprobs(fwd.make_dual(x, torch.ones_like(x)), t, 2)
    with pytest.raises(RuntimeError, match="derivative"):
        torch.func.jvp(lambda y: torch.ops.fdl.token_logprobs(y, t, 2)[0], (x,), (x,))
    with pytest.raises(RuntimeError, match="derivative"):  # it would hand out zeros
        torch.func.grad(lambda y: torch.ops.fdl.token_logprobs(y, t, 2)[0].sum())(x)
    assert torch.func.grad(lambda y: (y + torch.ops.fdl.token_logprobs(y.detach(), t, 2)[0][:, None]).sum())(x).shape == x.shape
    y = torch.func.vmap(lambda y: torch.ops.fdl.token_logprobs(y, t, 2)[0])(torch.randn(2, 3, 10, device="meta"))
    assert y.shape == (2, 3)
    r = torch.ops.fdl.token_logprobs(x.clone().requires_grad_(), t, 2)
    assert not any(o.requires_grad for o in r)  # as with plain tensors: a backward pass says so
    q = torch.empty(2, 4, 64, dtype=torch.bfloat16, device="meta")
    k = torch.empty(8, 16, 2, 64, dtype=torch.bfloat16, device="meta")
    table, lens = torch.empty((2, 2), dtype=torch.int32, device="meta"), torch.empty(2, dtype=torch.int32, device="meta")
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="derivative"):
            torch.ops.fdl.paged_decode_attn(q, k, fwd.make_dual(k, torch.ones_like(k)), table, lens, 0.1,
                                            torch.empty_like(q))
