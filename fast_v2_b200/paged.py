"""Paged KV cache: a pool of pages shared by all sequences, and the operators
of a serving step over it.

A page holds ``page_size`` tokens of one sequence, for all KV heads of a
layer; ``block_table[b]`` (int32) names the pages of sequence b, a *slot* is
``page * page_size + offset``.  Unlike :class:`StaticKVCache`, which reserves
``max_seq_len`` rows per sequence, memory follows the tokens that are there.
One step runs

    build_slots       table entries, slots and positions of the new tokens
    norm_rope_store   q/k/v split, head norms, rotary positions, K/V -> pages
    decode_attention  one query token per sequence over its pages
    release_pages     pages of finished sequences back to the pool

Everything runs on torch's current stream and stays on the device: lengths,
tables and the pool are read and updated by the kernels, so a step can be
captured in a CUDA graph and replayed.  Forward only: nothing is recorded for
autograd, and inputs with forward-mode tangents are refused.

:class:`PagedKVCache` keeps the buffers of a model and calls the operators.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.compiler import is_compiling

from . import _lib

MAX_BATCH = 4096

_lib.load_if_built()


def _call(name: str, *args) -> None:
    """An operator without a result: straight into the library for plain CUDA
    tensors, through torch.ops.fdl otherwise and while compiling."""
    if is_compiling():
        getattr(torch.ops.fdl, name)(*args)
        return
    if getattr(_lib.direct(), name)(*args) is NotImplemented:
        getattr(torch.ops.fdl, name)(*args)


def build_slots(lens, n_new, block_table, free_pages, free_count, page_size: int, slots, positions, cu_seqlens,
                new_lens=None, new_count=None) -> None:
    """Extend the block table by ``n_new[b]`` tokens per sequence and write
    the slot and position of each (packed, sequence after sequence).

    lens, n_new int32 [B]; block_table int32 [B, max_pages], new entries are
    written in place; free_pages int32, a stack whose first free_count[0]
    entries are free; free_count int32 [2] (the second entry is scratch, 0).
    Writes slots, positions int64 [rows] (-1 and 0 behind the last token),
    cu_seqlens int32 [B + 1], and the new lengths and free count to
    new_lens [B] and new_count [2] (no values needed before), in place on lens
    and free_count where not given.  A sequence that cannot be served (no free
    page, no room in its table row or in ``slots``, no table entry for the page
    it has begun) is refused whole and reported in the device status: slots -1,
    its length unchanged.
    """
    _call("page_slots", lens, n_new, block_table, free_pages, free_count, page_size, slots, positions, cu_seqlens,
          new_lens, new_count)


def release_pages(done, lens, block_table, free_pages, free_count, page_size: int) -> None:
    """Return the pages of the sequences with ``done[b]`` (bool [B]) to the
    pool; their table entries become -1 and their lengths 0.  The pool counts no
    owners: a page that stands in the table rows of two sequences goes back with
    the first, and once more with the second."""
    _lib.ensure_ops()
    torch.ops.fdl.page_release(done, lens, block_table, free_pages, free_count, page_size)


def rope_frequencies(rot_dim: int, base: float = 1e6, *, factor: float = 1.0, original_len: Optional[int] = None,
                     beta_fast: float = 32.0, beta_slow: float = 1.0, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq fp32 [rot_dim / 2], scale of cos and sin) of rotary positions.

    factor 1: base ** (-2j / rot_dim), scale 1.  factor > 1 without
    original_len: positions divided by the factor (linear interpolation).
    With original_len (the length the model was trained on), by parts as in
    YaRN (Peng et al. 2023): frequencies that turn more than beta_fast times
    over original_len stay, those below beta_slow are divided by the factor,
    a linear ramp over the index in between; cos and sin are scaled by
    0.1 ln(factor) + 1.
    """
    if rot_dim % 2 or rot_dim < 2:
        raise ValueError(f"rope_frequencies: rot_dim={rot_dim} must be even and positive")
    if factor < 1:
        raise ValueError(f"rope_frequencies: factor={factor} must be at least 1")
    f = base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    scale = 1.0
    if factor > 1 and original_len is None:
        f = f / factor
    elif factor > 1:
        def index(turns):  # the pair that makes this many turns over original_len
            return rot_dim * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo = max(math.floor(index(beta_fast)), 0)
        hi = min(math.ceil(index(beta_slow)), rot_dim - 1)
        ramp = ((torch.arange(rot_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    return f.to(device=device, dtype=torch.float32), scale


def norm_rope_store(y, positions, inv_freq, q, k_pages, v_pages, slots, *, q_weight=None, k_weight=None,
                    eps: float = 1e-6, interleaved: bool = False, rope_scale: float = 1.0) -> None:
    """Split the rows of the fused projection ``y`` [rows, (hq + 2 hkv) * D]
    (bf16 or fp16), norm each query and key head where a weight [D] is given,
    turn the first 2 * len(inv_freq) elements of these heads by positions *
    inv_freq, and write q [rows, hq, D] and the K and V rows into their slots
    of the pages [num_pages, page_size, hkv, D] (slot -1: not stored).

    interleaved: pairs (2j, 2j + 1) instead of (j, j + rot / 2).  D a multiple of
    16 up to 256, len(inv_freq) a multiple of 8.  fp32
    arithmetic, one rounding; the angle of a far position is exact (fp64).
    q may not share memory with y, nor two rows a slot.
    """
    _call("norm_rope_store", y, positions, inv_freq, q_weight, k_weight, eps, interleaved, rope_scale, q, k_pages,
          v_pages, slots)


def decode_attention(q, k_pages, v_pages, block_table, lens, scale: Optional[float] = None, out=None):
    """Attention of one query token per sequence, q [B, hq, D] (bf16 or fp16,
    D 64, 128 or 256), over the first lens[b] (int32 [B]) tokens of its pages
    [num_pages, page_size, hkv, D].  Returns [B, hq, D] (``out`` if given);
    a sequence of length 0 gives zeros.  scale: D ** -0.5 if not given.  ``out``
    may not share memory with the inputs.

    How the work is shared out follows from the table's width, not from the
    lengths, which stay on the device: where a caller knows that they are short,
    a slice block_table[:, :n] that covers them is faster (30 sequences of 320
    keys 6.0 us, in a table for 32768 tokens 10.5)."""
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _call("paged_decode_attn", q, k_pages, v_pages, block_table, lens, q.shape[-1] ** -0.5 if scale is None else scale,
          out)
    return out


class PagedKVCache:
    """Pages, block table, lengths and free pages of one model's sequences.

    ``k_pages[l]`` / ``v_pages[l]`` are [num_pages, page_size, kv_heads, D].
    ``batch`` rows exist from the start, all empty; a row is taken by adding
    tokens to it and freed by :meth:`release`.
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, batch: int, max_seq_len: int,
                 num_kv_heads: int, head_dim: int, dtype: torch.dtype, device):
        _lib.ensure_ops()
        if not 1 <= batch <= MAX_BATCH:
            raise ValueError(f"PagedKVCache: batch={batch} is outside [1, {MAX_BATCH}]")
        if min(num_layers, num_pages, page_size, max_seq_len, num_kv_heads) < 1:
            raise ValueError("PagedKVCache: layers, pages, page size, length and heads must be positive")
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        self.batch, self.max_seq_len = batch, max_seq_len
        shape = (num_pages, page_size, num_kv_heads, head_dim)
        self.k_pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.v_pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((batch, -(-max_seq_len // page_size)), -1, **i32)
        self.lens = torch.zeros(batch, **i32)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)  # page 0 is taken first
        self.free_count = torch.tensor([num_pages, 0], **i32)

    def extend(self, n_new: torch.Tensor, rows: int):
        """Make room for n_new[b] (int32 [batch]) tokens per sequence; ``rows``
        >= their sum.  Returns (slots, positions, cu_seqlens) of the packed
        tokens; ``lens`` counts them from now on."""
        slots, positions = torch.empty((2, rows), dtype=torch.int64, device=self.lens.device).unbind(0)
        cu = torch.empty(self.batch + 1, dtype=torch.int32, device=self.lens.device)
        build_slots(self.lens, n_new, self.block_table, self.free_pages, self.free_count, self.page_size, slots,
                    positions, cu)
        return slots, positions, cu

    def store(self, layer: int, y, positions, slots, inv_freq, q_heads: int, **kw):
        """norm_rope_store into this layer's pages; returns q [rows, q_heads, D]."""
        q = torch.empty((y.shape[0], q_heads, self.k_pages[layer].shape[3]), dtype=y.dtype, device=y.device)
        norm_rope_store(y, positions, inv_freq, q, self.k_pages[layer], self.v_pages[layer], slots, **kw)
        return q

    def attend(self, layer: int, q, scale: Optional[float] = None, out=None):
        """One query token per sequence, q [batch, hq, D], over its pages."""
        return decode_attention(q, self.k_pages[layer], self.v_pages[layer], self.block_table, self.lens, scale, out)

    def release(self, done: torch.Tensor) -> None:
        """Free the rows with done[b] (bool [batch])."""
        release_pages(done, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size)
