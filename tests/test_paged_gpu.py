"""GPU tests of the paged-cache operators against plain 64-bit implementations
(tests/_paged_ref.py, which derives the tolerances)."""
import pytest
import torch

from fast_v2_b200 import _lib, paged, scoring
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


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ slots
def _slots_case(seed, B, page, max_len, new, zero=0.3):
    g = torch.Generator().manual_seed(seed)
    lens = [0 if torch.rand((), generator=g) < zero else int(torch.randint(0, max_len + 1, (), generator=g))
            for _ in range(B)]
    n_new = [int(torch.randint(0, new + 1, (), generator=g)) for _ in range(B)]
    width = R.pages_of(max_len + new, page)
    need = sum(R.pages_of(a + n, page) - R.pages_of(a, page) for a, n in zip(lens, n_new))
    table, free, _ = R.make_table(g, lens, page, width, need + 3, DEV)
    return lens, n_new, table, free


def _run_slots(lens, n_new, table, free, count, page, rows, in_place):
    L, C = i32(lens), i32([count, 0])
    slots = torch.full((rows,), -7, dtype=torch.int64, device=DEV)
    pos = torch.full((rows,), -7, dtype=torch.int64, device=DEV)
    cu = torch.full((len(lens) + 1,), -7, dtype=torch.int32, device=DEV)
    nl, nc = (None, None) if in_place else (torch.full_like(L, -7), i32([-7, 0]))
    paged.build_slots(L, i32(n_new), table, free, C, page, slots, pos, cu, nl, nc)
    if not in_place:
        assert L.tolist() == list(lens) and C.tolist() == [count, 0]
    nl, nc = (L, C) if in_place else (nl, nc)
    assert C[1] == 0
    return slots.tolist(), pos.tolist(), cu.tolist(), table.tolist(), nl.tolist(), int(nc[0])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,page,max_len,new", [(1, 16, 0, 1), (1, 1, 5, 40), (3, 16, 40, 1), (64, 16, 300, 1),
                                                (5, 7, 20, 33), (257, 16, 100, 50), (300, 20, 64, 9),
                                                (4096, 8, 30, 3), (2, 64, 5000, 70000), (31, 128, 1, 500)])
def test_slots(B, page, max_len, new, in_place):
    lens, n_new, table, free = _slots_case(B + page, B, page, max_len, new)
    rows = sum(n_new) + (B % 3) * 100
    ref = R.slots_plain(lens, n_new, table.tolist(), free.tolist(), free.numel(), page, rows)
    got = _run_slots(lens, n_new, table.clone(), free, free.numel(), page, rows, in_place)
    for name, a, b in zip(("slots", "positions", "cu", "table", "lens", "count"), got, ref):
        assert a == b, name
    assert not ref[6]


@pytest.mark.parametrize("what", ["pool", "table", "rows", "negative"])
@pytest.mark.parametrize("B", [7, 600])
def test_slots_refuses_whole_requests(what, B):
    page = 8
    lens, n_new, table, free = _slots_case(B, B, page, 60, 30)
    count, rows = free.numel(), sum(n_new) + 5
    if what == "pool":
        count = count // 2
    elif what == "table":
        lens[B // 2], n_new[B // 2] = 0, table.shape[1] * page + 1
        rows += n_new[B // 2]
    elif what == "rows":
        rows = rows // 3
    else:
        lens[1], n_new[2] = -4, -1
    ref = R.slots_plain(lens, n_new, table.tolist(), free.tolist(), count, page, rows)
    got = _run_slots(lens, n_new, table.clone(), free, count, page, rows, True)
    for name, a, b in zip(("slots", "positions", "cu", "table", "lens", "count"), got, ref):
        assert a == b, name
    assert ref[6]
    code, info = _lib.last_device_error()
    assert code == 2 and info in ref[6]


def test_slots_without_rows_and_strided_table():
    table = torch.full((2, 9), -1, dtype=torch.int32, device=DEV)[:, :4]
    got = _run_slots([0, 3], [0, 0], table, i32([5, 6]), 2, 4, 0, True)
    assert got[2] == [0, 0, 0] and got[4] == [0, 3] and got[5] == 2
    full = torch.full((2, 9), -1, dtype=torch.int32, device=DEV)
    got = _run_slots([0, 0], [5, 1], full[:, :4], i32([5, 6, 7]), 3, 4, 6, True)
    assert got[0] == [28, 29, 30, 31, 24, 20]
    assert full.tolist() == [[7, 6] + [-1] * 7, [5] + [-1] * 8]


def test_release_returns_pages_in_order():
    lens, _, table, free = _slots_case(5, 40, 8, 100, 0)
    F = torch.cat([free, torch.full((int((table >= 0).sum()),), -5, dtype=torch.int32, device=DEV)])
    L, C = i32(lens), i32([free.numel(), 0])
    done = torch.zeros(40, dtype=torch.bool, device=DEV)
    done[::3] = True
    expect = free.tolist()
    for b in range(0, 40, 3):
        expect += [p for p in table[b].tolist() if p >= 0]
    before = table.clone()
    paged.release_pages(done, L, table, F, C, 8)
    assert C.tolist() == [len(expect), 0] and F[: len(expect)].tolist() == expect
    for b in range(40):
        assert int(L[b]) == (0 if b % 3 == 0 else lens[b])
        assert table[b].tolist() == ([-1] * table.shape[1] if b % 3 == 0 else before[b].tolist())
    # nothing done: nothing changes
    paged.release_pages(torch.zeros_like(done), L, table, F, C, 8)
    assert C.tolist() == [len(expect), 0]


def test_release_without_room_or_with_a_bad_length_changes_nothing():
    table = i32([[3, 4], [5, -1]])
    L, C, F = i32([10, 2]), i32([1, 0]), i32([9, 0])
    paged.release_pages(torch.tensor([True, True], device=DEV), L, table, F, C, 8)  # 3 pages, room for 1
    assert _lib.last_device_error() == (1, 4)
    assert L.tolist() == [10, 2] and C.tolist() == [1, 0] and table.tolist() == [[3, 4], [5, -1]]
    L = i32([100, 2])
    paged.release_pages(torch.tensor([True, True], device=DEV), L, table, F, C, 8)
    assert _lib.last_device_error() == (2, 0)
    assert L.tolist() == [100, 0] and C.tolist() == [2, 0] and F.tolist() == [9, 5]


# ------------------------------------------------------------------ rope
def _rope_case(seed, rows, hq, hkv, D, rot, dt, far, norm, page=16, layout="nhd"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    y = torch.randn(rows, (hq + 2 * hkv) * D, generator=g, device=DEV).to(dt)
    pages = R.pages_of(max(rows, 1), page) + 2
    shape = (pages, page, hkv, D)
    if layout == "nhd":
        k, v = (torch.full(shape, 7.0, dtype=dt, device=DEV) for _ in range(2))
    else:
        k, v = (torch.full((pages, hkv, page, D), 7.0, dtype=dt, device=DEV).transpose(1, 2) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:rows].contiguous()
    pos = torch.randint(0, far, (rows,), generator=g, device=DEV)
    inv, _ = paged.rope_frequencies(rot, 1e6, device=DEV) if rot else (torch.empty(0, device=DEV), 1.0)
    w = [(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dt) if norm else None for _ in range(2)]
    return y, pos, inv, slots, k, v, w


def _check_rope(y, pos, inv, slots, k, v, w, hq, hkv, D, inter, scale=1.0, eps=1e-6):
    rows = y.shape[0]
    q = torch.full((rows, hq, D), 5.0, dtype=y.dtype, device=DEV)
    paged.norm_rope_store(y, pos, inv, q, k, v, slots, q_weight=w[0], k_weight=w[1], eps=eps, interleaved=inter,
                          rope_scale=scale)
    x = y.reshape(rows, hq + 2 * hkv, D)
    h = R.half_step(y.dtype)
    tiny = 2.0 ** -25 if y.dtype == HF else 0.0
    rq, sq = R.rope_plain(x[:, :hq], pos, inv, inter, scale, w[0], eps)
    rk, sk = R.rope_plain(x[:, hq:hq + hkv], pos, inv, inter, scale, w[1], eps)
    R.assert_within("q", q, rq, rq.abs() * h + sq * (1 + h) + tiny)
    page = k.shape[1]
    keep = slots >= 0
    at = slots[keep]
    R.assert_within("k", k[at // page, at % page], rk[keep], (rk.abs() * h + sk * (1 + h) + tiny)[keep])
    assert torch.equal(v[at // page, at % page], x[:, hq + hkv:][keep])
    rest = torch.ones(k.shape[:2], dtype=torch.bool, device=DEV)
    rest[at // page, at % page] = False
    assert bool((k[rest] == 7).all()) and bool((v[rest] == 7).all())  # other slots as they were
    return q


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rows,hq,hkv,D,rot,dt,norm", [
    (1, 1, 1, 16, 16, BF, True), (1, 28, 4, 128, 128, BF, True), (33, 28, 4, 128, 64, HF, True),
    (7, 12, 2, 128, 32, BF, False), (65, 14, 2, 64, 64, HF, False), (5, 3, 1, 80, 32, BF, True),
    (9, 16, 2, 256, 256, BF, True), (4, 2, 2, 96, 96, HF, True), (3, 64, 8, 256, 128, HF, True),
    (11, 5, 5, 48, 16, BF, True), (6, 4, 1, 32, 0, BF, True), (2000, 28, 4, 128, 128, BF, True)])
def test_norm_rope_store(rows, hq, hkv, D, rot, dt, norm, inter):
    y, pos, inv, slots, k, v, w = _rope_case(rows + D, rows, hq, hkv, D, rot, dt, 5000, norm)
    slots[rows // 2::3] = -1
    _check_rope(y, pos, inv, slots, k, v, w, hq, hkv, D, inter)


@pytest.mark.parametrize("inter", [False, True])
def test_norm_rope_far_positions_and_scaling(inter):
    inv, scale = paged.rope_frequencies(128, 1e6, factor=32.0, original_len=32768, device=DEV)
    y, pos, _, slots, k, v, w = _rope_case(3, 40, 8, 2, 128, 128, HF, 2 ** 40, True)
    pos[0], pos[1], pos[2] = 0, -3, 2 ** 24 + 1
    # past 2^53 turns / 2^-30 an fp64 angle keeps fewer than 2^-22 of a turn; 2^20 is the longest context in use
    pos[3:] = pos[3:] % (1 << 20)
    _check_rope(y, pos, inv, slots, k, v, w, 8, 2, 128, inter, scale)


@pytest.mark.parametrize("page,layout", [(1, "nhd"), (20, "nhd"), (16, "hnd"), (64, "hnd")])
def test_norm_rope_page_layouts_and_strided_rows(page, layout):
    y, pos, inv, slots, k, v, w = _rope_case(9, 50, 6, 2, 64, 64, BF, 999, True, page, layout)
    wide = torch.zeros(50, y.shape[1] + 40, dtype=BF, device=DEV)
    wide[:, 8:8 + y.shape[1]] = y
    _check_rope(wide[:, 8:8 + y.shape[1]], pos, inv, slots, k, v, w, 6, 2, 64, False)


def test_norm_rope_one_norm_only_and_zero_rows():
    y, pos, inv, slots, k, v, w = _rope_case(2, 10, 6, 2, 64, 32, BF, 999, True)
    _check_rope(y, pos, inv, slots, k, v, [w[0], None], 6, 2, 64, True)
    _check_rope(y, pos, inv, slots, k, v, [None, w[1]], 6, 2, 64, False)
    _check_rope(torch.zeros_like(y), pos, inv, slots, k, v, w, 6, 2, 64, False)  # norm of a zero head: zeros
    q = torch.empty(0, 6, 64, dtype=BF, device=DEV)
    paged.norm_rope_store(y[:0], pos[:0], inv, q, k, v, slots[:0])


def test_norm_rope_slots_outside_the_pool_are_skipped_and_reported():
    y, pos, inv, slots, k, v, w = _rope_case(2, 10, 6, 2, 64, 32, BF, 999, True)
    bad = slots.clone()
    bad[3] = k.shape[0] * k.shape[1]
    q = torch.empty(10, 6, 64, dtype=BF, device=DEV)
    paged.norm_rope_store(y, pos, inv, q, k, v, bad)
    assert _lib.last_device_error() == (1, int(bad[3]))
    assert int((k == 7).all(-1).all(-1).sum()) == k.shape[0] * k.shape[1] - 9
    bad[3] = -2
    paged.norm_rope_store(y, pos, inv, q, k, v, bad)
    assert _lib.last_device_error() == (1, -2)


def test_norm_rope_v_keeps_its_bits():
    y, pos, inv, slots, k, v, w = _rope_case(4, 3, 2, 1, 64, 64, BF, 9, False)
    y[:, 3 * 64:] = torch.tensor([float("nan"), float("inf"), -0.0, 1e-40], device=DEV).to(BF).repeat(16)
    q = torch.empty(3, 2, 64, dtype=BF, device=DEV)
    paged.norm_rope_store(y, pos, inv, q, k, v, slots)
    got = v[slots // 16, slots % 16][:, 0]
    assert torch.equal(got.view(torch.int16), y[:, 3 * 64:].contiguous().view(torch.int16))


# ------------------------------------------------------------------ attention
def _attn_case(seed, lens, hq, hkv, D, page, dt, layout="nhd", q_scale=2.0, poison=True):
    g = torch.Generator().manual_seed(seed)
    width = max(1, R.pages_of(max(lens), page)) + 1
    table, _, n = R.make_table(g, lens, page, width, 2, DEV)
    gd = torch.Generator(device=DEV).manual_seed(seed)
    shape = (n, page, hkv, D)
    k, v = (torch.randn(shape, generator=gd, device=DEV).to(dt) for _ in range(2))
    if layout == "hnd":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    if poison:  # what lies behind a sequence is never looked at
        for b, ln in enumerate(lens):
            if ln % page:
                p = int(table[b, ln // page])
                k[p, ln % page:] = float("nan")
                v[p, ln % page:] = float("inf")
        used = set(table.flatten().tolist())
        for p in range(n):
            if p not in used:
                k[p] = float("inf")
                v[p] = float("nan")
    q = (q_scale * torch.randn(len(lens), hq, D, generator=gd, device=DEV)).to(dt)
    return q, k, v, table, i32(lens)


def _check_attn(q, k, v, table, lens, scale=None, **kw):
    s = q.shape[-1] ** -0.5 if scale is None else scale
    out = paged.decode_attention(q, k, v, table, lens, scale, **kw)
    ref, bound = R.attn_plain(q, k, v, table, lens, s)
    R.assert_within("attention", out, ref, bound)
    return out


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("hq,hkv,D", [(28, 4, 128), (12, 2, 128), (1, 1, 64), (16, 16, 64), (8, 1, 256), (20, 1, 64),
                                      (64, 4, 128), (33, 1, 128), (6, 2, 256)])
def test_attention_lengths(hq, hkv, D, dt):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 127, 200, 0, 513, 1000]
    _check_attn(*_attn_case(hq + D, lens, hq, hkv, D, 16, dt))


@pytest.mark.parametrize("page,layout", [(1, "nhd"), (3, "nhd"), (8, "hnd"), (20, "nhd"), (20, "hnd"), (64, "hnd"),
                                         (256, "nhd"), (1000, "nhd")])
def test_attention_pages(page, layout):
    lens = [1, page, page + 1, 2 * page - 1, 333, 0, 777]
    _check_attn(*_attn_case(page, lens, 14, 2, 128, page, BF, layout))


@pytest.mark.parametrize("lens", [[1], [0], [2], [31], [5000], [40001], [0, 0, 0], [1] * 300, [130] * 40,
                                  [20000, 1, 1, 1, 3, 0, 9000], list(range(150)),
                                  [1000, 1, 0, 63, 64, 65, 129, 1023] * 5])
def test_attention_shapes_of_batches(lens):
    _check_attn(*_attn_case(len(lens), lens, 28, 4, 128, 16, BF))


@pytest.mark.parametrize("hq,hkv,D", [(28, 4, 128), (64, 4, 128), (16, 16, 64), (64, 2, 64), (6, 6, 256)])
@pytest.mark.parametrize("most", [30, 45, 48, 49, 100, 256, 257])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_of_many_short_sequences(hq, hkv, D, most, page):
    lens = [i * 37 % (most + 1) for i in range(330 // hkv * 4 // min(4, hkv) + 300 // hkv)]
    lens[0], lens[1] = most, 0
    q, k, v, table, n = _attn_case(most, lens, hq, hkv, D, page, HF if most % 2 else BF)
    _check_attn(q, k, v, table[:, : R.pages_of(most, page)], n)


@pytest.mark.parametrize("dt,page", [(BF, 16), (HF, 20)])
@pytest.mark.parametrize("hq,hkv,D", [(28, 4, 128), (64, 4, 128), (33, 1, 128), (20, 1, 64), (64, 2, 64), (16, 1, 256),
                                      (3, 3, 256)])
def test_attention_on_one_line(hq, hkv, D, dt, page):
    """Long caches: the tiles of all sequences are shared out over the GPU and
    the pieces joined."""
    _check_attn(*_attn_case(hq, [9000, 5, 0, 700, 64, 16389], hq, hkv, D, page, dt))


def test_attention_on_one_line_with_many_sequences():
    lens = [1] * 150 + [3000] + [0] * 50 + [64, 65, 1500] * 30 + [0]
    _check_attn(*_attn_case(5, lens, 12, 2, 128, 16, BF))
    _check_attn(*_attn_case(6, [0] * 290 + [2000], 12, 2, 128, 16, BF))


def test_attention_peaked_and_flat_scores():
    for qs in (0.0, 30.0):
        q, k, v, table, lens = _attn_case(3, [700, 64, 1], 8, 2, 128, 16, BF, q_scale=qs)
        _check_attn(q, k, v, table, lens)
    # scores that grow along the sequence, and fall (the running maximum moves at every tile, or never)
    q, k, v, table, lens = _attn_case(4, [900, 900], 8, 2, 64, 16, HF, poison=False, q_scale=0.5)
    for b, sign in ((0, 1), (1, -1)):
        at = table[b, :57].long()
        ramp = torch.linspace(-1, 1, 57 * 16, device=DEV).view(57, 16, 1, 1) * sign
        k[at] = (k[at].float() * 0.1 + ramp * q[b].float().mean(0).sign()).to(HF)
    _check_attn(q, k, v, table, lens, 1.0)


def test_attention_strided_q_and_out():
    q, k, v, table, lens = _attn_case(8, [50, 3, 99], 12, 2, 128, 16, BF)
    fused = torch.zeros(3, 16 * 128, dtype=BF, device=DEV)
    fused[:, 128:13 * 128] = q.reshape(3, -1)
    base = torch.full((3, 14, 128), 9.0, dtype=BF, device=DEV)
    out = _check_attn(fused[:, 128:13 * 128].view(3, 12, 128), k, v, table, lens, out=base[:, 1:13])
    assert torch.equal(out, base[:, 1:13]) and bool((base[:, 0] == 9).all()) and bool((base[:, 13] == 9).all())
    wide = torch.full((5, table.shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    wide[:3, :-3] = table
    assert torch.equal(paged.decode_attention(q, k, v, wide[:3, :-3], lens), out.contiguous())


def test_attention_rows_that_share_pages():
    q, k, v, table, lens = _attn_case(8, [160, 10, 99], 12, 2, 128, 16, BF, poison=False)
    table[2, :7] = table[0, :7]  # a shared prompt
    _check_attn(q, k, v, table, lens)


def test_attention_hides_bad_pages_and_reports_them():
    q, k, v, table, lens = _attn_case(8, [160, 10, 99, 40], 12, 2, 128, 16, BF)
    table[0, 3], table[0, 7], table[1, 0] = -1, k.shape[0], 1 << 30
    _check_attn(q, k, v, table, lens)
    code, info = _lib.last_device_error()
    assert code == 1 and info in (-1, k.shape[0], 1 << 30)


def test_attention_clamps_lengths_and_reports_them():
    q, k, v, table, lens = _attn_case(8, [160, 10, 99], 12, 2, 128, 16, BF, poison=False)
    full = table.shape[1] * 16
    table[0, -1] = table[1, 0]
    out = paged.decode_attention(q, k, v, table, i32([10 ** 9, -5, 99]))
    assert _lib.last_device_error()[0] == 2
    ref, bound = R.attn_plain(q, k, v, table, i32([full, 0, 99]), 128 ** -0.5)
    R.assert_within("attention", out, ref, bound)


def test_attention_empty_batch_and_empty_pool():
    q, k, v, table, lens = _attn_case(8, [16], 12, 2, 128, 16, BF)
    assert paged.decode_attention(q[:0], k, v, table[:0], lens[:0]).shape == (0, 12, 128)
    out = paged.decode_attention(q, k[:0], v[:0], table[:, :0], i32([0]))
    assert bool((out == 0).all())


def test_attention_of_infinite_and_nan_values_in_sight():
    q, k, v, table, lens = _attn_case(8, [40, 40], 4, 2, 64, 16, BF, poison=False)
    v[int(table[0, 1]), 3, 0] = float("inf")
    out = paged.decode_attention(q, k, v, table, lens)
    assert bool((out[0, :2] == float("inf")).all()) and bool(out[0, 2:].isfinite().all()) and bool(out[1].isfinite().all())
    k[int(table[1, 0]), 0, 1] = float("nan")
    out = paged.decode_attention(q, k, v, table, lens)
    assert bool(out[1, 2:].isnan().all()) and bool(out[1, :2].isfinite().all())


def test_attention_past_32_bit_offsets():
    """K and V of 2^31 elements and more each; only the pages in use are filled."""
    page, hkv, D = 64, 4, 128
    n = (1 << 31) // (page * hkv * D) + 40
    k, v = (torch.empty(n, page, hkv, D, dtype=BF, device=DEV) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(1)
    table = i32([[n - 1, 0, n - 30, n // 2], [n - 2, n - 3, 7, 9]])
    for p in table.flatten().tolist():
        k[p] = torch.randn(page, hkv, D, generator=g, device=DEV).to(BF)
        v[p] = torch.randn(page, hkv, D, generator=g, device=DEV).to(BF)
    q = torch.randn(2, 28, D, generator=g, device=DEV).to(BF)
    _check_attn(q, k, v, table, i32([250, 100]))
    y = torch.randn(2, 36 * D, generator=g, device=DEV).to(BF)
    slots = torch.tensor([n * page - 1, (n - 30) * page + 2], device=DEV)
    pos = torch.tensor([5, 6], device=DEV)
    inv, _ = paged.rope_frequencies(D, device=DEV)
    paged.norm_rope_store(y, pos, inv, q, k, v, slots)
    assert torch.equal(v[n - 1, 63], y[0, 32 * D:].view(4, D)) and torch.equal(v[n - 30, 2], y[1, 32 * D:].view(4, D))


def test_attention_on_another_stream_and_twice_at_once():
    a = _attn_case(1, [3000, 20, 500], 28, 4, 128, 16, BF)
    b = _attn_case(2, [100, 9000], 28, 4, 128, 16, BF)
    ra, rb = paged.decode_attention(*a), paged.decode_attention(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            got.append((paged.decode_attention(*a), ra))
        with torch.cuda.stream(s2):
            got.append((paged.decode_attention(*b), rb))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, y)  # and the same bits on every run


def test_attention_in_two_graphs_replayed_at_once():
    a = _attn_case(1, [3000, 20, 500], 28, 4, 128, 16, BF)
    b = _attn_case(2, [100, 9000], 28, 4, 128, 16, BF)
    want = [paged.decode_attention(*a), paged.decode_attention(*b)]
    graphs, outs, streams = [], [], []
    for c in (a, b):
        out = torch.empty_like(c[0])
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st):
            paged.decode_attention(*c, out=out)
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=st):
                paged.decode_attention(*c, out=out)
        graphs.append(g)
        outs.append(out)
        streams.append(st)
    for out in outs:
        out.fill_(3)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)
    # new lengths in place are seen by the next replay
    a[4].copy_(i32([100, 0, 400]))
    graphs[0].replay()
    torch.cuda.synchronize()
    ref, bound = R.attn_plain(*a, 128 ** -0.5)
    R.assert_within("replayed", outs[0], ref, bound)


def test_paged_ops_refuse_what_does_not_fit():
    q, k, v, table, lens = _attn_case(8, [16, 3], 12, 2, 128, 16, BF)
    ok = dict(q=q, k=k, v=v, t=table, n=lens)
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(q=q[:, :, ::2]), dict(k=k[:, :, :, :64], v=v[:, :, :, :64]),
                dict(v=v[:, :8]), dict(q=q[:, :11]), dict(t=table[:1]), dict(t=table.long()), dict(n=lens.long()),
                dict(n=lens[:1]), dict(n=lens.cpu()), dict(t=table.cpu()), dict(q=q[0])):
        a = ok | bad
        with pytest.raises(RuntimeError):
            paged.decode_attention(a["q"], a["k"], a["v"], a["t"], a["n"])
    y, pos, inv, slots, k, v, w = _rope_case(2, 10, 6, 2, 64, 32, BF, 999, True)
    q = torch.empty(10, 6, 64, dtype=BF, device=DEV)
    for args in ((y.float(), pos, inv, q, k, v, slots), (y, pos.int(), inv, q, k, v, slots),
                 (y, pos, inv.double(), q, k, v, slots), (y, pos, inv, q[:9], k, v, slots),
                 (y, pos, inv[:3], q, k, v, slots), (y, pos, inv, q, k, v[:1], slots), (y, pos, inv, q, k, v, slots[:9]),
                 (y[:, :576], pos, inv, q, k, v, slots), (y, pos, inv, q.half(), k, v, slots)):
        with pytest.raises(RuntimeError):
            paged.norm_rope_store(*args)
    with pytest.raises(RuntimeError):
        paged.norm_rope_store(y, pos, inv, q, k, v, slots, q_weight=w[0].float())


# ------------------------------------------------------------------ a run of them together
@pytest.mark.parametrize("dt,graph", [(BF, False), (HF, False), (BF, True)])
def test_a_serving_run(dt, graph):
    """Sequences of different lengths are prefilled, decoded token by token,
    released and taken again; every step's attention and scores are compared
    with plain ones over a cache kept densely on the side."""
    B, hq, hkv, D, page, V, steps = 5, 6, 2, 64, 8, 700, 12
    g = torch.Generator(device=DEV).manual_seed(0)
    cache = paged.PagedKVCache(1, 40, page, B, 64, hkv, D, dt, DEV)
    inv, _ = paged.rope_frequencies(D, 1e4, device=DEV)
    head = (torch.randn(hq * D, V, generator=g, device=DEV) * 0.3).to(dt)
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dt) for _ in range(2))
    dense = [[] for _ in range(B)]  # (k, v) rows per sequence, as the kernel stored them
    h = R.half_step(dt)

    def remember(y, pos, n):
        x = y.view(-1, hq + 2 * hkv, D)
        rk, sk = R.rope_plain(x[:, hq:hq + hkv], pos, inv, False, 1.0, kw)
        t = 0
        for b in range(B):
            for _ in range(n[b]):
                dense[b].append((rk[t], sk[t] + rk[t].abs() * h, x[t, hq + hkv:].clone()))
                t += 1

    def compare():
        """The pages hold what was put there, in order."""
        for b in range(B):
            assert int(cache.lens[b]) == len(dense[b])
            for p, (rk, bk, rv) in enumerate(dense[b]):
                pg = int(cache.block_table[b, p // page])
                R.assert_within("k", cache.k_pages[0][pg, p % page], rk, bk * (1 + h) + 2 ** -25)
                assert torch.equal(cache.v_pages[0][pg, p % page], rv)

    n = [9, 0, 8, 1, 20]
    y = torch.randn(sum(n), (hq + 2 * hkv) * D, generator=g, device=DEV).to(dt)
    slots, pos, cu = cache.extend(i32(n), sum(n))
    cache.store(0, y, pos, slots, inv, hq, q_weight=qw, k_weight=kw)
    assert cu.tolist() == [0, 9, 9, 17, 18, 38]
    remember(y, pos, n)
    compare()

    n_new = i32([1] * B)
    y = torch.empty(B, (hq + 2 * hkv) * D, dtype=dt, device=DEV)
    targets = torch.randint(0, V, (B,), generator=g, device=DEV)

    def step():
        slots, pos, _ = cache.extend(n_new, B)
        q = cache.store(0, y, pos, slots, inv, hq, q_weight=qw, k_weight=kw)
        o = cache.attend(0, q)
        logits = o.view(B, -1) @ head
        return pos, q, o, logits, scoring.token_logprobs(logits, targets, 5)

    replay = None
    if graph:  # captured after a warm-up on the side, whose changes are taken back
        keep = [t.clone() for t in (cache.lens, cache.block_table, cache.free_pages, cache.free_count)]
        y.normal_(generator=g)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step()
        torch.cuda.current_stream().wait_stream(st)
        replay = torch.cuda.CUDAGraph()
        with torch.cuda.graph(replay):
            outs = step()
        for t, s in zip((cache.lens, cache.block_table, cache.free_pages, cache.free_count), keep):
            t.copy_(s)
    for i in range(steps):
        y.copy_(torch.randn(y.shape, generator=g, device=DEV))
        if i == 6:  # sequence 4 ends, its row is taken again
            done = torch.tensor([False] * 4 + [True], device=DEV)
            cache.release(done)
            dense[4] = []
        if replay is not None:
            replay.replay()
            pos, q, o, logits, sc = outs
        else:
            pos, q, o, logits, sc = step()
        assert pos.tolist() == [len(d) for d in dense]
        remember(y, pos, [1] * B)
        ref, bound = R.attn_plain(q, cache.k_pages[0], cache.v_pages[0], cache.block_table, cache.lens, D ** -0.5)
        R.assert_within("attention", o, ref, bound)
        lp, ent, tlp, tok, bl, be = R.scores_plain(logits, targets, 5)
        R.assert_within("logprob", sc.logprob, lp, bl + lp.abs() * R.U32)
        R.assert_within("entropy", sc.entropy, ent, be)
        assert torch.equal(sc.top_token, tok)
        R.assert_within("top", sc.top_logprob, tlp, bl[:, None] + tlp.abs() * R.U32)
    compare()
    held = sum(R.pages_of(len(d), page) for d in dense)
    assert int(cache.free_count[0]) == 40 - held
    pages = [p for row in cache.block_table.tolist() for p in row if p >= 0]
    assert len(pages) == held and sorted(pages + cache.free_pages[: 40 - held].tolist()) == list(range(40))


# ------------------------------------------------------------------ ways to call
class _Sub(torch.Tensor):
    """A subclass without behaviour of its own: calls go through torch.ops."""


def test_direct_and_dispatched_calls_agree():
    a = _attn_case(1, [300, 20, 500], 28, 4, 128, 16, BF)
    want = paged.decode_attention(*a)
    out = torch.empty_like(want)
    assert _lib.direct().paged_decode_attn(*a, 128 ** -0.5, out) is None  # plain tensors need no dispatcher
    assert torch.equal(out, want)
    assert _lib.direct().paged_decode_attn(a[0].as_subclass(_Sub), *a[1:], 128 ** -0.5, out) is NotImplemented
    out.zero_()
    torch.ops.fdl.paged_decode_attn(*a, 128 ** -0.5, out)
    assert torch.equal(out, want)
    out.zero_()
    paged.decode_attention(a[0].as_subclass(_Sub), *a[1:], out=out)
    assert torch.equal(out, want)
    x = torch.randn(9, 1000, device=DEV)
    t = torch.arange(9, device=DEV)
    r = scoring.token_logprobs(x, t, 3)
    for other in (torch.ops.fdl.token_logprobs(x, t, 3), scoring.token_logprobs(x.as_subclass(_Sub), t, 3)):
        for u, v in zip(r, other):
            assert torch.equal(u, torch.Tensor(v) if isinstance(v, _Sub) else v)
    assert all(not u.requires_grad for u in r)


def test_compiled_calls():
    a = _attn_case(1, [300, 20, 500], 28, 4, 128, 16, BF)
    x = torch.randn(9, 1000, device=DEV)
    t = torch.arange(9, device=DEV)

    def f(a, x, t):
        o = paged.decode_attention(*a)
        r = scoring.token_logprobs(x * 2, t, 3)
        return o + 1, r.logprob, r.top_token

    want = f(a, x, t)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(a, x, t)
    for u, v in zip(want, got):
        assert torch.equal(u, v)


def test_calls_from_threads():
    import threading

    a = _attn_case(1, [300, 20, 500], 28, 4, 128, 16, BF)
    want = paged.decode_attention(*a)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(paged.decode_attention(*a), want):
                    bad.append(1)

    ts = [threading.Thread(target=work) for _ in range(4)]
    for th in ts:
        th.start()
    for th in ts:
        th.join()
    assert not bad
