"""GPU tests of the counts and tables that one step of build_slots hands to the
next."""
import pytest
import torch

from fast_v2_b200 import _lib, paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.fixture(autouse=True)
def _ops():
    _lib.ensure_ops()
    _lib.last_device_error()
    yield
    code, info = _lib.last_device_error()
    assert code == 0, f"device error {code} (info {info}) left by the test"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def i64(n):
    return torch.full((n,), -7, dtype=torch.int64, device=DEV)


@pytest.mark.parametrize("garbage", [-1, 1, 12345])
@pytest.mark.parametrize("rows", [1, 3000])
def test_new_count_serves_as_the_next_calls_count(rows, garbage):
    """new_lens and new_count need no values before the call, and are lens and
    free_count of the next one -- with one CTA and with many."""
    B, page, pages = 3, 8, 2000
    table = torch.full((B, 1500), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(pages, dtype=torch.int32, device=DEV)
    lens, count = i32([0] * B), i32([pages, 0])
    n_new = i32([rows, 0, 0])
    for step in range(1, 4):
        new_lens, new_count = i32([garbage] * B), i32([garbage] * 2)
        slots, pos, cu = i64(rows), i64(rows), i32([0] * (B + 1))
        paged.build_slots(lens, n_new, table, free, count, page, slots, pos, cu, new_lens, new_count)
        assert new_lens.tolist() == [step * rows, 0, 0]
        assert new_count.tolist() == [pages - -(-step * rows // page), 0]
        assert pos.tolist() == list(range((step - 1) * rows, step * rows))
        lens, count = new_lens, new_count
    used = table[table >= 0].tolist()
    assert len(set(used)) == len(used) == -(-3 * rows // page)


def _build(lens, n_new, table, free, page, rows):
    L, C = i32(lens), i32([len(free), 0])
    slots, pos, cu = i64(rows), i64(rows), i32([0] * (len(lens) + 1))
    T = i32(table)
    paged.build_slots(L, i32(n_new), T, i32(free), C, page, slots, pos, cu)
    return slots.tolist(), L.tolist(), C.tolist(), T.tolist()


def test_a_request_whose_begun_page_is_missing_is_refused_whole():
    # page 4: row 0 has 5 tokens and no page for the fifth; rows 1 and 3 are whole; row 2 gets nothing
    slots, lens, count, table = _build([5, 4, 6, 0], [6, 2, 0, 3], [[7, -1, -1], [8, -1, -1], [9, -1, -1], [-1] * 3],
                                       [0, 1, 2, 3], 4, 12)
    assert _lib.last_device_error() == (2, 0)
    assert slots == [-1] * 6 + [12, 13] + [8, 9, 10] + [-1]
    assert lens == [5, 6, 6, 3] and count == [2, 0]
    assert table == [[7, -1, -1], [8, 3, -1], [9, -1, -1], [2, -1, -1]]
    # a hole in a page that is full already is not in the way of new tokens
    slots, lens, count, table = _build([8], [2], [[-1, 5, -1]], [3], 4, 2)
    assert slots == [12, 13] and lens == [10] and count == [0, 0] and table == [[-1, 5, 3]]


@pytest.mark.parametrize("B,n", [(300, 2), (2000, 1), (40, 30)])
def test_missing_pages_among_many_requests(B, n):
    page, width = 8, 6
    lens = [b * 7 % 40 if b % 3 else 0 for b in range(B)]
    n_new = [n if lens[b] + n <= page * width else 0 for b in range(B)]
    table, pool = [], iter(range(B * width))
    for ln in lens:
        table.append([next(pool) if i < -(-ln // page) else -1 for i in range(width)])
    free = list(pool)
    hole = [b for b in range(B) if b % 5 == 1 and lens[b] % page and n_new[b]]
    for b in hole:
        table[b][lens[b] // page] = -1
    top, want_slots, want_lens = len(free), [], []
    want = [list(r) for r in table]
    for b in range(B):
        if b in hole:
            want_slots += [-1] * n_new[b]
            want_lens.append(lens[b])
            continue
        for p in range(lens[b], lens[b] + n_new[b]):
            if p % page == 0:
                top -= 1
                want[b][p // page] = free[top]
            want_slots.append(want[b][p // page] * page + p % page)
        want_lens.append(lens[b] + n_new[b])
    slots, got_lens, count, got = _build(lens, n_new, table, free, page, len(want_slots))
    code, info = _lib.last_device_error()
    assert hole and code == 2 and info in hole
    assert slots == want_slots and got_lens == want_lens and count == [top, 0] and got == want


def test_a_negative_page_on_the_stack_is_reported():
    slots, lens, count, table = _build([0, 0], [2, 1], [[-1], [-1]], [4, -3], 4, 3)
    assert _lib.last_device_error() == (1, -3)
    assert slots == [-1, -1, 16] and lens == [2, 1] and count == [0, 0]
