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
