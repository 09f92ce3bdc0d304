"""Keys and values in pages at the ends of what the calls take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("free", [6, 1])                 # room for the three pages, and not
def test_rows_up_to_the_largest_number(free):
    """Slots of 2^31 - 5 rows, with rows of another's in front of them and behind."""
    from ditango_b200 import _capi
    tokens, guard = 2 ** 31 - 5, 1 << 20
    slots = torch.full((guard + tokens + guard,), 7, dtype=torch.int32, device="cuda")
    table, lens, new, pages, count = _i([[0, -1, -1, -1], [-1] * 4]), _i([16, 0]), _i([20, 3]), _i([7, 6, 5, 4, 3, 2, 1, 0]), _i([free])
    cu, out, left, missing = _i([9] * 3), _i([9, 9]), _i([9]), _i([9])
    rc = _capi.load().dtb_extend_pages(table.data_ptr(), lens.data_ptr(), new.data_ptr(), pages.data_ptr(), count.data_ptr(), 2, 4, 8, 16,
                                       slots.data_ptr() + 4 * guard, tokens, cu.data_ptr(), out.data_ptr(), left.data_ptr(), missing.data_ptr(),
                                       torch.cuda.current_stream().cuda_stream)
    _capi.check(rc, "dtb_extend_pages")
    assert bool((slots[:guard] == 7).all()) and bool((slots[guard + tokens:] == 7).all())
    rows = slots[guard:guard + tokens]
    if free == 6:
        assert rows[:23].tolist() == [32 + i for i in range(16)] + [48 + i for i in range(4)] + [64 + i for i in range(3)]
        assert (missing.item(), left.item(), out.tolist(), cu.tolist()) == (0, 3, [36, 3], [0, 20, 23])
        rows = rows[23:]
    else:
        assert (missing.item(), left.item(), out.tolist(), cu.tolist()) == (2, 1, [16, 0], [0, 0, 0])
    for part in rows.split(1 << 28):
        assert bool((part == -1).all())
