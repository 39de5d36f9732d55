"""amp_device_status reports what kernels met one kind at a time, and loses none of it."""
import pytest
import torch

from amp_b200 import paged
from amp_b200._lib import lib

pytestmark = pytest.mark.gpu


def bad_page():
    """A page id outside the pool: skipped by the decode."""
    q = torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16, device="cuda")
    table, ctx = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[5]], [3]))
    paged.paged_attn_decode(q, pool, pool, table, ctx, 16)


def bad_row():
    """A row outside the table: skipped."""
    table, ctx, rows = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in ((2, 3), 2, 1))
    paged.free_sequences(table, ctx, rows + 7)


def message():
    return lib().amp_last_error().decode()


@pytest.mark.parametrize("order", [(bad_page, bad_row), (bad_row, bad_page)])
def test_both_kinds_are_reported(order, cuda, amp_lib):
    assert amp_lib.amp_device_status(1) == 0
    for kind in order:
        kind()
    for _ in range(2):                                     # reading alone clears nothing
        assert amp_lib.amp_device_status(0) == -1 and "page id" in message()
    assert amp_lib.amp_device_status(1) == -1 and "page id" in message()
    assert amp_lib.amp_device_status(1) == -1 and "row" in message()
    assert amp_lib.amp_device_status(1) == 0
    bad_row()
    assert amp_lib.amp_device_status(1) == -1 and "row" in message()
    assert amp_lib.amp_device_status(1) == 0
