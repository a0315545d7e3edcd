"""Limits and overlaps that the adapters' entry point accepts or refuses, before any GPU is asked (pointers are made up)."""
import pytest

from test_device_operator_refusals import adapters

OUT = 1 << 28


def test_most_rows():
    rc, err = adapters(rows=1 << 25, x=None)
    assert rc != 0 and "null" in err, err
    rc, err = adapters(rows=(1 << 25) + 1, x=None)
    assert rc != 0 and "rows must be between 0 and 33554432" in err, err


# buffer of 128 columns: out takes 32 .. 63 (M = 32), x and base lie at some column of it
@pytest.mark.parametrize("x_at,base_at,refused", [
    (64, 0, False), (64, 96, False), (64, None, False), (63, None, True), (0, None, True), (64, 31, True), (64, 33, True), (65, 0, True), (64 + 128, 0, False), (64, 128, False), (64, 128 + 33, True),
])
def test_columns_of_one_buffer(x_at, base_at, refused):
    """x [6, 64], base and out [6, 32] as columns of one array with rows of 128: neighbours in memory that share no element.  (K = 64 columns from 65 on reach the next row's first.)"""
    import torch
    at = lambda c: None if c is None else (1 << 28) + 4 * c  # noqa: E731
    kw = dict(x=at(x_at), ldx=128, rows=6, base=at(base_at), ldb=128, out=at(32), ldo=128)
    if x_at == 65:
        kw["out"] = at(0)  # (row n + 1 of out begins where row n of x ends)
        kw["base"] = None
    if not refused and torch.cuda.is_available():
        pytest.skip("a call with made-up pointers that is not refused")
    rc, err = adapters(**kw)
    assert rc != 0 and ("overlap" in err) == refused, err


def test_other_strides_are_refused_where_the_ranges_meet():
    rc, err = adapters(x=OUT + 4 * 32, ldx=64, rows=6, out=OUT, ldo=128)
    assert "out and x overlap" in err
    rc, err = adapters(x=OUT, ldx=0, rows=6, out=OUT + 4 * 64, ldo=0)
    assert rc != 0
