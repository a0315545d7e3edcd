"""The largest numbers of rows and slots of rsv_adapters_apply, and blocks of 4096 rows with few rows behind them."""
import pytest

from test_gpu_adapters import apply, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [4095, 4096])
@pytest.mark.parametrize("rows", [20, 700, 5000, 9000])
def test_many_slots(rows, slots):
    d = make(rows, 24, 40, slots, 4)
    check(d, apply(d))


@pytest.mark.parametrize("rows", [4095, 4096, 4097, 4128, 4129, 8193])
def test_rows_around_a_block(rows):
    d = make(rows, 32, 40, 5, 8)
    check(d, apply(d))


def test_most_rows():
    import torch
    import rwkv_rsv_b200 as rsv
    rows, slots = 1 << 25, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda most, *s: torch.randint(-most, most + 1, s, generator=g, device="cuda")  # noqa: E731
    x, base, A, B = n(9, rows, 1).float(), n(99, rows, 1).float(), n(5, slots, 1, 1).half(), n(5, slots, 1, 1).half()
    index, scales = torch.randint(-1, slots, (rows,), generator=g, device="cuda", dtype=torch.int32), n(3, slots).float()
    out = torch.full((rows, 1), float("nan"), device="cuda")
    rsv.Adapters(A, B, scales=scales).apply(x, index, out, base=base)
    times = torch.cat([(A.float() * B.float())[:, 0, 0] * scales, torch.zeros(1, device="cuda")])  # (-1: the last one)
    assert torch.equal(out, base + x * times[index.long()][:, None])
    with pytest.raises(rsv.RsvError, match="33554432"):
        more = torch.zeros(1, device="cuda")
        rsv.Adapters(A, B).apply(more.expand(rows + 1, 1), torch.zeros(rows + 1, dtype=torch.int32, device="cuda"), torch.zeros(rows + 1, 1, device="cuda"))
