"""Low-rank adapters whose ranks, activations or products lie far apart (rsv_adapters_apply) against float64.

The bound, by component, with size = |base| + scale |B| (|A| |x|): fp32 activations are two tf32 numbers, at most 2^-22 of a value off; the first product adds up to 160 sums of
16 products, each rounded at 2^-24 of the running sum, with random signs 2^-20 together; a value of A x is kept to 2^-20 of itself or its largest part for fp32 outputs and 2^-17 for 16-bit ones;
up to 200 products of these are summed in steps of 8 or 16 ranks, under 2^-20 likewise; the scale and base round twice, 2^-23.  Together under 2^-18 of size for fp32 outputs, and
for 16-bit ones under 2^-16 and half a step of the type."""
import math

import pytest

from test_gpu_adapters import apply, exact

pytestmark = pytest.mark.gpu

TYPES = [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


def apart(rows, K, M, most, x, w, up, down, inverse, slots=2, seed=0):
    """Half of the ranks with rows of A `up` times as large, the other half with rows `down` times; B has one half of the outputs for each (block diagonal), or (inverse) all of
    them, with columns that undo it."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + rows + K)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    h = most // 2
    A, B = n(slots, most, K) / math.sqrt(K), n(slots, M, most) * 0.2
    A[:, :h] *= up
    A[:, h:] *= down
    if inverse:
        B[:, :, h:] *= up / down
    else:
        B[:, : M // 2, h:] = 0
        B[:, M // 2:, :h] = 0
    return {"x": n(rows, K).to(getattr(torch, x)), "A": A.to(getattr(torch, w)), "B": B.to(getattr(torch, w)), "base": torch.zeros(rows, M, dtype=getattr(torch, x), device="cuda"),
            "ranks": None, "scales": torch.rand(slots, generator=g, device="cuda") + 0.5, "index": torch.arange(rows, device="cuda", dtype=torch.int32) % slots}


def check(d, least=0.0):
    """(least: what smaller weights of B but 0 count as in `size`.)"""
    import torch
    out = apply(d)
    want = exact(d["x"], d["index"], d["A"], d["B"], d["ranks"], d["scales"], d["base"])
    size = exact(d["x"].abs(), d["index"], d["A"].abs(), torch.where(d["B"] == 0, 0.0, d["B"].double().abs().clamp(min=least)), d["ranks"], d["scales"], d["base"].abs())
    xt = d["x"].dtype
    room = 2.0**-18 * size if xt == torch.float32 else 2.0**-16 * size + torch.finfo(xt).eps / 2 * want.abs() * 1.001
    room += torch.finfo(xt).smallest_normal * torch.finfo(xt).eps  # (16-bit outputs under the smallest normal one)
    worst = ((out.double() - want).abs() / room).max()
    assert torch.isfinite(want).all() and worst <= 1, float(worst)


SPREADS = [(1.0, 2.0**-6), (1.0, 2.0**-10), (8.0, 2.0**-10), (2.0**10, 2.0**-10), (2.0**13, 2.0**-11)]


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("up,down", SPREADS)
@pytest.mark.parametrize("rows,K,M,most", [(1, 64, 64, 8), (5, 2560, 640, 16), (40, 200, 99, 64), (300, 128, 96, 32), (2000, 256, 64, 64), (64, 64, 512, 200)])
def test_ranks_of_different_size_for_different_outputs(rows, K, M, most, up, down, x, w):
    if x == "float16" and up > 2.0**8:
        up, down = up / 2.0**8, down  # (outputs stay in range)
    check(apart(rows, K, M, most, x, w, up, down, False))


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("apart_by", [2.0**6, 2.0**10, 2.0**13])
@pytest.mark.parametrize("rows,K,M,most", [(3, 2560, 256, 16), (33, 256, 300, 64), (1200, 128, 64, 64)])
def test_small_rows_of_a_with_large_columns_of_b(rows, K, M, most, apart_by, x, w):
    check(apart(rows, K, M, most, x, w, 1.0, 1.0 / apart_by, True))


@pytest.mark.parametrize("w", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 9, 64])
def test_one_row_with_values_far_apart_among_others(rows, w):
    """Only one row of the tile has them: activations that a single rank picks, 2^40 apart."""
    import torch
    d = apart(rows, 64, 64, 16, "float32", w, 1.0, 1.0, False, slots=1)
    d["A"][0] = 0
    d["A"][0, torch.arange(16), torch.arange(16)] = 1.0
    d["x"][rows // 2, :8] *= 2.0**20
    d["x"][rows // 2, 8:16] *= 2.0**-20
    check(d)


@pytest.mark.parametrize("w", ["float16", "bfloat16"])
@pytest.mark.parametrize("size", [1e-25, 1e-12, 1e12, 1e25, 1e33])
def test_small_and_large_activations(size, w):
    d = apart(20, 128, 96, 16, "float32", w, 1.0, 2.0**-10, False)
    d["x"] *= size
    check(d)


@pytest.mark.parametrize("w", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 20])
def test_activations_next_to_the_largest_float(rows, w):
    """Values that round to infinity in fewer bits: A x of 3.4e38 2^-10 and, with A = 1, of 3.4e38 itself."""
    import torch
    top = torch.finfo(torch.float32).max
    d = apart(rows, 64, 64, 8, "float32", w, 1.0, 1.0, False, slots=1)
    for a, b in ((2.0**-10, 1.0), (1.0, 2.0**-10)):
        d["x"][:] = 0
        d["x"][:, 3] = top
        d["x"][rows // 2, 3] = -top
        d["A"].fill_(a)
        d["B"].zero_()
        d["B"][:, :, 0] = b
        check(d)


@pytest.mark.parametrize("w", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 20])
def test_an_infinite_rank_leaves_finite_ones_finite(rows, w):
    """A x of +inf (an overflow) in one rank and of about -3e35 in another: their sum is +inf, not inf - inf."""
    import torch
    d = apart(rows, 64, 64, 8, "float32", w, 1.0, 1.0, False, slots=1)
    d["x"][:] = 0
    d["x"][:, 5] = 3e38
    d["A"].zero_()
    d["A"][:, 0, 5] = 100.0
    d["A"][:, 1, 5] = -(2.0**-10)
    d["B"].zero_()
    d["B"][:, :, :2] = 1.0
    assert (apply(d) == float("inf")).all()


@pytest.mark.parametrize("x,w", TYPES)
def test_infinities_and_nan_as_in_a_sum_of_products(x, w):
    """Infinite and NaN activations come out as the sum of products has them, and only in their rows."""
    import torch
    inf, nan = float("inf"), float("nan")
    d = apart(20, 64, 64, 8, x, w, 1.0, 1.0, False, slots=1)
    want = apply(d)
    d["A"].abs_().clamp_(min=0.01)
    d["B"].fill_(0.5)
    want = apply(d)
    for row, v in ((2, inf), (3, -inf), (4, nan), (11, inf)):
        d["x"][row, 7] = v
    bits = torch.tensor([0x7F800001], dtype=torch.int32, device="cuda").view(torch.float32)  # a NaN whose low bits alone tell it from infinity
    if x == "float32":
        d["x"][5, 9] = bits[0]
    got = apply(d)
    assert (got[2] == inf).all() and (got[3] == -inf).all() and torch.isnan(got[4]).all() and (got[11] == inf).all()
    bad = [2, 3, 4, 11]
    if x == "float32":
        assert torch.isnan(got[5]).all()
        bad.append(5)
    rest = [n for n in range(20) if n not in bad]
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("size", [2.0**-15, 2.0**-18, 2.0**-22])
@pytest.mark.parametrize("rows,K,M,most", [(1, 2, 40, 2), (40, 64, 72, 16), (900, 64, 64, 64)])
def test_weights_under_the_smallest_normal_fp16(rows, K, M, most, size, x, w):
    """B of 2^-15 and less, down to 2^-24, next to ranks of other sizes: as exact as with weights of 2^-14, which is 2^-18 (2^-16) of 2^-14 |A| |x|."""
    d = apart(rows, K, M, most, x, w, 1.0, 2.0**-8, True)
    d["B"] = (d["B"].double() * size * 5).clamp(-4 * size, 4 * size).to(d["B"].dtype)
    check(d, 2.0**-14 if w == "float16" else 0.0)
