"""Low-rank adapters of many requests (rsv_adapters_apply) against float64.

Most inputs are small whole numbers, whose products and sums stay under 2^24: fp32 holds them exactly in any order, so fp32 outputs have to be equal to the
exact result, and 16-bit outputs to the exact result rounded once.  For other numbers the bound is derived at the test."""
import numpy as np
import pytest

import rwkv_rsv_b200 as rsv

pytestmark = pytest.mark.gpu


def exact(x, index, A, B, ranks, scales, base):
    import torch
    out = base.double().clone() if base is not None else torch.zeros(x.shape[0], B.shape[1], dtype=torch.float64, device=x.device)
    ix = index.tolist()
    for s in range(A.shape[0]):
        rows = [n for n, i in enumerate(ix) if i == s]
        if rows:
            r = A.shape[1] if ranks is None else int(ranks[s])
            t = x[rows].double() @ A[s, :r].double().T
            out[rows] += (1.0 if scales is None else float(scales[s])) * (t @ B[s, :, :r].double().T)
    return out


def whole(g, shape, most, dtype):
    import torch
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def make(rows, K, M, slots, most, x="float32", w="float16", seed=0, ranks=True, scales=True, none=True, pad=(0, 0, 0, 0), order="shuffled"):
    """Whole numbers; what lies behind a slot's rank and between padded rows is NaN."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + rows + 3 * K + 7 * M)
    xt, wt = getattr(torch, x), getattr(torch, w)

    def padded(shape, most_, dtype, extra):
        buf = torch.full((*shape[:-1], shape[-1] + extra), float("nan"), dtype=dtype, device="cuda")
        v = buf[..., :shape[-1]]
        v.copy_(whole(g, shape, most_, dtype))
        return v

    d = {"x": padded((rows, K), 3, xt, pad[0]), "A": padded((slots, most, K), 1, wt, pad[1]), "B": padded((slots, M, most), 2, wt, pad[2]), "base": padded((rows, M), 100, xt, pad[3])}
    d["ranks"] = torch.randint(0, most + 1, (slots,), generator=g, device="cuda", dtype=torch.int32) if ranks else None
    if ranks:
        for s, r in enumerate(d["ranks"].tolist()):
            d["A"][s, r:] = float("nan")
            d["B"][s, :, r:] = float("nan")
    d["scales"] = whole(g, (slots,), 2, torch.float32) if scales else None
    ix = torch.arange(rows, device="cuda") % slots if order != "one" else torch.full((rows,), slots - 1, device="cuda")
    if order == "shuffled":
        ix = ix[torch.randperm(rows, generator=g, device="cuda")]
    elif order == "sorted":
        ix = ix.sort().values
    if none:
        ix = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.2, torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, -1, slots + 5), ix)
    d["index"] = ix.to(torch.int32)
    return d


def apply(d, base=True, out=None):
    import torch
    out = torch.full((d["x"].shape[0], d["B"].shape[1]), float("nan"), dtype=d["x"].dtype, device="cuda") if out is None else out
    rsv.Adapters(d["A"], d["B"], ranks=d["ranks"], scales=d["scales"]).apply(d["x"], d["index"], out, base=d["base"] if base else None)
    return out


def check(d, out, base=True):
    import torch
    want = exact(d["x"], d["index"], d["A"], d["B"], d["ranks"], d["scales"], d["base"] if base else None)
    assert want.abs().max() < 2**24
    want = want.to(out.dtype)
    bad = (out != want).nonzero()
    assert torch.equal(out, want), (bad.shape[0], bad[:4].tolist(), out[tuple(bad[0])], want[tuple(bad[0])])


TYPES = [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("rows,K,M,slots,most", [
    (1, 1, 1, 1, 1), (1, 2560, 2560, 1, 16), (2, 64, 128, 3, 8), (3, 100, 36, 2, 5), (16, 128, 96, 1, 16), (17, 1001, 777, 4, 13), (31, 520, 264, 40, 32), (64, 2560, 512, 64, 16),
    (65, 333, 2049, 3, 64), (200, 512, 2048, 8, 24), (130, 256, 640, 2, 128), (40, 264, 136, 3, 256), (513, 1024, 320, 5, 64), (1000, 128, 64, 300, 4),
])
def test_exact_in_whole_numbers(rows, K, M, slots, most, x, w):
    d = make(rows, K, M, slots, most, x, w)
    check(d, apply(d))


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("pad", [(0, 0, 0, 0), (3, 5, 7, 9), (4, 8, 8, 4)])
@pytest.mark.parametrize("rows,K,M,slots,most", [(2000, 640, 96, 4, 64), (2100, 1000, 52, 3, 48), (1000, 256, 320, 4, 128), (1111, 333, 77, 2, 256), (4200, 128, 64, 5, 64)])
def test_many_rows_of_large_adapters(rows, K, M, slots, most, pad, x, w):
    """Tiles of 32 and 64 rows."""
    d = make(rows, K, M, slots, most, x, w, pad=pad)
    check(d, apply(d))


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("rows,slots", [(1, 1), (7, 1), (8, 1), (9, 1), (16, 2), (17, 2), (33, 4), (40, 40)])
@pytest.mark.parametrize("most", [1, 8, 9, 16, 17, 33, 64, 65, 100])
def test_few_rows_of_an_adapter(rows, slots, most, x, w):
    """Up to eight rows of an adapter are the smaller operand."""
    d = make(rows, 200, 72, slots, most, x, w, ranks=rows != 8, none=False)
    check(d, apply(d))


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("order", ["sorted", "one", "shuffled"])
def test_orders_of_rows(order, x, w):
    d = make(300, 512, 256, 7, 16, x, w, order=order, none=order == "shuffled")
    check(d, apply(d))


@pytest.mark.parametrize("ranks,scales,base", [(False, False, True), (True, False, False), (False, True, False), (True, True, True)])
def test_what_may_be_left_out(ranks, scales, base):
    d = make(50, 200, 120, 6, 20, ranks=ranks, scales=scales)
    check(d, apply(d, base), base)


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("pad", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (2, 4, 2, 6), (8, 8, 8, 8), (3, 5, 7, 9)])
def test_strides(pad, x, w):
    d = make(45, 256, 192, 5, 16, x, w, pad=pad)
    check(d, apply(d))


@pytest.mark.parametrize("x,w", [("float32", "float16"), ("float16", "float16")])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_starts_off_the_wide_loads(shift, x, w):
    import torch
    d = make(33, 256, 192, 5, 16, x, w)
    for k in ("x", "A", "B", "base"):
        buf = torch.zeros(d[k].numel() + 8, dtype=d[k].dtype, device="cuda")
        v = buf[shift:shift + d[k].numel()].view(d[k].shape)
        v.copy_(d[k])
        d[k] = v
    buf = torch.full((33 * 192 + 8,), float("nan"), dtype=d["x"].dtype, device="cuda")
    out = buf[shift:shift + 33 * 192].view(33, 192)
    check(d, apply(d, out=out))
    assert torch.isnan(buf[:shift]).all() and torch.isnan(buf[shift + 33 * 192:]).all()


def test_in_place_and_rows_around_untouched():
    import torch
    d = make(40, 512, 320, 9, 16)
    big = torch.full((44, 330), 7.0, device="cuda")
    out = big[2:42, 5:325]
    out.copy_(d["base"])
    want = exact(d["x"], d["index"], d["A"], d["B"], d["ranks"], d["scales"], d["base"])
    d["base"] = out
    apply(d, out=out)
    assert torch.equal(out.double(), want)
    big[2:42, 5:325] = 7.0
    assert (big == 7.0).all()


def test_shared_row_of_activations_and_base():
    """One vector for all rows (stride 0): each row through its own adapter."""
    import torch
    d = make(24, 256, 128, 24, 8, none=False)
    d["x"], d["base"] = d["x"][:1].expand(24, 256), d["base"][:1].expand(24, 128)
    check(d, apply(d))


def test_a_row_of_nan_stays_in_its_row():
    import torch
    d = make(40, 512, 320, 3, 16)
    want = apply(d)
    bad = 11
    d["index"][bad] = 1
    d["ranks"][1] = 16
    d["A"].nan_to_num_(1.0)
    d["B"].nan_to_num_(1.0)
    want = apply(d)
    d["x"][bad, 100] = float("nan")
    got = apply(d)
    assert torch.isnan(got[bad]).all()
    rest = [n for n in range(40) if n != bad]
    assert torch.equal(got[rest], want[rest])
    d["x"][bad, 100] = float("inf")
    d["A"][1, :, 100] = 1.0
    d["B"][1] = 1.0
    d["scales"][1] = 1.0
    assert (apply(d)[bad] == float("inf")).all()


@pytest.mark.parametrize("x,w", TYPES)
@pytest.mark.parametrize("rows,K,M,slots,most", [(5, 2560, 2560, 3, 16), (300, 10240, 2560, 4, 64), (77, 2500, 999, 9, 200)])
def test_any_numbers(rows, K, M, slots, most, x, w):
    """Values over six orders of magnitude.  fp32 sums: a chain of c additions, each rounded or cut at 2^-23 of the running sum, is off by c 2^-24 of its size on average of the
    two; chains are at most K / 16 long (640) and a running sum of terms of random sign is about 1 / sqrt(K) of the terms' absolute sum (0.01 for 10240), with 3 for its tails:
    640 * 0.03 * 2^-24 < 2^-19 of the absolute sum.  The same for the second product (at most 256 terms), the scale and the addition of base; then half a step of out's type."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(K + rows)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    xt, wt = getattr(torch, x), getattr(torch, w)
    spread = 10.0 ** (torch.rand(rows, K, generator=g, device="cuda") * (6 if x == "float32" else 3) - (3 if x == "float32" else 2))
    d = {"x": (n(rows, K) * spread).to(xt), "A": (n(slots, most, K) / K**0.5).to(wt), "B": (n(slots, M, most) * 0.2).to(wt), "base": n(rows, M).to(xt),
         "ranks": torch.randint(1, most + 1, (slots,), generator=g, device="cuda", dtype=torch.int32), "scales": torch.rand(slots, generator=g, device="cuda") + 0.5,
         "index": torch.randint(-1, slots, (rows,), generator=g, device="cuda", dtype=torch.int32)}
    out = apply(d)
    want = exact(d["x"], d["index"], d["A"], d["B"], d["ranks"], d["scales"], d["base"])
    size = exact(d["x"].abs(), d["index"], d["A"].abs(), d["B"].abs(), d["ranks"], d["scales"], d["base"].abs())
    room = 2.0**-19 * size + torch.finfo(xt).eps / 2 * want.abs() * 1.001
    assert ((out.double() - want).abs() <= room).all(), ((out.double() - want).abs() / room).max()


def test_captured_two_graphs_other_streams():
    import torch
    d, e = make(64, 2560, 1280, 64, 16), make(200, 1024, 2560, 8, 32, seed=1)
    wd, we = apply(d), apply(e)
    ad, ae = (rsv.Adapters(q["A"], q["B"], ranks=q["ranks"], scales=q["scales"]) for q in (d, e))
    od, oe = torch.zeros_like(wd), torch.zeros_like(we)
    torch.cuda.synchronize()
    g1, g2, s1, s2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.graph(g1):
        ad.apply(d["x"], d["index"], od, base=d["base"])
    with torch.cuda.graph(g2):
        ae.apply(e["x"], e["index"], oe, base=e["base"])
    for _ in range(3):
        od.zero_(), oe.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        ad.apply(d["x"], d["index"], od, base=d["base"], stream=s2)
        torch.cuda.synchronize()
        assert torch.equal(od, wd) and torch.equal(oe, we)
    # a replay reads indices and adapters anew
    d["index"].copy_(d["index"].flip(0))
    d["scales"].mul_(2)
    g1.replay()
    torch.cuda.synchronize()
    check(d, od)


def test_python_refusals():
    import torch
    d = make(6, 64, 32, 3, 8, none=False)
    for A, B, kw in ((d["A"][0], d["B"], {}), (d["A"].float(), d["B"].float(), {}), (d["A"], d["B"].bfloat16(), {}), (d["A"], d["B"][:2], {}), (d["A"], d["B"].transpose(1, 2), {}),
                     (d["A"][:, :, ::2], d["B"], {}), (d["A"], d["B"], dict(ranks=d["ranks"].long())), (d["A"], d["B"], dict(scales=d["scales"][:2]))):
        with pytest.raises(rsv.RsvError):
            rsv.Adapters(A, B, **kw)
    ad, out = rsv.Adapters(d["A"], d["B"]), torch.zeros(6, 32, device="cuda")
    for bad in (dict(x=d["x"][:, :60]), dict(x=d["x"].double()), dict(x=d["x"].bfloat16()), dict(x=d["x"].t()), dict(index=d["index"].long()), dict(index=d["index"][:5]), dict(out=out.half()),
                dict(out=out[:5]), dict(base=out.half()), dict(base=torch.zeros(5, 32, device="cuda")), dict(out=out.cpu()), dict(out=out[:1].expand(6, 32))):
        a = dict(x=d["x"], index=d["index"], out=out, base=None) | bad
        with pytest.raises(rsv.RsvError):
            ad.apply(a["x"], a["index"], a["out"], base=a["base"])
