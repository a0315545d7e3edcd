"""Tokens drawn from given random numbers (rsv_draw_tokens) against the definition in 64 bits, token for token: sums of the operator are exact, so a token can
differ from the 64-bit one only where u lies within about 1e-12 of a border between two tokens, which no seed here comes near.

Log-probabilities are computed in fp64 from weights of F >= 40 bits after the point (each off by half a unit, all V <= 2^17 of them by 2^-30 of the largest at most,
where F = 45) and rounded to fp32 once: |error| <= 2^-24 |value| + 2^-29."""
import ctypes
import math

import numpy as np
import pytest

import rwkv_rsv_b200 as rsv

pytestmark = pytest.mark.gpu


def reference(l, T, k, p, m, u):
    """(token, log-probability) of one row, in float64."""
    l = np.asarray(l, np.float64) + 0.0
    V = l.size
    if np.isnan(l).any():
        return -1, math.nan
    mx = l.max()
    if mx == -math.inf:
        return -1, -math.inf
    if not T > 0:
        return int(np.argmax(l)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(l == mx, 0.0, (l - mx) / np.float64(np.float32(T)))
    fall = np.argsort(-l, kind="stable")
    if 0 < k < V:
        fall = fall[:k]
    w = np.where(z[fall] >= -40 * math.log(2), np.exp(z[fall]), 0.0)
    keep = w > 0
    p, m = float(np.float32(p)), float(np.float32(m))
    if 0 < p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep &= before < p * w.sum()
    if m > 0:
        keep &= w >= min(m, 1.0)
    at = np.sort(fall[keep])
    w = np.exp(z[at])
    u = float(np.float32(u))
    u = 0.0 if not u > 0 else u
    hit = min(int((np.cumsum(w) <= u * w.sum()).sum()), at.size - 1)
    return int(at[hit]), float(z[at[hit]] - math.log(w.sum()))


def check(logits, params, u, token, logprob=None):
    lg, u = logits.float().cpu().numpy(), u.cpu().numpy()
    par, got = params.cpu().numpy(), token.cpu().numpy()
    lp = None if logprob is None else logprob.cpu().numpy()
    for r in range(lg.shape[0]):
        want, wlp = reference(lg[r], par[r, 0], int(par.view(np.uint32)[r, 1]), par[r, 2], par[r, 3], u[r])
        assert got[r] == want, (r, par[r], u[r], got[r], want)
        if lp is not None:
            assert (math.isnan(wlp) and math.isnan(lp[r])) or lp[r] == wlp or abs(lp[r] - wlp) <= 2.0**-24 * abs(wlp) + 2.0**-29, (r, par[r], lp[r], wlp)


def run(logits, params, u, stream=None):
    import torch
    R = logits.shape[0]
    token, logprob = torch.full((R,), -7, dtype=torch.int32, device="cuda"), torch.full((R,), 7.0, device="cuda")
    rsv.draw_tokens(logits, params, u, token, logprob, stream=stream)
    return token, logprob


def every_setting(V):
    """Temperature, top-k, top-p and min-p in combinations, one row each."""
    rows = [(T, k, p, m) for T in (0.0, 0.3, 1.0, 2.5) for k in (0, 1, 7, 50, 300, 900, 5000) for p, m in ((1.0, 0.0), (0.9, 0.0), (0.3, 0.0), (1.0, 0.1), (0.95, 0.02), (0.999, 0.0))]
    rows += [(1e-30, 0, 1.0, 0.0), (1e30, 0, 0.5, 0.0), (float("inf"), 3, 1.0, 0.0), (1.0, V, 1.0, 0.0), (1.0, V - 1, 0.999999, 0.0), (1.0, 0, 1e-9, 0.0), (1.0, 0, 0.0, 1.0), (1.0, 0, 1.5, 2.0),
             (-1.0, 5, 0.5, 0.5), (float("nan"), 0, 1.0, 0.0), (1.0, 0, float("nan"), float("nan")), (1.0, 2**32 - 1, -1.0, -1.0)]
    return rows


def inputs(V, dtype, kind, seed, offset=0, stride=None, rows=None):
    import torch
    rows = rows or every_setting(V)
    R = len(rows)
    g = np.random.default_rng(seed)
    if kind == "peaked":
        l = g.standard_normal((R, V)) * 2.5
        l[np.arange(R)[:, None], g.integers(0, V, (R, 6))] += g.random((R, 6)) * np.linspace(0, 14, R)[:, None]
    elif kind == "equal":
        l = np.zeros((R, V)) - 3.25
    elif kind == "steps":  # few different values, so that every cut falls among equal ones
        l = g.integers(-3, 4, (R, V)) * 0.5
    elif kind == "wide":
        l = g.standard_normal((R, V)) * 30
    elif kind == "flat":
        l = g.standard_normal((R, V)) * 0.3
    elif kind == "low":  # a few large logits in front of a flat rest
        l = g.standard_normal((R, V)) * 0.5
        l[np.arange(R)[:, None], g.integers(0, V, (R, 20))] += g.random((R, 20)) * 10
    elif kind == "fine":  # steps of 1/1000, two next to each other with most of the logits
        l = np.where(g.random((R, V)) < 0.8, 1.0 + 1e-3 * g.integers(0, 2, (R, V)), np.round(g.standard_normal((R, V)), 3))
    elif kind == "masked":
        l = np.where(g.random((R, V)) < 0.97, -np.inf, g.standard_normal((R, V)) * 3)
        l[:, g.integers(0, V)] = 1.0
    stride = stride or V
    buf = torch.full((R * stride + offset + 64,), float("nan"), dtype=dtype, device="cuda")
    view = buf[offset:offset + R * stride].view(R, stride)[:, :V]
    view.copy_(torch.from_numpy(l).to(dtype))
    T, k, p, m = zip(*rows)
    return view, torch.from_numpy(rsv.draw_params(T, k, p, m)).cuda(), torch.from_numpy(g.random(R).astype(np.float32)).cuda()


@pytest.mark.parametrize("kind", ["peaked", "equal", "steps", "wide", "masked"])
@pytest.mark.parametrize("V", [1, 2, 31, 257, 1000, 4096, 4099, 50003, 65536])
def test_every_setting(V, kind):
    import torch
    l, par, u = inputs(V, torch.float32, kind, V)
    check(l, par, u, *run(l, par, u))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("V,kind", [(1, "peaked"), (1001, "steps"), (4096, "peaked"), (50003, "peaked"), (65536, "peaked"), (131072, "peaked")])
def test_sixteen_bits(V, kind, dtype):
    import torch
    l, par, u = inputs(V, getattr(torch, dtype), kind, V + 1)
    check(l, par, u, *run(l, par, u))


@pytest.mark.parametrize("V", [100000, 131072, 200001, 1 << 20])
def test_large_vocabularies(V):
    import torch
    l, par, u = inputs(V, torch.float32, "peaked", V, rows=[(1.0, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 0, 1.0, 0.0), (1.0, 2000, 0.99, 0.01), (0.0, 0, 1.0, 0.0), (1.5, 0, 1.0, 0.05)])
    check(l, par, u, *run(l, par, u))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V,kind", [(8192, "flat"), (32000, "low"), (50003, "flat"), (65536, "low"), (65536, "fine"), (131072, "flat"), (131072, "low"), (300001, "flat"), (65536, "steps")])
def test_cuts_among_many_close_logits(V, kind, dtype):
    """Thousands of logits so near the cut, or equal to it, that no collection around it is small."""
    import torch
    rows = [(T, k, p, m) for T in (1.0, 0.7, 2.0) for k, p, m in ((0, 0.5, 0.0), (0, 0.9, 0.0), (0, 0.99, 0.0), (700, 1.0, 0.0), (1000, 0.9, 0.0), (3000, 0.95, 0.0), (0, 0.9, 0.3), (3000, 0.99, 0.7),
                                                                      (3000, 1.0, 0.5), (4000, 1.0, 0.9))]
    l, par, u = inputs(V, getattr(torch, dtype), kind, V + 3, rows=rows)
    check(l, par, u, *run(l, par, u))


@pytest.mark.parametrize("rows", [1, 2, 5, 40, 150, 700])
def test_numbers_of_rows(rows):
    """The same rows alone and among others give the same tokens."""
    import torch
    settings = (every_setting(65536) * 5)[:rows]
    l, par, u = inputs(65536, torch.float32, "peaked", rows, rows=settings)
    token, lp = run(l, par, u)
    check(l[:150], par[:150], u[:150], token[:150], lp[:150])
    for r in range(0, rows, max(1, rows // 7)):
        one, olp = run(l[r:r + 1], par[r:r + 1], u[r:r + 1])
        assert int(one) == int(token[r]) and (float(olp) == float(lp[r]))


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("offset,stride", [(0, 4100), (1, 4096), (2, 4097), (3, 4099), (5, 4111), (8, 5000)])
def test_any_start_and_stride(offset, stride, dtype):
    """(What lies between the rows is NaN.)"""
    import torch
    l, par, u = inputs(4096 if stride < 4100 else 4095, getattr(torch, dtype), "peaked", stride, offset, stride if stride >= 4096 else None)
    check(l, par, u, *run(l, par, u))


def test_same_row_for_all():
    """Rows that lie on each other (stride 0): many draws from one distribution follow it."""
    import torch
    R, V = 4096, 12
    l = torch.linspace(-2, 2, V, device="cuda")[None, :].expand(R, V)
    par = torch.from_numpy(rsv.draw_params(np.ones(R))).cuda()
    u = (torch.arange(R, device="cuda") + 0.5) / R
    token, _ = run(l, par, u)
    share = np.exp(np.linspace(-2, 2, V))
    share /= share.sum()
    counts = np.bincount(token.cpu().numpy(), minlength=V)
    assert np.abs(counts - share * R).max() <= 1.0  # evenly spaced u: every token's stretch holds its share, up to one at the ends together


def test_rows_without_a_token_and_odd_numbers():
    import torch
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    V = 5000
    l = torch.full((16, V), -1.0, device="cuda")
    l[0] = -inf
    l[1] = nan
    l[2, 77] = nan
    l[3] = -inf
    l[3, 4999] = -4.0
    l[4] = low
    l[5] = low
    l[5, 9] = 0.0
    l[6, [10, 4000]] = inf
    l[7] = inf
    l[8, 1] = torch.finfo(torch.float32).max
    l[9] = 0.0
    l[9, ::2] = -0.0
    u = torch.tensor([0.5, 0.5, 0.5, 0.9, 0.7, 0.9, 0.6, 0.3, 0.2, 0.5, 0.0, 1.0, 5.0, nan, -1.0, 1 - 2.0**-24], device="cuda")
    for row in ((1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 0, 0.8, 0.0), (1.0, 1500, 1.0, 0.3)):
        par = torch.from_numpy(rsv.draw_params(*([v] * 16 for v in row))).cuda()
        check(l, par, u, *run(l, par, u))


def test_borders_of_top_p_and_u():
    """Four equal tokens: half of them is two, and u picks by quarters."""
    import torch
    l = torch.full((8, 8), -30.0, device="cuda")
    l[:, 2:6] = 1.0
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.0, 0.5, 0.49999997, 0.99999994], device="cuda")
    par = torch.from_numpy(rsv.draw_params(1.0, 4, [1, 1, 1, 1, 0.5, 0.5, 0.5, 0.5000001], 0.0)).cuda()
    token, lp = run(l, par, u)
    assert token.tolist() == [2, 3, 4, 5, 2, 3, 2, 4]
    assert np.allclose(lp.cpu().numpy(), -np.log([4, 4, 4, 4, 2, 2, 2, 3]), rtol=2.0**-23, atol=0)


def test_captured_on_another_stream_and_two_at_once():
    import torch
    settings = every_setting(65536)[:64]
    l, par, u = inputs(65536, torch.float32, "peaked", 3, rows=settings)
    l2, par2, u2 = inputs(50003, torch.float32, "steps", 4, rows=settings)
    want, want2 = run(l, par, u), run(l2, par2, u2)
    token, lp = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    token2, lp2 = torch.zeros_like(want2[0]), torch.zeros_like(want2[1])
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rsv.draw_tokens(l, par, u, token, lp)
    for _ in range(3):
        token.zero_()
        torch.cuda.synchronize()
        g.replay()
        rsv.draw_tokens(l2, par2, u2, token2, lp2, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(token, want[0]) and torch.equal(token2, want2[0]) and torch.equal(lp2, want2[1])
    u.copy_(u.flip(0))
    g.replay()
    again = run(l, par, u)
    torch.cuda.synchronize()
    assert torch.equal(token, again[0]) and torch.equal(lp, again[1])


def test_without_logprobs_unsigned_tokens_and_neighbours_untouched():
    import torch
    l, par, u = inputs(4096, torch.float32, "peaked", 5, rows=every_setting(4096)[:10])
    want, _ = run(l, par, u)
    out = torch.full((14,), 123, dtype=torch.int32, device="cuda")
    rsv.draw_tokens(l, par, u, out[2:12])
    assert torch.equal(out[2:12], want) and out[[0, 1, 12, 13]].tolist() == [123] * 4
    un = torch.zeros(10, dtype=torch.uint32, device="cuda")
    rsv.draw_tokens(l, par, u, un)
    assert torch.equal(un.view(torch.int32), want)
    rsv.draw_tokens(l[:0], par[:0], u[:0], out[:0])


def test_python_refusals():
    import torch
    l, par, u = inputs(64, torch.float32, "peaked", 5, rows=every_setting(64)[:4])
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (dict(l=l.double()), dict(l=l.t()), dict(l=l[:, ::2]), dict(par=par[:3]), dict(par=par.double()), dict(u=u[:3]), dict(u=u.double()), dict(tok=tok.long()), dict(tok=tok.cpu()),
                dict(tok=tok[::2]), dict(lp=torch.zeros(3, device="cuda"))):
        a = dict(l=l, par=par, u=u, tok=tok, lp=None) | bad
        with pytest.raises(rsv.RsvError):
            rsv.draw_tokens(a["l"], a["par"], a["u"], a["tok"], a["lp"])
    with pytest.raises(rsv.RsvError):
        rsv._check(rsv.native().rsv_draw_tokens(99, None, 0, l.data_ptr(), 4, 64, 64, par.data_ptr(), u.data_ptr(), tok.data_ptr(), ctypes.c_void_p()))
    assert torch.cuda.current_device() == 0
