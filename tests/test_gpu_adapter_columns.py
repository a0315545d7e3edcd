"""Activations, base and output as columns of one array (rsv_adapters_apply): neighbours in memory that share no element."""
import numpy as np
import pytest

import rwkv_rsv_b200 as rsv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x,w", [("float32", "float16"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("rows,K,M,gap", [(1, 64, 32, 0), (6, 64, 32, 0), (70, 200, 77, 3), (300, 128, 256, 8)])
def test_columns_of_one_array(rows, K, M, gap, x, w):
    import torch
    from test_gpu_adapters import apply, check, make
    d = make(rows, K, M, 3, 8, x, w)
    width = K + 2 * M + 3 * gap
    big = torch.full((rows, width), 7.0, dtype=d["x"].dtype, device="cuda")
    out, xs, base = big[:, gap:gap + M], big[:, gap + M + gap:gap + M + gap + K], big[:, width - M:]
    xs.copy_(d["x"])
    base.copy_(d["base"])
    d["x"], d["base"] = xs, base
    want = big.clone()
    check(d, apply(d, out=out))
    want[:, gap:gap + M] = out
    assert torch.equal(big, want)
    # in place, beside the activations
    out.copy_(base)
    d["base"] = out
    from test_gpu_adapters import exact
    whole = exact(d["x"], d["index"], d["A"], d["B"], d["ranks"], d["scales"], d["base"]).to(out.dtype)
    apply(d, out=out)
    assert torch.equal(out, whole)


def test_columns_that_meet_are_refused():
    import torch
    big, ix = torch.zeros(6, 128, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    ad = rsv.Adapters(torch.zeros(1, 4, 64, device="cuda").half(), torch.zeros(1, 32, 4, device="cuda").half())
    for x, out, base in ((big[:, 31:95], big[:, :32], None), (big[:, 64:], big[:, 40:72], None), (big[:, 64:], big[:, :32], big[:, 31:63]), (big[:3, 64:], big[:3, :32], big[1:4, :32])):
        with pytest.raises(rsv.RsvError, match="overlap"):
            ad.apply(x, ix[:x.shape[0]], out, base=base)
