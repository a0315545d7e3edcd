"""What the operators on device memory refuse, before any GPU is asked: the C entry points with made-up pointers, and the Python layer with CPU tensors."""
import ctypes

import numpy as np
import pytest

import rwkv_rsv_b200 as rsv

P = 1 << 20  # an address that is never read


def draw(dtype=0, logits=P, rows=2, V=16, stride=16, params=P, u=P, tokens=P, logprobs=None, device=0):
    rc = rsv.native().rsv_draw_tokens(device, None, dtype, logits, rows, V, stride, params, u, tokens, logprobs)
    return rc, rsv.native().rsv_last_error().decode() if rc else ""


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(V=0), "V must be"), (dict(V=(1 << 22) + 1), "V must be"), (dict(rows=-1), "negative number"),
    (dict(rows=1 << 31), "too many rows"), (dict(stride=-1), "negative row stride"), (dict(logits=None), "null"), (dict(params=None), "null"), (dict(u=None), "null"),
    (dict(tokens=None), "null"), (dict(logits=P + 2), "aligned"), (dict(dtype=1, logits=P + 1), "aligned"), (dict(u=P + 2), "aligned"), (dict(logprobs=P + 1), "aligned"),
])
def test_draw_tokens_refuses(kw, says):
    rc, err = draw(**kw)
    assert rc != 0 and says in err and err.startswith("draw_tokens"), (rc, err)


def adapters(dtype=1, slots=2, max_rank=8, K=64, M=32, a=P, b=P, xtype=0, x=1 << 30, ldx=64, rows=2, index=P, base=None, ldb=32, out=1 << 28, ldo=32, a_row=64, **more):
    c = rsv._AdaptersC(dtype, slots, max_rank, K, M, a, more.get("a_slot", 512), a_row, b, more.get("b_slot", 256), more.get("b_row", 8), more.get("ranks"), more.get("scales"))
    rc = rsv.native().rsv_adapters_apply(0, None, ctypes.byref(c), xtype, x, ldx, rows, index, base, ldb, out, ldo)
    return rc, rsv.native().rsv_last_error().decode() if rc else ""


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=0), "adapters' dtype"), (dict(dtype=3), "adapters' dtype"), (dict(xtype=2), "activations"), (dict(dtype=2, xtype=1), "activations"), (dict(K=0), "K and M"),
    (dict(M=0), "K and M"), (dict(slots=0), "K and M"), (dict(slots=4097), "K and M"), (dict(max_rank=0), "max_rank"), (dict(max_rank=257), "max_rank"),
    (dict(rows=-1), "rows"), (dict(rows=(1 << 25) + 1), "rows"), (dict(ldx=-1), "negative stride"), (dict(a_row=-1), "negative stride"), (dict(b_slot=-1), "negative stride"),
    (dict(ldo=31), "overlap"), (dict(a=None), "null"), (dict(b=None), "null"), (dict(x=None), "null"), (dict(index=None), "null"), (dict(out=None), "null"),
    (dict(x=(1 << 30) + 2), "aligned"), (dict(a=P + 1), "aligned"), (dict(index=P + 2), "aligned"), (dict(scales=P + 2), "aligned"), (dict(out=1 << 30), "out and x overlap"),
    (dict(base=(1 << 28) + 4), "out and base overlap"), (dict(base=1 << 28, ldb=33), "out and base overlap"),
])
def test_adapters_refuse(kw, says):
    rc, err = adapters(**kw)
    assert rc != 0 and says in err and err.startswith("adapters"), (rc, err)


def test_no_rows_is_no_work_and_no_gpu_is_an_error():
    import torch
    assert draw(rows=0, logits=None)[0] == 0 and adapters(rows=0, x=None)[0] == 0
    if not torch.cuda.is_available():
        assert "no CUDA device" in draw()[1] and "no CUDA device" in adapters()[1]


def test_python_layer_refuses_tensors_of_the_host():
    import torch
    z = torch.zeros
    with pytest.raises(rsv.RsvError, match="CUDA tensor"):
        rsv.draw_tokens(z(2, 8), z(2, 4), z(2), z(2, dtype=torch.int32))
    with pytest.raises(rsv.RsvError, match="CUDA tensors"):
        rsv.Adapters(z(2, 4, 8, dtype=torch.float16), z(2, 8, 4, dtype=torch.float16))


def test_draw_params_rows():
    p = rsv.draw_params([0.5, 1.0], top_k=50, top_p=0.9, min_p=[0.0, 0.1])
    assert p.shape == (2, 4) and p.dtype == np.float32
    assert np.array_equal(p.view(np.uint32)[:, 1], [50, 50]) and np.array_equal(p[:, 3], np.float32([0, 0.1])) and np.array_equal(p[:, 0], np.float32([0.5, 1]))
    with pytest.raises(rsv.RsvError, match="top_k"):
        rsv.draw_params(top_k=-1)


def test_model_entry_points_refuse_null():
    L = rsv.native()
    for rc in (L.rsv_model_adapters_new(None, 1, 1), L.rsv_model_adapter_set(None, 0, 0, 0, 0, None, None, 1.0), L.rsv_state_set_adapter(None, 0, -1),
               L.rsv_sched_submit_adapter(None, None, 0, 1, None, -1, None), L.rsv_infer_draw(None, None, None, 0, None, 0.5, None, None)):
        assert rc != 0 and L.rsv_last_error().decode() == "null argument"
