"""Adapters of sessions inside the model, and tokens drawn behind it.

A checkpoint whose att.output and ffn.value lack some of their input columns, with an adapter that brings them back (A picks the columns, B holds them), is the whole
checkpoint: the same products, summed in another order.  That fixes what every path has to give without a second implementation."""
import os

import numpy as np
import pytest

import rwkv_rsv_b200 as rsv
from test_gpu_draw import reference

pytestmark = pytest.mark.gpu

RANK, LAYERS, C, F, V = 12, 4, 512, 2048, 4096
SITES = {"att.output": C, "ffn.value": F}


@pytest.fixture(scope="module")
def models(model_dir):
    """(whole, without the columns of set 0, without those of set 1) as checkpoints, and the adapters that undo it."""
    from safetensors.numpy import load_file, save_file
    whole = rsv.write_synthetic(os.path.join(model_dir, "whole.st"), "tiny", seed=3, quant=0)
    w = load_file(whole)
    g = np.random.default_rng(5)
    paths, adapters = [], []
    cols = {(s, l): g.permutation(K)[:2 * RANK].reshape(2, RANK) for s, K in SITES.items() for l in range(LAYERS)}
    for n in range(2):
        out, ad = dict(w), {}
        for l in range(LAYERS):
            for site, K in SITES.items():
                key, c = f"blocks.{l}.{site}.weight", cols[site, l][n]
                m = w[key].copy()
                A = np.zeros((RANK, K), np.float16)
                A[np.arange(RANK), c] = 2.0
                ad[site, l] = (A, m[:, c].copy())
                m[:, c] = 0
                out[key] = m
        paths.append(os.path.join(model_dir, f"part{n}.st"))
        save_file(out, paths[-1])
        adapters.append(ad)
    return whole, paths, adapters


def load(path, adapters=(), slots=3):
    b = rsv.ModelBuilder(path).build()
    if adapters:
        b.model.adapters_new(slots, 16)
        for slot, ad in adapters:
            for (site, l), (A, B) in ad.items():
                b.model.adapter_set(slot, l, site, A, B, scale=0.5)
    return b


PROMPT = np.random.default_rng(1).integers(0, V, 150).astype(np.uint32)


def near(a, b, tol=2e-5):
    """Both sides round activations to 2^-22 (two halves, or two tf32 numbers) and sum in fp32: a projection differs by about 2^-22 of the sum of its absolute products,
    which for 2048 terms of random sign is ten times what is left of it.  Eight projections, logits of about 1: 8 * 10 * 2^-22 = 2e-5."""
    return float(np.sqrt(np.mean((np.asarray(a) - np.asarray(b)) ** 2))) <= tol


def test_adapter_restores_the_whole_model(models):
    whole, paths, ads = models
    a, b = load(whole), load(paths[0], [(1, ads[0])])
    want = a.infer_seq(PROMPT)
    missing = b.infer_seq(PROMPT)
    assert not near(missing, want, 1e-3)
    b.reset()
    b.state.set_adapter(0, 1)
    assert near(b.infer_seq(PROMPT), want)
    assert np.abs(b.state_back() - a.state_back()).max() <= 1e-4  # (as against the oracle)
    for t in (7, 8, 9):  # token by token, behind the prompt
        assert near(b.infer_tokens([t]), a.infer_tokens([t]))
    assert near(b.infer(rsv.RnnInput(PROMPT[:40], 16, rsv.RnnOption.Full)), a.infer(rsv.RnnInput(PROMPT[:40], 16, rsv.RnnOption.Full)))
    assert list(b.infer_argmax_selfloop(5, 24)) == list(a.infer_argmax_selfloop(5, 24))
    sp = rsv.SamplerParams(temperature=0.8, top_k=40, top_p=0.9)
    assert list(b.infer_sample_selfloop(5, 24, sp)) == list(a.infer_sample_selfloop(5, 24, sp))
    # without the adapter again: as before, bit for bit
    b.state.set_adapter(0, -1)
    b.reset()
    assert np.array_equal(b.infer_seq(PROMPT), missing)


def test_sessions_with_different_adapters_share_steps(models):
    whole, paths, ads = models
    one = load(whole)
    b = load(paths[0], [(0, {k: (v[0], v[1] * 2) for k, v in ads[0].items()}), (2, ads[0])])
    prompts = [PROMPT[:n] for n in (31, 1, 64, 17, 50)]
    use = [2, -1, 2, 0, 2]
    st = b.model.create_batch_state(5)
    for s, a in enumerate(use):
        st.set_adapter(s, a)
    seeds = b.model.forward_seq_batch(st, prompts)
    got = b.model.collect_sample_selfloop_batch(b.model.submit_sample_selfloop_batch(st, seeds, 12, None))
    for s, a in enumerate(use):
        single = rsv.Bundle(b.model)
        single.state.set_adapter(0, a)
        single.infer_seq(prompts[s])
        assert list(single.infer_argmax_selfloop(int(seeds[s]), 12)) == list(got[s]), s
        if a == 2:
            one.reset()
            one.infer_seq(prompts[s])
            assert list(one.infer_argmax_selfloop(int(seeds[s]), 12)) == list(got[s]), s


def test_scheduler_sessions_with_adapters(models):
    whole, paths, ads = models
    one, b = load(whole), load(paths[1], [(1, ads[1])])
    plain = load(paths[1])
    sc = rsv.Scheduler(b.model, max_slots=3, chunk=32, max_rows=40)
    g = np.random.default_rng(9)
    jobs = [(PROMPT[:int(n)], int(k), a) for n, k, a in zip(g.integers(3, 90, 8), g.integers(1, 16, 8), [1, None, 1, 1, None, 1, None, 1])]
    ids = [sc.submit(p, k, adapter=a) for p, k, a in jobs]
    done = sc.run_until_done()
    for rid, (p, k, a) in zip(ids, jobs):
        m = one if a == 1 else plain
        m.reset()
        tok = int(np.argmax(m.infer_seq(p)))
        want = [tok] + (list(m.infer_argmax_selfloop(tok, k - 1)) if k > 1 else [])
        assert list(done[rid]) == want, (rid, a)


def test_changed_and_removed_adapters(models):
    whole, paths, ads = models
    b = load(paths[0], [(0, ads[0])])
    b.state.set_adapter(0, 0)
    a = b.infer_seq(PROMPT[:20])
    for (site, l) in ads[0]:
        b.model.adapter_set(0, l, site, None, None)
    b.reset()
    without = b.infer_seq(PROMPT[:20])
    b.state.set_adapter(0, None)
    b.reset()
    assert near(without, b.infer_seq(PROMPT[:20])) and not near(a, without, 1e-3)


def test_refusals(models):
    whole, paths, ads = models
    b = load(whole)
    A, B = ads[0]["att.output", 0]
    with pytest.raises(rsv.RsvError, match="no adapters"):
        b.model.adapter_set(0, 0, "att.output", A, B)
    with pytest.raises(rsv.RsvError, match="no such adapter"):
        b.state.set_adapter(0, 0)
    for args in ((0, 4), (4097, 4), (2, 0), (2, 257)):
        with pytest.raises(rsv.RsvError, match="between"):
            b.model.adapters_new(*args)
    b.model.adapters_new(2, 8)
    with pytest.raises(rsv.RsvError, match="already"):
        b.model.adapters_new(2, 8)
    for args, says in (((0, 0, "att.output", A, B), "rank"), ((2, 0, "att.output", A[:4], B[:, :4]), "slot"), ((0, 9, "att.output", A[:4], B[:, :4]), "layer"), ((0, 0, "ffn.value", A[:4], B[:, :4]), "go with")):
        with pytest.raises(rsv.RsvError, match=says):
            b.model.adapter_set(*args)
    for slot, a in ((0, 2), (0, -2), (1, 0)):
        with pytest.raises(rsv.RsvError):
            b.state.set_adapter(slot, a)
    sc = rsv.Scheduler(b.model, 1)
    with pytest.raises(rsv.RsvError, match="no such adapter"):
        sc.submit([1, 2], 3, adapter=2)


def test_infer_draw(tiny_paths):
    b = rsv.ModelBuilder(tiny_paths["int8"]).build()
    g = np.random.default_rng(2)
    for i, (T, k, p, m) in enumerate([(1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (1.3, 0, 0.8, 0.05), (0.0, 0, 1.0, 0.0), (1.0, 900, 0.95, 0.0)]):
        toks, u = g.integers(0, V, 5 + i), float(np.float32(g.random()))
        b.reset()
        logits = b.infer_tokens(toks)
        b.reset()
        tok, lp = b.infer_draw(toks, rsv.DrawParams(T, k, p, m), u)
        want, wlp = reference(logits, T, k, p, m, u)
        assert tok == want and abs(lp - wlp) <= 2.0**-24 * abs(wlp) + 2.0**-29
    for u in (-0.1, 1.0, float("nan")):
        with pytest.raises(rsv.RsvError, match="u must be"):
            b.infer_draw([1], rsv.DrawParams(), u)
    with pytest.raises(rsv.RsvError):
        b.infer_draw([], rsv.DrawParams(), 0.5)


def test_adapters_then_draw_on_device_memory():
    """The two operators one after the other, as a server's head uses them: shared logits, adapters beside the head, a token each; then the same captured."""
    import torch
    R, K, M, n, r = 48, 256, 4096, 5, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    x, W = torch.randn(R, K, generator=g, device="cuda"), torch.randn(M, K, generator=g, device="cuda") * 0.1
    A, B = (torch.randn(n, r, K, generator=g, device="cuda") * 0.1).half(), (torch.randn(n, M, r, generator=g, device="cuda") * 0.3).half()
    index = torch.randint(-1, n, (R,), generator=g, device="cuda", dtype=torch.int32)
    par, u = torch.from_numpy(rsv.draw_params(np.linspace(0.6, 1.4, R), 0, 0.95, 0.01)).cuda(), torch.rand(R, generator=g, device="cuda")
    base = x @ W.T
    ad, tok, lp = rsv.Adapters(A, B), torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, device="cuda")
    logits = base.clone()
    ad.apply(x, index, logits, base=logits)
    rsv.draw_tokens(logits, par, u, tok, lp)
    want = base.double()
    for i in range(R):
        if index[i] >= 0:
            want[i] += B[index[i]].double() @ (A[index[i]].double() @ x[i].double())
    assert float((logits.double() - want).abs().max()) < 1e-4
    lg, pr = logits.cpu().numpy(), par.cpu().numpy()
    for i in range(R):
        assert int(tok[i]) == reference(lg[i], pr[i, 0], 0, pr[i, 2], pr[i, 3], float(u[i]))[0]
    again, lg2 = torch.zeros_like(tok), torch.empty_like(logits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ad.apply(x, index, lg2, base=base)
        rsv.draw_tokens(lg2, par, u, again)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(lg2, logits) and torch.equal(again, tok)
