"""Sessions with and without adapters of one model: what a step launches, and adapters beside int8 weights."""
import numpy as np
import pytest

import rwkv_rsv_b200 as rsv

pytestmark = pytest.mark.gpu

LAYERS, C, F, V = 4, 512, 2048, 4096


def adapted(path, slots=2, rank=4, seed=1):
    b = rsv.ModelBuilder(path).build()
    b.model.adapters_new(slots, rank)
    g = np.random.default_rng(seed)
    for l in range(LAYERS):
        for site, K in (("att.output", C), ("ffn.value", F)):
            b.model.adapter_set(1, l, site, g.standard_normal((rank, K)).astype(np.float16) * np.float16(0.05), g.standard_normal((C, rank)).astype(np.float16) * np.float16(0.05))
    return b


def run(sc, model, jobs):
    """Tokens of every job, and the launches that took."""
    before = model.launch_count()
    ids = [sc.submit(p, n, adapter=a) for p, n, a in jobs]
    done = sc.run_until_done()
    return [list(done[i]) for i in ids], model.launch_count() - before


PROMPTS = [np.random.default_rng(s).integers(0, V, n).astype(np.uint32) for s, n in ((0, 40), (1, 17), (2, 64))]


@pytest.mark.parametrize("quant", ["fp16", "int8"])
def test_steps_of_plain_sessions_launch_no_adapters(tiny_paths, quant):
    """... whether or not an earlier session of the same slots had one, and whether or not another slot has one that takes no part in the step."""
    b = adapted(tiny_paths[quant])
    plain = [(p, 6, None) for p in PROMPTS]
    sc = rsv.Scheduler(b.model, max_slots=3, chunk=32, max_rows=64)
    run(sc, b.model, plain)  # (a model's first steps lay out weights)
    want, fresh = run(sc, b.model, plain)
    one, with_adapter = run(sc, b.model, [(p, 6, 1) for p in PROMPTS])
    assert with_adapter > fresh and one != want
    again, after = run(sc, b.model, plain)
    assert again == want and after == fresh, (after, fresh)
    mixed, between = run(sc, b.model, [(PROMPTS[0], 6, None), (PROMPTS[1], 6, 1), (PROMPTS[2], 6, None)])
    assert mixed == [want[0], one[1], want[2]] and fresh < between <= with_adapter
    # one session of three has the adapter, and is done before the others begin to generate
    long = np.concatenate([PROMPTS[0]] * 8)
    for first in (None, 1):
        sc2 = rsv.Scheduler(b.model, max_slots=2, chunk=32, max_rows=64)
        sc2.submit(PROMPTS[1][:2], 1, adapter=first)
        sc2.submit(long, 4)
        sc2.step(), b.model.synchronize()
        before = b.model.launch_count()
        sc2.run_until_done()
        if first is None:
            rest = b.model.launch_count() - before
        else:
            assert b.model.launch_count() - before == rest


def test_adapters_beside_int8_weights(tiny_paths):
    """Prompt and token by token agree, and an adapter of rank 0 or scale 0 changes nothing (bit for bit: out = base + 0)."""
    b = adapted(tiny_paths["int8"])
    toks = PROMPTS[2]
    plain = b.infer_seq(toks)
    b.reset()
    b.state.set_adapter(0, 0)  # rank 0 at every site
    assert np.array_equal(b.infer_seq(toks), plain)
    b.reset()
    b.state.set_adapter(0, 1)
    seq = b.infer_seq(toks)
    b.reset()
    one = b.infer_tokens(toks)
    assert np.abs(seq - plain).max() > 1e-2
    assert float(np.sqrt(np.mean((seq - one) ** 2))) <= 1e-3  # (as the paths of the model itself against its oracle)
