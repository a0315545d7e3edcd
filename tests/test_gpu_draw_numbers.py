"""Random numbers next to 1 that Bundle.infer_draw takes."""
import numpy as np
import pytest

import rwkv_rsv_b200 as rsv

pytestmark = pytest.mark.gpu


TOKENS = np.arange(3, 20, dtype=np.uint32)


@pytest.mark.parametrize("u", [1 - 1e-9, 1 - 2.0**-25, 1 - 2.0**-53])
def test_any_u_under_one_is_drawn(tiny_paths, u):
    """A double under 1 may round to 1 as a float: it counts as the largest float under 1."""
    b = rsv.ModelBuilder(tiny_paths["fp16"]).build()
    want = b.infer_draw(TOKENS, rsv.DrawParams(), float(np.nextafter(np.float32(1), np.float32(0))))
    b.reset()
    assert b.infer_draw(TOKENS, rsv.DrawParams(), u) == want
    for bad in (1.0, 1 + 1e-9, -1e-3, float("nan")):
        with pytest.raises(rsv.RsvError, match="u must be"):
            b.infer_draw([1], rsv.DrawParams(), bad)
