"""What Model.adapter_set refuses."""
import numpy as np
import pytest

import rwkv_rsv_b200 as rsv

pytestmark = pytest.mark.gpu


def test_adapter_set_refuses_what_fp16_cannot_hold(tiny_paths):
    b = rsv.ModelBuilder(tiny_paths["fp16"]).build()
    b.model.adapters_new(2, 4)
    A, B = np.full((4, 512), 0.5, np.float32), np.full((512, 4), 0.5, np.float32)
    for a, c in ((A * 2e5, B), (A, B * 2e5), (A, -B * 2e5)):
        with pytest.raises(rsv.RsvError, match="float16"):
            b.model.adapter_set(0, 0, "att.output", a, c)
    b.model.adapter_set(0, 0, "att.output", A * 65504 * 2, B)  # the largest fp16 number itself
    for args in ((0, 0, "att.key", None, None), (0, 0, "att.key", A, B)):
        with pytest.raises(rsv.RsvError, match="att.key"):
            b.model.adapter_set(*args)
