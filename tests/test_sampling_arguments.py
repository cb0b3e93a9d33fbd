"""Engine.set_sampling's whole numbers, before the engine is looked at."""
import pytest

import xpu_playground_amd as xpu
from xpu_playground_amd import qwen3


@pytest.mark.parametrize("numbers", [dict(top_k=-1), dict(top_k=1 << 32), dict(top_k=(1 << 32) + 5), dict(top_k=2.0),
                                     dict(seed=-1), dict(seed=1 << 64)])
def test_numbers_that_fields_do_not_hold(numbers):
    """Cut to 32 bits, 2^32 + 5 would be a top-k of 5."""
    eng = qwen3.Engine.__new__(qwen3.Engine)
    eng.lib, eng.handle = xpu.library(), None
    with pytest.raises(ValueError, match="fit"):
        eng.set_sampling(1.0, **numbers)
    with pytest.raises(xpu.XpuError, match="null engine"):
        eng.set_sampling(1.0, top_k=(1 << 32) - 1, seed=(1 << 64) - 1)
