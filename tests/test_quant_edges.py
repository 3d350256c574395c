"""CPU checks of the quantised paged K/V cache's refusals at its edges."""
import pytest

from sandyrt_amd import _lib
from tests.test_quant_cache import POS, TABLE, cache, other, tensor


def test_outputs_that_repeat_memory():
    """A broadcast q is read; as its own output several rows would be one."""
    for shape, strides in [((3, 4, 1, 64), (256, 0, 64, 1)), ((3, 4, 2, 64), (512, 128, 0, 1)), ((3, 4, 1, 64), (0, 64, 64, 1)),
                           ((3, 4, 1, 64), (256, 64, 64, 0))]:
        q = tensor(shape, strides=strides)
        with pytest.raises(_lib.SandyError, match="output rows must not share memory"):
            _lib.call("sandy_hip_quant_paged_attention", q, cache(), other(), TABLE, POS, None, 0, -1.0, q, None, 0, stream=0)
