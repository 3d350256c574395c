"""CPU checks of the quantised paged K/V cache's refusals at its edges, and its choice between kernels."""
import ctypes

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


def test_few_rows_a_sequence_keep_the_tiles_that_split():
    """A call on 16-row tiles splits a wide table's keys and so needs a workspace; the
    prompt kernel, which does not, takes many workgroups of more rows than such a tile."""
    need = ctypes.c_size_t(0)

    def splits(batch, q_heads, tokens, heads, dim=64, dtype=_lib.BF16):
        _lib.dcall("sandy_hip_quant_paged_attention_workspace", tensor((batch, q_heads, tokens, dim), dtype),
                   cache(prefix=heads, inner=dim), tensor((batch, 1024), _lib.I32), 0, ctypes.byref(need))
        return need.value > 0

    for batch, q_heads, tokens, heads in ((48, 32, 2, 4), (96, 32, 2, 4), (120, 32, 2, 4), (40, 12, 16, 12), (64, 16, 4, 4), (20, 12, 2, 12)):
        assert splits(batch, q_heads, tokens, heads)
        assert splits(batch, q_heads, tokens, heads, 128)
    assert splits(63, 32, 3, 4) and not splits(64, 32, 3, 4)              # 252 and 256 workgroups
    assert splits(47, 32, 3, 4, 128) and not splits(48, 32, 3, 4, 128)    # 188 and 192
    assert splits(48, 32, 3, 4, 128, _lib.F32) and not splits(64, 32, 3, 4, 128, _lib.F32)
    assert splits(64, 32, 3, 4, 256, _lib.F32) and not splits(64, 32, 3, 4, 256)


def test_forced_splits_of_many_tiles(monkeypatch):
    """More workgroups than a launch can have are not asked for."""
    need = ctypes.c_size_t(0)
    monkeypatch.setenv("SANDY_QUANT_SPLITS", "256")
    for batch in (3, 9000, 1 << 20):
        _lib.dcall("sandy_hip_quant_paged_attention_workspace", tensor((batch, 16, 1, 64)), cache(prefix=8),
                   tensor((batch, 4096), _lib.I32), 0, ctypes.byref(need))
        units, part = 8 * batch, 16 * (64 + 2) * 4
        splits = max(1, need.value // part // units)
        assert splits == min(256, max(1, (2 ** 32 - 1) // 256 // units))
