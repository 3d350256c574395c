"""CPU checks of sample: the refusals of its entry points and of its Python function, and the plain form on cases that can
be counted by hand."""
import ctypes

import numpy as np
import pytest
import torch

from sandyrt_amd import _lib, ops
from tests import sample_reference as R
from tests.test_quant_cache import tensor

F32, BF16, I32, I64 = _lib.F32, _lib.BF16, _lib.I32, _lib.I64


def workspace(logits):
    need = ctypes.c_size_t(0)
    _lib.dcall("sandy_hip_sample_workspace", logits, ctypes.byref(need))
    return need.value


def test_refusals():
    f, i = tensor((3,), F32), tensor((3,), I64)
    big = tensor((3, 100000))
    default = dict(logits=tensor((3, 1000)), temperature=f, top_k=i, top_p=f, min_p=f, uniforms=f, ids=i, probs=f, work=0x100000,
                   bytes=1 << 40)
    for kw, message in [
        (dict(logits=None), "logits must be"),
        (dict(logits=tensor((1000,))), "logits must be"),
        (dict(logits=tensor((3, 1000), I32)), "logits must be"),
        (dict(logits=tensor((3, 0))), "must have a vocabulary"),
        (dict(logits=tensor((3, (1 << 24) + 1))), "above 2\\^24"),
        (dict(logits=tensor(((1 << 17) + 1, 2))), "more than 2\\^17 rows"),
        (dict(logits=tensor((3, 1000), strides=[1000, 2])), "unit inner stride"),
        (dict(logits=tensor((3, 1000), data=0)), "null"),
        (dict(temperature=i), "contiguous f32"),
        (dict(temperature=tensor((2,), F32)), "contiguous f32"),
        (dict(top_p=tensor((3,), BF16)), "contiguous f32"),
        (dict(min_p=tensor((3,), F32, strides=[2])), "contiguous f32"),
        (dict(min_p=tensor((3, 1), F32)), "contiguous f32"),
        (dict(top_k=f), "top_k must be"),
        (dict(top_k=tensor((4,), I32)), "top_k must be"),
        (dict(uniforms=None), "uniforms must be"),
        (dict(uniforms=tensor((4,), F32)), "uniforms must be"),
        (dict(uniforms=tensor((3,), F32, data=0)), "uniforms must be"),
        (dict(ids=f), "ids must be"),
        (dict(ids=None), "ids must be"),
        (dict(probs=i), "probs must be"),
        (dict(logits=big, work=None), "needs a workspace"),
        (dict(logits=big, work=0x100008), "16-byte aligned"),
        (dict(logits=big, bytes=workspace(big) - 1), "needs a workspace"),
    ]:
        with pytest.raises(_lib.SandyError, match=message):
            _lib.call("sandy_hip_sample", *{**default, **kw}.values(), stream=0)
    e = tensor((0,), F32)
    _lib.call("sandy_hip_sample", tensor((0, 1000)), None, None, None, None, e, tensor((0,), I64), None, None, 0, stream=0)
    assert workspace(tensor((0, 1000))) == 0
    assert 0 == workspace(tensor((1, 1))) < workspace(tensor((64, 262144), F32))


def test_python_refusals():
    u = torch.zeros(3)
    with pytest.raises(ops.SandyError, match="must live on the GPU"):
        ops.sample(torch.zeros(3, 10), u)
    with pytest.raises(ops.SandyError, match=r"\[rows, vocab\]"):
        ops.sample(torch.zeros(10), u)


def test_reference():
    l = [1.0, 3.0, 3.0, -np.inf, 2.0, 3.0]
    assert R.draw(l, 0.0, t=0.0) == (1, 1.0)
    assert R.draw(l, 0.5, k=2) == (2, 0.5) and R.draw(l, 0.49, k=2) == (1, 0.5)
    assert set(R.kept_weights(l, k=4)) == {1, 2, 4, 5}
    assert set(R.kept_weights(l, k=4, least=0.5)) == {1, 2, 5} and set(R.kept_weights(l, least=0.36)) == {1, 2, 4, 5}
    assert set(R.kept_weights([0.0] * 8, p=0.5)) == {0, 1, 2, 3} and set(R.kept_weights([0.0] * 8, p=0.51)) == {0, 1, 2, 3, 4}
    assert set(R.kept_weights([0.0] * 8, k=4, p=0.5)) == {0, 1} and set(R.kept_weights(l, p=0.0)) == {1}
    assert R.draw([-np.inf, np.nan], 0.3) == (-1, 0.0)
    assert R.draw([0.0, np.inf, np.inf], 0.5) == (2, 0.5)
