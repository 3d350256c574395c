"""Drawing tokens on the GPU, what the settings and logits may hold at their edges, rows of one workgroup and rows in parts."""
import numpy as np
import pytest
import torch

from sandyrt_amd import ops
from tests.test_gpu_sample import check, f32, model_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [1, 300, 8192, 8193, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_uniform_number_of_minus_zero(vocab, dtype):
    """-0.0 is 0.0: the first token that is kept."""
    x = model_logits(np.random.default_rng(vocab), 4, vocab, dtype)
    for s in ({}, dict(k=[1, 2, 40, 3000]), dict(p=[0.1, 0.5, 0.9, -0.0]), dict(t=[-0.0, 0.7, 1.0, 3.0], k=[0, 50, 7, 2000], p=[0.9, 0.8, 1.0, 0.95], least=[-0.0, 0.1, 0.0, 0.02])):
        signed, plain = check(x, [-0.0] * 4, **s), check(x, [0.0] * 4, **s)
        assert torch.equal(signed[0], plain[0]) and torch.equal(signed[1], plain[1])
    ops.check_device_errors()


@pytest.mark.parametrize("vocab", [5000, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_of_every_kind(vocab, dtype):
    """NaN, signalling ones among them, beside the likeliest tokens: never drawn, and their neighbours keep their ranks."""
    rng = np.random.default_rng(vocab)
    x = model_logits(rng, 6, vocab, dtype)
    kinds = {torch.float32: (0x7f800001, 0xff800001, 0x7fc00000, 0xffffffff), torch.bfloat16: (0x7f81, 0xff81, 0x7fc0, 0xffff)}[dtype]
    bits = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    width = 32 if dtype == torch.float32 else 16
    top = x.float().argmax(1).tolist()
    for r, at in enumerate(top):
        for i in range(4):
            kind = kinds[(r + i) % 4]
            bits[r, at ^ (i + 1) if at ^ (i + 1) < vocab else at - 1] = kind - (1 << width) if kind >> (width - 1) else kind
    assert torch.isnan(x).sum() >= 18
    for u in (0.0, 0.4, 1 - 2.0 ** -24):
        for s in ({}, dict(t=[0.0] * 6), dict(k=[1, 3, 50, 2000, 0, 2]), dict(p=[0.5, 0.9, 0.99, 0.3, 0.8, 0.95], least=[0.0, 0.1, 0.0, 0.3, 0.01, 0.0])):
            check(x, [u] * 6, **s)
    check(x.mul_(float("nan")), [0.5] * 6)  # nothing left
