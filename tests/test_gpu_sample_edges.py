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
