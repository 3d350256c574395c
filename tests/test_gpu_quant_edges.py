"""The quantised paged K/V cache on the GPU where it can go wrong: sums that
cancel."""
import numpy as np
import pytest
import torch

from tests import quant_reference as R
from tests.helpers import from_f32, rng
from tests.test_gpu_quant_cache import BF16, cuda, empty, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from sandyrt_amd import ops
    return ops


def attend(ops, q, kc, vc, table, pos, what="", **kw):
    """check(), the weights held like everything else in fp32's 24 bits."""
    got = ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array(pos)), **kw)
    ops.check_device_errors()
    want, slack = R.attention(f64(q), R.Cache.of(kc), R.Cache.of(vc), table, pos, [q.shape[2]] * q.shape[0],
                              kw.get("window", 0), kw.get("scale", -1.0))
    R.assert_attention(got, want, slack, what)
    return got


# the decode kernel, the prompt kernel (head dims that are multiples of 16)
FORMS = {"decode": 1 << 30, "prompt": 1}


@pytest.fixture
def form(monkeypatch, request):
    monkeypatch.setenv("SANDY_QUANT_PROMPT_WGS", str(FORMS[request.param]))
    return request.param


# ------------------------------------------------------------------ sums that cancel
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("form", FORMS, indirect=True)
def test_weights_keep_24_bits(ops, form, fmt):
    """Two keys whose values cancel to a few thousandths: what a weight loses shows
    above the output's own rounding.  (A weight held to 16 bits is off by up to
    2^-16, the bound here is about 65 roundings of 2^-24, 2^-18.)"""
    r = rng(3)
    B, hq, heads, dim = 512, 8, 2, 16
    c = [empty(ops, 1, heads, 16, dim, fmt, i) for i in (1, 2)]
    for x in c:
        x.pool.copy_(torch.from_numpy(r.integers(-127, 128, x.pool.shape)).cuda().float().to(x.pool.dtype))
    c[0].scales.fill_(121)
    c[1].scales.fill_(127)
    x = np.zeros((B, hq, 2, dim), np.float32)
    x[..., 0] = 0.4 * r.standard_normal(x.shape[:3])
    attend(ops, from_f32(x, BF16), *c, np.zeros((B, 1), np.int32), [1] * B, window=2, scale=0.25)
