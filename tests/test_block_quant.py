"""CPU checks of the operators over rows and weights in 8 bits: the refusals of their entry points (host checks,
before any device work) and of their Python functions."""
import pytest
import torch

from sandyrt_amd import _lib, ops
from tests.test_quant_cache import tensor

U8, F32, BF16, I32, I64 = _lib.U8, _lib.F32, _lib.BF16, _lib.I32, _lib.I64


def refused(name, cases, default):
    for kw, message in cases:
        args = {**default, **kw}
        with pytest.raises(_lib.SandyError, match=message):
            _lib.call(name, *args.values(), stream=0)


def test_block_quant_refusals():
    default = dict(x=tensor((3, 300)), block_rows=1, payload=tensor((3, 300), U8), scales=tensor((3, 3), U8))
    refused("sandy_hip_block_quant", [
        (dict(block_rows=2), "block_rows must be 1 or 128"),
        (dict(block_rows=0), "block_rows must be 1 or 128"),
        (dict(x=None), "x must be f32 or bf16"),
        (dict(x=tensor((3, 300), I32)), "x must be f32 or bf16"),
        (dict(x=tensor((300,))), "rank 2 or 3"),
        (dict(x=tensor((3, 300), data=0)), "x is null"),
        (dict(x=tensor((3, 299))), "x's shape"),
        (dict(payload=None), "requires payloads and scales"),
        (dict(payload=tensor((3, 300))), "must be u8"),
        (dict(payload=tensor((3, 300), U8, data=0)), "null"),
        (dict(payload=tensor((3, 300), U8, strides=[1, 3])), "unit inner stride"),
        (dict(payload=tensor((3, 300), U8, strides=[299, 1])), "without overlap"),
        (dict(payload=tensor((3, 300), U8, strides=[0, 1])), "without overlap"),
        (dict(payload=tensor((3, 300), U8, strides=[-300, 1])), "without overlap"),
        (dict(scales=tensor((3, 2), U8)), "scales must be"),
        (dict(scales=tensor((1, 3), U8)), "block_rows"),
        (dict(scales=tensor((3, 3), U8, strides=[4, 1])), "contiguous"),
        (dict(block_rows=128), "block_rows"),
        (dict(x=tensor((2, 3, 300)), payload=tensor((2, 3, 300), U8, strides=[899, 300, 1]), scales=tensor((2, 3, 3), U8)),
         "without overlap"),
        (dict(x=tensor((2, 3, 300)), payload=tensor((2, 3, 300), U8), scales=tensor((3, 3, 3), U8)), "scales must be"),
    ], default)
    for rows in ((0, 300), (3, 0)):  # nothing to do
        _lib.call("sandy_hip_block_quant", tensor(rows), 1, tensor(rows, U8), tensor((rows[0], -(-rows[1] // 128)), U8), stream=0)


def test_block_dequant_refusals():
    refused("sandy_hip_block_dequant", [
        (dict(out=tensor((3, 300), I32)), "contiguous f32 or bf16"),
        (dict(out=tensor((3, 301))), "payloads' shape"),
        (dict(out=tensor((3, 300), strides=[301, 1])), "contiguous"),
        (dict(out=tensor((3, 300), data=0)), "out is null"),
        (dict(scales=tensor((2, 3), U8)), "scales must be"),
    ], dict(payload=tensor((3, 300), U8), scales=tensor((3, 3), U8), out=tensor((3, 300))))


def linear_args(**kw):
    args = dict(x=tensor((3, 304), U8), xs=tensor((3, 3), U8), w=tensor((200, 304), U8), ws=tensor((2, 3), U8), bias=None,
                out=tensor((3, 200)))
    return {**args, **kw}


def test_quant_linear_refusals():
    refused("sandy_hip_quant_linear", [
        (dict(x=tensor((3, 288), U8)), "contracting dimension"),
        (dict(x=tensor((3, 304), BF16)), "must be u8"),
        (dict(x=tensor((3, 0), U8), xs=tensor((3, 0), U8), w=tensor((200, 0), U8), ws=tensor((2, 0), U8)), "positive dimensions"),
        (dict(w=tensor((0, 304), U8), ws=tensor((0, 3), U8), out=tensor((3, 0))), "positive dimensions"),
        (dict(x=tensor((200, 304), U8), xs=tensor((2, 3), U8), out=tensor((200, 200))), "scale for every row"),
        (dict(x=tensor((3, 304), U8, strides=[312, 1])), "16-byte boundaries"),
        (dict(x=tensor((3, 304), U8, data=0x10008)), "16-byte boundaries"),
        (dict(w=tensor((200, 304), U8, strides=[305, 1])), "16-byte boundaries"),
        (dict(w=tensor((200, 304), U8, strides=[1 << 24, 1])), "2\\^22 bytes"),
        (dict(x=tensor((2, 3, 304), U8, strides=[1024, 304, 1]), xs=tensor((2, 3, 3), U8), out=tensor((2, 3, 200))), "evenly spaced"),
        (dict(x=tensor((2, 3, 304), U8), xs=tensor((2, 3, 3), U8), out=tensor((2, 3, 200), strides=[900, 200, 1])), "evenly spaced"),
        (dict(out=tensor((3, 200), I32)), "f32 or bf16"),
        (dict(out=tensor((3, 201))), "output shape"),
        (dict(out=tensor((4, 200))), "output shape"),
        (dict(out=tensor((1, 3, 200))), "output shape"),
        (dict(out=tensor((3, 200), strides=[1, 3])), "unit inner stride"),
        (dict(out=tensor((3, 200), strides=[199, 1])), "evenly spaced"),
        (dict(out=tensor((3, 200), data=0)), "out is null"),
        (dict(w=tensor((1, 200, 304), U8), ws=tensor((1, 2, 3), U8)), "weight must be rank 2"),
        (dict(bias=tensor((200,), F32)), "bias must be"),
        (dict(bias=tensor((199,))), "bias must be"),
        (dict(bias=tensor((200,), strides=[2])), "bias must be"),
    ], linear_args())
    _lib.call("sandy_hip_quant_linear", *linear_args(x=tensor((0, 304), U8), xs=tensor((0, 3), U8), out=tensor((0, 200))).values(),
              stream=0)


def test_quant_moe_matmul_refusals():
    default = dict(x=tensor((9, 304), U8), xs=tensor((9, 3), U8), offsets=tensor((5,), I64), w=tensor((4, 200, 304), U8),
                   ws=tensor((4, 2, 3), U8), out=tensor((9, 200)))
    refused("sandy_hip_quant_moe_matmul", [
        (dict(x=tensor((1, 9, 304), U8), xs=tensor((1, 9, 3), U8), out=tensor((1, 9, 200))), "expects ranks"),
        (dict(w=tensor((200, 304), U8), ws=tensor((2, 3), U8)), "expects ranks"),
        (dict(offsets=tensor((4,), I64)), "expert_offsets must be"),
        (dict(offsets=tensor((5,), F32)), "expert_offsets must be"),
        (dict(offsets=tensor((5,), I64, strides=[2])), "expert_offsets must be"),
        (dict(offsets=None), "expert_offsets must be"),
        (dict(w=tensor((4, 200, 304), U8, strides=[200 * 304 + 8, 304, 1])), "16-byte boundaries"),
        (dict(ws=tensor((4, 3, 3), U8)), "scales must be"),
    ], default)


def test_python_refusals():
    q = ops.QuantMatrix.empty((3, 300), device="cpu")
    assert q.payload.shape == (3, 300) and q.payload.stride(0) == 304 and q.scales.shape == (3, 3)
    assert ops.QuantMatrix.empty((2, 300, 256), 128, device="cpu").scales.shape == (2, 3, 2)
    x = torch.zeros(3, 300)
    for call in (lambda: ops.block_quant(x), lambda: ops.block_dequant(q), lambda: ops.quant_linear(q, q),
                 lambda: ops.quant_moe_matmul(q, torch.zeros(2, dtype=torch.int64), q)):
        with pytest.raises(ops.SandyError, match="must live on the GPU"):
            call()
    with pytest.raises(ops.SandyError, match="block_rows"):
        ops.block_quant(x, 64)
    with pytest.raises(ops.SandyError, match="rank 2 or 3"):
        ops.block_quant(x[0])
    with pytest.raises(ops.SandyError, match="float8_e4m3fn"):
        ops.quant_linear(ops.QuantMatrix(q.payload.view(torch.uint8), q.scales), q)
    with pytest.raises(ops.SandyError, match="uint8"):
        ops.block_dequant(ops.QuantMatrix(q.payload, q.scales.int()))
