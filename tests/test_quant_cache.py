"""CPU checks of the quantised paged K/V cache: the refusals of its entry
points (host checks, before any device work) and of its Python functions, and
the reference's own arithmetic."""
import ctypes

import numpy as np
import pytest
import torch

from sandyrt_amd import _lib, ops
from tests import quant_reference as R


def tensor(shape, dtype=_lib.BF16, strides=None, data=0x10000):
    t = _lib.SandyTensor()
    t.data, t.dtype, t.rank = data, dtype, len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        t.dims[i], t.strides[i] = shape[i], step
        step *= shape[i]
    for i, s in enumerate(strides or []):
        t.strides[i] = s
    return ctypes.byref(t)


def cache(pool=0x100000, scales=0x200000, format=0, page_size=16, prefix=2, inner=64, num_pages=8):
    return ctypes.byref(_lib.SandyQuantCache(pool, scales, format, 0, page_size, prefix, inner, num_pages))


def other(**kw):
    return cache(pool=0x300000, scales=0x400000, **kw)


TABLE, POS = tensor((3, 4), _lib.I32), tensor((3,), _lib.I64)


def append(k=None, v=None, kc=None, vc=None, table=TABLE, pos=POS, counts=None):
    k = tensor((3, 2, 5, 64)) if k is None else k
    v = k if v is None else v
    _lib.call("sandy_hip_quant_paged_append", k, v or None, kc or cache(), other() if vc is None else (vc or None), table, pos,
              counts, stream=0)


def test_append_refusals():
    for kw, message in [
        (dict(k=tensor((2, 5, 64))), r"rows must be \[B, heads, T, D\]"),
        (dict(k=tensor((3, 2, 5, 64), _lib.I32)), "f32 or bf16"),
        (dict(v=tensor((3, 2, 6, 64))), "same shape and dtype"),
        (dict(v=tensor((3, 2, 5, 64), _lib.F32)), "same shape and dtype"),
        (dict(v=0), "v and its cache or neither"),
        (dict(vc=0), "v and its cache or neither"),
        (dict(k=tensor((3, 4, 5, 64))), "the cache's heads and head dim"),
        (dict(k=tensor((3, 2, 5, 32))), "the cache's heads and head dim"),
        (dict(vc=cache()), "must not share memory"),
        (dict(vc=cache(pool=0x100000 + 8 * 2 * 16 * 64 - 1, scales=0x400000)), "must not share memory"),
        (dict(vc=cache(pool=0x300000, scales=0x200000 - 15)), "must not share memory"),
        (dict(vc=other(format=1)), "same format and shape"),
        (dict(vc=other(num_pages=9)), "same format and shape"),
        (dict(kc=cache(format=2)), "int8 or e4m3"),
        (dict(kc=cache(page_size=24)), "power of two"),
        (dict(kc=cache(page_size=0)), "power of two"),
        (dict(kc=cache(num_pages=0)), "must have pages"),
        (dict(kc=cache(prefix=0)), "must have pages"),
        (dict(kc=cache(pool=0)), "pool or scales is null"),
        (dict(kc=cache(scales=0)), "pool or scales is null"),
        (dict(kc=cache(page_size=1 << 25)), "above 2\\^30 elements"),
        (dict(kc=cache(prefix=1 << 30, num_pages=(1 << 31) - 1)), "too many pages"),
        (dict(table=tensor((2, 4), _lib.I32)), "block table must be"),
        (dict(table=tensor((3, 4), _lib.I64)), "block table must be"),
        (dict(table=tensor((3, 4), _lib.I32, strides=(1, 3))), "block table must be"),
        (dict(table=tensor((3, 1 << 27), _lib.I32)), "more than 2\\^30 rows"),
        (dict(pos=tensor((2,), _lib.I64)), "position_offsets must be"),
        (dict(pos=tensor((3,), _lib.F32)), "position_offsets must be"),
        (dict(pos=tensor((3,), _lib.I64, strides=(2,))), "position_offsets must be"),
        (dict(counts=tensor((4,), _lib.I32)), "counts must be"),
        (dict(counts=tensor((3,), _lib.F32)), "counts must be"),
    ]:
        with pytest.raises(_lib.SandyError, match=message):
            append(**kw)


def test_read_refusals():
    def read(k=None, v=None, kc=None, vc=None, pos=POS):
        k = tensor((3, 2, 5, 64)) if k is None else k
        _lib.call("sandy_hip_quant_paged_read", kc or cache(), other() if vc is None else (vc or None), TABLE, pos, None,
                  k, k if v is None else (v or None), stream=0)

    for kw, message in [
        (dict(v=0), "and v's or neither"),
        (dict(vc=0), "and v's or neither"),
        (dict(k=tensor((3, 2, 5, 64), strides=(640, 64, 128, 1))), "must be contiguous"),
        (dict(k=tensor((3, 2, 5, 64), _lib.I64)), "f32 or bf16"),
        (dict(v=tensor((3, 2, 5, 64), _lib.F32)), "same shape and dtype"),
        (dict(k=tensor((3, 2, 5, 32))), "the cache's heads and head dim"),
        (dict(vc=other(inner=32)), "same format and shape"),
        (dict(pos=tensor((3, 2), _lib.I64)), "position_offsets must be"),
    ]:
        with pytest.raises(_lib.SandyError, match=message):
            read(**kw)


def test_attention_refusals():
    def attend(q=None, out=None, kc=None, vc=None, window=0, counts=None, table=TABLE):
        q = tensor((3, 4, 1, 64)) if q is None else q
        _lib.call("sandy_hip_quant_paged_attention", q, kc or cache(), other() if vc is None else (vc or None), table,
                  POS, counts, window, -1.0, q if out is None else out, None, 0, stream=0)

    for kw, message in [
        (dict(q=tensor((3, 4, 64))), r"expects q \[B, Hq, T, D\]"),
        (dict(q=tensor((3, 4, 1, 64), _lib.I32)), "unsupported dtype"),
        (dict(q=tensor((3, 4, 1, 32))), "head dimension mismatch"),
        (dict(q=tensor((3, 5, 1, 64))), "divisible by kv_heads"),
        (dict(q=tensor((3, 4, 1, 1024)), kc=cache(inner=1024)), "above 512"),
        (dict(out=tensor((3, 4, 1, 64), _lib.F32)), "output shape mismatch"),
        (dict(out=tensor((3, 4, 2, 64))), "output shape mismatch"),
        (dict(window=-1), "window must be >= 0"),
        (dict(vc=0), "requires q and caches"),
        (dict(vc=other(format=1)), "same format and shape"),
        (dict(q=tensor((2, 4, 1, 64))), "block table must be"),
        (dict(counts=tensor((2,), _lib.I64)), "counts must be"),
    ]:
        with pytest.raises(_lib.SandyError, match=message):
            attend(**kw)


def test_attention_workspace_refusals():
    """The workspace a call of these sizes needs, and calls that bring less."""
    need = ctypes.c_size_t(7)

    def query(q, kc=None, table=TABLE):
        _lib.dcall("sandy_hip_quant_paged_attention_workspace", q, kc or cache(), table, 0, ctypes.byref(need))
        return need.value

    assert query(tensor((3, 4, 1, 64))) == 0          # 64 keys: one workgroup a head
    assert query(tensor((3, 4, 0, 64))) == 0
    wide = tensor((3, 4096), _lib.I32)
    bytes_ = query(tensor((3, 4, 1, 64)), table=wide)
    assert bytes_ > 0 and bytes_ % 16 == 0
    assert query(tensor((3, 4, 1, 20)), cache(inner=20), wide) == 0  # the general kernel needs none
    for work, size in ((None, 0), (0x10000, bytes_ - 1), (0x10008, bytes_)):
        with pytest.raises(_lib.SandyError, match=f"workspace of {bytes_} bytes"):
            _lib.call("sandy_hip_quant_paged_attention", tensor((3, 4, 1, 64)), cache(), other(), wide, POS, None, 0, -1.0,
                      tensor((3, 4, 1, 64)), work, size, stream=0)
    with pytest.raises(_lib.SandyError, match="divisible by kv_heads"):
        query(tensor((3, 5, 1, 64)))
    with pytest.raises(_lib.SandyError, match="requires a block table"):
        query(tensor((3, 4, 1, 64)), table=tensor((3,), _lib.I32))


def test_sizes_past_the_indices():
    """Views that repeat memory: counts past 32 bits, products past 64."""
    big = 1 << 30
    pos, table = tensor((1,), _lib.I64), tensor((1, 4), _lib.I32)
    many = 1 << 31
    for k, kc, tab, at in [
        (tensor((1, 2, big + 1, 64)), cache(), table, pos),
        (tensor((many, 2, 1, 64)), cache(), tensor((many, 4), _lib.I32), tensor((many,), _lib.I64)),
        (tensor((many - 1, 2, big, 64)), cache(), tensor((many - 1, 4), _lib.I32), tensor((many - 1,), _lib.I64)),
    ]:
        with pytest.raises(_lib.SandyError, match="too large"):
            _lib.call("sandy_hip_quant_paged_append", k, None, kc, None, tab, at, None, stream=0)
        with pytest.raises(_lib.SandyError, match="too large"):
            _lib.call("sandy_hip_quant_paged_read", kc, None, tab, at, None, k, None, stream=0)
    need = ctypes.c_size_t(0)
    for shape in [(1, 2 * big + 2, 1, 64), (1, 4, big + 1, 64), (many, 4, 1, 64), (1 << 30, 1 << 28, 1 << 10, 64)]:
        q = tensor(shape)
        with pytest.raises(_lib.SandyError, match="too large"):
            _lib.dcall("sandy_hip_quant_paged_attention_workspace", q, cache(), table, 0, ctypes.byref(need))
        with pytest.raises(_lib.SandyError, match="too large"):
            _lib.call("sandy_hip_quant_paged_attention", q, cache(), other(), table, pos, None, 0, -1.0, q, None, 0, stream=0)


def test_read_outputs_of_other_lengths():
    c = ops.QuantPagedCache.empty(4, 2, 16, 64, device="cpu")
    table, pos = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(_lib.SandyError, match="the call's rows"):
        ops.quant_paged_read(c, None, table, pos, 3, k_out=torch.zeros(1, 2, 4, 64))


def test_python_refusals():
    pool, scales = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    with pytest.raises(_lib.SandyError, match="int8 or e4m3"):
        ops.QuantPagedCache.empty(4, 2, 16, 64, "int4", device="cpu")
    with pytest.raises(_lib.SandyError, match="int8 or e4m3"):
        ops.QuantPagedCache(pool.float(), scales).pack()
    with pytest.raises(_lib.SandyError, match="contiguous"):
        ops.QuantPagedCache(pool.transpose(1, 2), scales).pack()
    with pytest.raises(_lib.SandyError, match="scales must be"):
        ops.QuantPagedCache(pool, scales[:3]).pack()
    with pytest.raises(_lib.SandyError, match="scales must be"):
        ops.QuantPagedCache(pool, scales.int()).pack()
    c, d = (ops.QuantPagedCache.empty(4, 2, 16, 64, f, device="cpu") for f in ("int8", "e4m3"))
    assert c.pool.dtype == torch.int8 and d.pool.dtype == torch.float8_e4m3fn and not d.pool.float().any()
    x, table, pos = torch.zeros(1, 2, 1, 64), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(_lib.SandyError, match="must live on the GPU"):
        ops.quant_paged_append(x, x, c, d, table, pos)
    with pytest.raises(_lib.SandyError, match="must live on the GPU"):
        ops.quant_paged_read(c, None, table, pos, 3)
    with pytest.raises(_lib.SandyError, match="must live on the GPU"):
        ops.quant_paged_attention(x, c, c, table, pos)
    far = ops.QuantPagedCache(pool.to("meta"), scales.to("meta"))
    with pytest.raises(_lib.SandyError, match="must live on"):
        ops.quant_paged_read(far, None, table, pos, 3)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_reference_arithmetic(fmt):
    """The reference against e4m3's and int8's own definitions, and the bound of
    a payload that was rounded again and again."""
    r = np.random.default_rng(1)
    x = np.concatenate([r.uniform(-R.LARGEST[fmt], R.LARGEST[fmt], 4000), r.standard_normal(2000) * 0.02, [0.0]])
    got = R.round_payload(x, fmt)
    want = torch.from_numpy(x).float()
    want = torch.round(want) if fmt == "int8" else want.to(torch.float8_e4m3fn).float()
    near = R.round_payload(x.astype(np.float32).astype(np.float64), fmt)
    np.testing.assert_array_equal(near, want.double().numpy())
    assert np.abs(got).max() <= R.LARGEST[fmt]
    assert R.code_of(3.4e38, fmt) == R.code_of(float("nan"), fmt) == 255
    for amax in (1.0, 126.9, 127.0, 127.0001, 448.0, 448.1, 2.9e38, 1e-45, 0.0):
        c = R.code_of(amax, fmt)
        assert 1 <= c <= 254 and amax * 2.0 ** (127 - c) <= R.LARGEST[fmt]
        assert c == 1 or amax * 2.0 ** (128 - c) > R.LARGEST[fmt]
    c = R.Cache(1, 1, 16, 4, fmt)
    first = r.standard_normal((1, 1, 1, 4))
    c.append(first, [[0]], [0], [1])
    for i in range(1, 16):  # each row louder than the last: the scale grows every time
        c.append(r.standard_normal((1, 1, 1, 4)) * 1.7 ** i + 1.7 ** i, [[0]], [i], [1])
    off = np.abs(c.rows_of([0], 0, 1) - first[0])
    step = 2.0 ** (int(c.code[0, 0]) - 127) * (1.0 if fmt == "int8" else 2.0 ** -9)
    assert (off <= np.maximum(step, 0 if fmt == "int8" else np.abs(first[0]) * 2.0 ** -4)).all()
