"""The quantised paged K/V cache on the GPU where it can go wrong: sums that
cancel, values next to the largest and smallest that a block holds,
prompts of several rounds of keys, long appended blocks, switches, graphs, and
streams that come and go."""
import ctypes

import numpy as np
import pytest
import torch

from tests import quant_reference as R
from tests.helpers import from_f32, rng
from tests.test_gpu_quant_cache import BF16, F32, assert_same, cuda, empty, f64, filled, loud_rows, make_table

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


# ------------------------------------------------------------------ values next to the largest
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("T,dim", [(1, 64), (33, 64), (5, 128), (19, 256), (3, 36)])
def test_values_near_the_largest(ops, form, T, dim, fmt, dtype):
    """Means of values up to the largest that a block holds are finite, also where
    the weights' sum times them is not; ordinary and tiny values beside them count."""
    r = rng(35 + T)
    n, top = 220, R.LARGEST[fmt] * 2.0 ** (121 if fmt == "int8" else 119)
    table, pages = make_table(r, [n], 16)
    k, v = (r.standard_normal((1, 4, n, dim)) for _ in range(2))
    v[:, 0] = top * r.uniform(0.5, 1, v[:, 0].shape)     # one sign: the mean is as large
    v[:, 1, 96:160] *= 2.0 ** 118                         # some blocks in the middle
    v[:, 2, :16] *= 2.0 ** 110                            # of next to no weight
    k[:, 2, :16] *= 1e-3
    v[:, 3, 200:] *= 1e-37
    v[:, 3, 100:112] = top * r.choice([-1, 1], v[:, 3, 100:112].shape)
    k, v = (from_f32(x.astype(np.float32), dtype) for x in (k, v))
    if dtype == BF16:  # not rounded past it
        v = v.clamp(-top, top)
    kc, vc = (empty(ops, pages, 4, 16, dim, fmt, i) for i in (1, 2))
    ops.quant_paged_append(k, v, kc, vc, cuda(table), cuda(np.zeros(1, np.int64)))
    assert (vc.scales[int(table[0, 0]), 0] > 240).all() and not (vc.scales == 255).any()
    q = r.standard_normal((1, 8, T, dim)).astype(np.float32)
    for scale in (-1.0, 1.0):  # flat, and one key outweighing the others
        got = attend(ops, from_f32(q, dtype), kc, vc, table, [n - T], f"scale {scale}", scale=scale)
        assert torch.isfinite(got).all() and got[0, 0].abs().max() > 2.0 ** 126


@pytest.mark.parametrize("merge_kernel", [0, 1])
@pytest.mark.parametrize("splits,T,dim,dtype", [(1, 1, 64, BF16), (5, 1, 128, F32), (40, 1, 64, BF16), (40, 2, 256, BF16), (17, 9, 64, F32)])
def test_splits_with_values_near_the_largest(ops, monkeypatch, splits, T, dim, dtype, merge_kernel):
    """Some splits, and some rounds of a wave's keys, with such values and the others without."""
    ops._quant_workspace.cache_clear()
    monkeypatch.setenv("SANDY_QUANT_SPLITS", str(splits))
    monkeypatch.setenv("SANDY_QUANT_MERGE_KERNEL", str(merge_kernel))
    r = rng(splits + T)
    ctx = [9000, 700]
    table, kc, vc = filled(ops, r, ctx, 2, dim, 16, "int8", 5)
    for at in (5, 300, 301, 500):  # pages of the first sequence: keys 80.., 4800.., 8000..
        vc.scales[int(table[0, at]), 0] = 248
    vc.scales[int(table[1, 20]), 1] = 246
    q = from_f32(2 * r.standard_normal((2, 8, T, dim)).astype(np.float32), dtype)
    got = attend(ops, q, kc, vc, table, [c - T for c in ctx])
    assert torch.isfinite(got).all()
    assert torch.equal(got, attend(ops, q, kc, vc, table, [c - T for c in ctx]))
    attend(ops, q, kc, vc, table, [c - T for c in ctx], window=1500)
    ops._quant_workspace.cache_clear()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("dim", [64, 112])
def test_keys_of_the_smallest_scale(ops, form, dim, dtype):
    """Loud queries of the quietest keys: scores of ordinary size."""
    r = rng(37)
    table, kc, vc = filled(ops, r, [60], 2, dim, 16, "int8", 3)
    kc.scales.fill_(1)
    x = np.zeros((1, 8, 5, dim), np.float32)
    x[..., 3] = 2.0 ** 120 * r.uniform(-1, 1, x.shape[:3])
    attend(ops, from_f32(x, dtype), kc, vc, table, [55])
    # factors that underflow: every key weighs the same, the masked ones nothing
    attend(ops, from_f32(x, dtype), kc, vc, table, [55], window=20, scale=1e-30)


# ------------------------------------------------------------------ long prompts and appends
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("form", ["prompt"], indirect=True)
@pytest.mark.parametrize("hq,heads,dim", [(8, 2, 64), (4, 2, 96), (4, 1, 256)])
def test_prompts_behind_long_contexts(ops, form, hq, heads, dim, fmt, dtype):
    """A wave takes 32 pairs of key tiles a round, the four 4096 keys: contexts on
    both sides of one round and of two, windows that begin in the second, a NaN block
    and a page that is not there behind the first."""
    from sandyrt_amd._lib import SandyError
    r = rng(dim)
    T = 5
    ctx = [4095, 4096, 4097, 4128, 8193, 9000]
    table, kc, vc = filled(ops, r, ctx, heads, dim, 16, fmt, 7)
    kc.scales[int(table[5, 400]), 0] = 255   # keys 6400 .. 6415
    vc.scales[int(table[4, 300]), heads - 1] = 255
    q = from_f32(r.standard_normal((len(ctx), hq, T, dim)).astype(np.float32), dtype)
    pos = [c - T for c in ctx]
    attend(ops, q, kc, vc, table, pos)
    attend(ops, q, kc, vc, table, pos, window=2500)  # from key 6500 of the last
    attend(ops, q, kc, vc, table, pos, window=4100)
    missing = table.copy()
    missing[:, 270] = 10 ** 6   # keys 4320 .. 4335
    got = ops.quant_paged_attention(q, kc, vc, cuda(missing), cuda(np.array(pos)))
    with pytest.raises(SandyError, match="block id outside the pool"):
        ops.check_device_errors()
    # as if those keys were not there: the same tables without the page
    for b in (4, 5):
        less = np.delete(table[b:b + 1], 270, 1)
        want, slack = R.attention(f64(q[b:b + 1]), R.Cache.of(kc), R.Cache.of(vc), less, [pos[b] - 16], [T], 0, -1.0)
        R.assert_attention(got[b:b + 1], want, slack, f"sequence {b}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [2, 3])
def test_few_queries_of_many_sequences(ops, T, dtype):
    """Batches on both sides of the choice between the kernels: one and two 16-row tiles
    a kv head, mixed contexts."""
    r = rng(T)
    ctx = [4500 if b == 40 else int(r.integers(T, 300)) for b in range(96)]
    table, kc, vc = filled(ops, r, ctx, 4, 64, 16, "e4m3", 5)
    q = from_f32(r.standard_normal((96, 32, T, 64)).astype(np.float32), dtype)
    attend(ops, q, kc, vc, table, [c - T for c in ctx])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,dim,rows,shift,steps", [
    (2, 100, 16, 0, [3, 20, 40]), (1, 36, 128, 0, [40, 100, 200]), (2, 128, 32, 1, [5, 30, 60]),
    (1, 256, 64, 0, [20, 64, 100]), (2, 256, 128, 0, [70, 128, 100])])
def test_appends_of_large_blocks(ops, heads, dim, rows, shift, steps, fmt, dtype):
    """Blocks of more pieces than a workgroup's registers hold, by element and by
    eight, written in several calls whose rows get louder: kept rows are rounded
    again.  (`shift`: rows that are not 16-byte aligned.)"""
    r = rng(dim + rows)
    B = 2
    table, pages = make_table(r, [sum(steps) + 7] * B, rows)
    kc, vc = empty(ops, pages, heads, rows, dim, fmt, 1), empty(ops, pages, heads, rows, dim, fmt, 2)
    kr, vr = R.Cache.of(kc), R.Cache.of(vc)
    pos = np.array([0, 7])
    for i, n in enumerate(steps):
        k, v = (torch.zeros(B, heads, n, dim + shift, dtype=dtype, device="cuda")[..., shift:].copy_(
            loud_rows(r, (B, heads, n, dim), dtype) * 3.0 ** i) for _ in range(2))
        ops.quant_paged_append(k, v, kc, vc, cuda(table), cuda(pos))
        kr.append(f64(k), table, pos, [n] * B)
        vr.append(f64(v), table, pos, [n] * B)
        pos = pos + n
        assert_same(kc, kr, f"k, step {i}")
        assert_same(vc, vr, f"v, step {i}")
    ops.check_device_errors()


# ------------------------------------------------------------------ switches and streams
def test_switches_between_calls(ops, monkeypatch):
    """A switch that changes a call's workspace, set after a call of the same sizes."""
    r = rng(41)
    table, kc, vc = filled(ops, r, [2000, 900], 2, 64, 16, "int8", 3)
    q = from_f32(r.standard_normal((2, 8, 3, 64)).astype(np.float32), BF16)
    ops._quant_workspace.cache_clear()
    for name, value in (("SANDY_QUANT_SPLITS", "2"), ("SANDY_QUANT_SPLITS", "15"), ("SANDY_QUANT_PROMPT_WGS", "1"),
                        ("SANDY_QUANT_SPLITS", "1"), ("SANDY_QUANT_PROMPT_WGS", "100000"), ("SANDY_QUANT_SPLITS", "4")):
        monkeypatch.setenv(name, value)
        attend(ops, q, kc, vc, table, [1997, 897])


def split_call(ops, T=1, dim=64):
    r = rng(43)
    table, kc, vc = filled(ops, r, [6000, 2000], 4, dim, 16, "int8", 3)
    q = from_f32(r.standard_normal((2, 32, T, dim)).astype(np.float32), BF16)
    args = (q, kc, vc, cuda(table), cuda(np.array([6000 - T, 2000 - T])))
    want, slack = R.attention(f64(q), R.Cache.of(kc), R.Cache.of(vc), table, [6000 - T, 2000 - T], [T, T], 0, -1.0)
    return args, want, slack


@pytest.mark.parametrize("splits", [2, 16, 17, 40, 255])
@pytest.mark.parametrize("T,dim,dtype", [(1, 64, BF16), (3, 96, F32), (2, 128, BF16), (1, 256, F32)])
def test_both_joins_give_the_same_bits(ops, monkeypatch, T, dim, dtype, splits):
    r = rng(splits + dim)
    table, kc, vc = filled(ops, r, [9000, 3, 1100], 2, dim, 16, "int8", 5)
    for at in (5, 300, 301):
        vc.scales[int(table[0, at]), 0] = 248
    q = from_f32(r.standard_normal((3, 8, T, dim)).astype(np.float32), dtype)
    args = (q, kc, vc, cuda(table), cuda(np.array([9000 - T, 0, 1100 - T])))
    monkeypatch.setenv("SANDY_QUANT_SPLITS", str(splits))
    last = ops.quant_paged_attention(*args)
    monkeypatch.setenv("SANDY_QUANT_MERGE_KERNEL", "1")
    assert torch.equal(ops.quant_paged_attention(*args), last)
    ops.check_device_errors()


def test_graphs_without_counters(ops, monkeypatch):
    """Captured calls past the counters that the library has for them, beside one that
    has its own and eager calls; every replay checked."""
    args, want, slack = split_call(ops)
    first = ops.quant_paged_attention(*args)
    R.assert_attention(first, want, slack, "eager")
    graphs = []
    for limit in (None, "0", "7", None):
        if limit is not None:
            monkeypatch.setenv("SANDY_QUANT_CAPTURE_WORDS", limit)
        else:
            monkeypatch.delenv("SANDY_QUANT_CAPTURE_WORDS", raising=False)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = ops.quant_paged_attention(*args)
        graphs.append((graph, out, limit))
    for _ in range(4):
        for graph, out, limit in graphs:
            out.zero_()
            graph.replay()
            assert torch.equal(ops.quant_paged_attention(*args), first)
            torch.cuda.synchronize()
            assert torch.equal(out, first), f"captured with {limit}"
    ops.check_device_errors()


def test_streams_that_come_and_go(ops):
    """Streams destroyed one after the other, whose handles may be given again."""
    from sandyrt_amd import _lib
    hip = _lib.lib()
    hip.hipStreamCreate.restype = hip.hipStreamDestroy.restype = ctypes.c_int
    args, want, slack = split_call(ops)
    first = ops.quant_paged_attention(*args)
    R.assert_attention(first, want, slack)
    torch.cuda.synchronize()
    for i in range(80):
        handle = ctypes.c_void_p()
        assert hip.hipStreamCreate(ctypes.byref(handle)) == 0
        with torch.cuda.stream(torch.cuda.ExternalStream(handle.value)):
            for _ in range(2):
                out = ops.quant_paged_attention(*args)
            torch.cuda.current_stream().synchronize()
        assert hip.hipStreamDestroy(handle) == 0
        assert torch.equal(out, first), f"stream {i}"
    assert torch.equal(ops.quant_paged_attention(*args), first)
    ops.check_device_errors()
