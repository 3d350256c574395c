"""The quantised paged K/V cache on the GPU against numpy in 64 bits: payloads
and scales bit for bit after any appends, rows read back exactly, attention
within its type's rounding and the error bound of fp32 sums."""
import numpy as np
import pytest
import torch

from tests import quant_reference as R
from tests.helpers import from_f32, rng

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
WEIGHT = 2.0 ** -15


@pytest.fixture(scope="module")
def ops():
    from sandyrt_amd import ops
    return ops


def cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def empty(ops, pages, heads, rows, dim, fmt, seed=0):
    """A cache whose bytes are what earlier use left: payloads of any value (no
    NaN byte), scales of any exponent."""
    r = rng(seed)
    c = ops.QuantPagedCache.empty(pages, heads, rows, dim, fmt)
    junk = r.integers(0, 0x7f, (pages, heads, rows, dim), dtype=np.uint8) | (r.integers(0, 2, (pages, heads, rows, dim), dtype=np.uint8) << 7)
    if fmt == "int8":
        junk[junk == 0x80] = 0
    c.pool.view(torch.uint8).copy_(cuda(junk))
    c.scales.copy_(cuda(r.integers(100, 150, (pages, heads), dtype=np.uint8)))
    return c


def make_table(r, lengths, rows, spare=3):
    """Block table [B, width] of distinct pages; unused entries name none."""
    need = [-(-n // rows) for n in lengths]
    perm = r.permutation(sum(need) + spare).astype(np.int32)
    table = np.full((len(lengths), max(max(need), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, sum(need) + spare


def f64(t):
    return t.detach().cpu().double().numpy()


def assert_same(cache, ref, what=""):
    got = R.Cache.of(cache)
    np.testing.assert_array_equal(got.code, ref.code, err_msg=f"{what}: scales")
    np.testing.assert_array_equal(got.payload, ref.payload, err_msg=f"{what}: payloads")


def loud_rows(r, shape, dtype):
    """Rows of very different loudness, [B, heads, T, D]."""
    x = r.standard_normal(shape) * np.exp(r.standard_normal(shape[:3] + (1,)) * 2)
    return from_f32(x.astype(np.float32), dtype)


# ------------------------------------------------------------------ append and read
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,dim,rows", [(4, 64, 16), (2, 256, 16), (3, 80, 32), (2, 128, 128), (2, 5, 4), (1, 64, 1), (2, 24, 2)])
def test_appends_of_any_length(ops, heads, dim, rows, fmt, dtype):
    """Chunk after chunk of ragged lengths, single rows among them, every page
    filled in several pieces; rows behind a sequence's last one stay as they were."""
    r = rng(heads * dim + rows)
    B, steps = 3, [7, 1, 1, 30, 1, 2, 41, 1]
    counts = [[min(n, max(0, n - (b * 5) % (n + 1))) for b in range(B)] for n in steps]
    total = [sum(c[b] for c in counts) for b in range(B)]
    table, pages = make_table(r, [t + 1 for t in total], rows)
    kc, vc = empty(ops, pages, heads, rows, dim, fmt, 1), empty(ops, pages, heads, rows, dim, fmt, 2)
    kr, vr = R.Cache.of(kc), R.Cache.of(vc)
    pos = np.zeros(B, np.int64)
    for n, cnt in zip(steps, counts):
        # K and V as neighbouring heads of one projection's rows
        kv = loud_rows(r, (B, n, 2 * heads, dim), dtype).transpose(1, 2)
        k, v = kv[:, :heads], kv[:, heads:]
        ops.quant_paged_append(k, v, kc, vc, cuda(table), cuda(pos), counts=cuda(np.array(cnt), torch.int32))
        kr.append(f64(k), table, pos, cnt)
        vr.append(f64(v), table, pos, cnt)
        pos += cnt
    ops.check_device_errors()
    assert_same(kc, kr, "k")
    assert_same(vc, vr, "v")
    for out in (BF16, F32):
        first, n = np.array([0, 3, 1]), 60
        got_k, got_v = ops.quant_paged_read(kc, vc, cuda(table), cuda(first, torch.int32), n,
                                            counts=cuda(np.minimum(n, pos - first)), dtype=out)
        for got, ref in ((got_k, kr), (got_v, vr)):
            for b in range(B):
                m = int(min(n, pos[b] - first[b]))
                np.testing.assert_array_equal(f64(got[b, :, :m]), ref.rows_of(table[b], first[b], m))
                assert not got[b, :, m:].any()
    ops.check_device_errors()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_values(ops, fmt):
    """Borders of the scale, zeros, subnormals and the largest numbers; K alone;
    element-strided rows."""
    top = R.LARGEST[fmt]
    rows = [np.zeros(8), np.full(8, top), np.full(8, np.nextafter(np.float32(top), np.float32(1e9))), np.full(8, 1e-45),
            np.full(8, 3.4e38), np.array([1e-40, 2.0 ** -126, -2.0 ** -120, 0, 0, 0, 0, 0]), np.full(8, -top * 2.0 ** -126),
            np.linspace(-1, 1, 8), np.array([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, top, 3.5])]
    x = np.stack(rows).astype(np.float32)[None, None]  # [1, 1, 9, 8]
    table = np.arange(12, dtype=np.int32)[None]
    for strided in (False, True):
        t = cuda(x)
        if strided:
            t = torch.stack([t, t + 1], -1)[..., 0]
        for rows_per_page in (1, 16):
            c = empty(ops, 12, 1, rows_per_page, 8, fmt, 3)
            ref = R.Cache.of(c)
            ops.quant_paged_append(t, None, c, None, cuda(table), cuda(np.zeros(1, np.int64)))
            ref.append(x.astype(np.float64), table, [0], [9])
            assert_same(c, ref)
            got, none = ops.quant_paged_read(c, None, cuda(table), cuda(np.zeros(1, np.int64)), 9, dtype=F32)
            assert none is None
            np.testing.assert_array_equal(f64(got[0]), ref.rows_of(table[0], 0, 9))
    ops.check_device_errors()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 7])
def test_append_not_finite(ops, fmt, dim):
    """A block given an infinity or NaN reads as NaN until it starts anew; its
    neighbours do not."""
    c = empty(ops, 3, 2, 4, dim, fmt)
    ref = R.Cache.of(c)
    table = np.array([[2, 0, 1]], np.int32)
    x = rng(5).standard_normal((1, 2, 10, dim))
    x[0, 1, 1, 3], x[0, 0, 6, 0] = np.inf, np.nan

    def put(rows, at):
        t = from_f32(rows.astype(np.float32), BF16)
        ops.quant_paged_append(t, None, c, None, cuda(table), cuda(np.array([at])))
        ref.append(f64(t), table, [at], [rows.shape[2]])
        assert_same(c, ref, f"rows from {at}")

    put(x, 0)
    assert (ref.code == 255).sum() == 2
    put(x[:, :, :1], 10)
    put(x[:, :, 2:4], 3)   # the block with the infinity: still NaN
    got, _ = ops.quant_paged_read(c, None, cuda(table), cuda(np.zeros(1, np.int64)), 11, dtype=F32)
    np.testing.assert_array_equal(f64(got[0]), ref.rows_of(table[0], 0, 11))
    put(x[:, :, 2:4], 0)   # anew
    assert ref.code[2, 1] != 255
    ops.check_device_errors()


def test_append_records_what_it_cannot_write(ops):
    from sandyrt_amd._lib import SandyError
    r = rng(9)
    table = np.array([[0, 1], [2, 9], [3, 4], [5, 6], [7, 8]], np.int32)
    x = loud_rows(r, (5, 2, 6, 64), BF16)
    for bad, message, pos, counts in [
            ("row", "rows outside the block table", [0, -1, 27, 2 ** 40, 8], [6, 6, 6, 6, 6]),
            ("block", "block id outside the pool", [0, 13, 8, 8, 8], [6] * 5),
            ("count", "counts out of range", [0, 8, 8, 8, 8], [6, 6, 7, -1, 0])]:
        c = empty(ops, 9, 2, 16, 64, "int8", 4)
        ref = R.Cache.of(c)
        ops.quant_paged_append(x, None, c, None, cuda(table), cuda(np.array(pos)), counts=cuda(np.array(counts)))
        with pytest.raises(SandyError, match=message):
            ops.check_device_errors()
        kept = {"row": [0, 4], "block": [0, 2, 3, 4], "count": [0, 1, 2]}[bad]
        for b in kept:
            ref.append(f64(x)[b:b + 1], table[b:b + 1], pos[b:b + 1], [6])
        if bad == "block":  # the page that is there takes its rows
            ref.append(f64(x)[1:2], table[1:2], [13], [3])
        assert_same(c, ref, bad)
    c = empty(ops, 9, 2, 16, 64, "int8", 4)
    got, _ = ops.quant_paged_read(c, None, cuda(table), cuda(np.array([30, -2, 0, 0, 0])), 4)
    with pytest.raises(SandyError, match="rows outside the block table"):
        ops.check_device_errors()
    assert not got[0, :, 2:].any() and not got[1, :, :2].any()
    got, _ = ops.quant_paged_read(c, None, cuda(table), cuda(np.full(5, 14)), 4)
    with pytest.raises(SandyError, match="block id outside the pool"):
        ops.check_device_errors()
    assert not got[1, :, 2:].any() and got[1, :, :2].any()


def test_empty_calls(ops):
    c = empty(ops, 4, 2, 16, 64, "int8")
    before = c.pool.clone()
    table, pos = torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    x = torch.zeros(0, 2, 3, 64, device="cuda")
    ops.quant_paged_append(x, x, c, empty(ops, 4, 2, 16, 64, "int8"), table, pos)
    assert ops.quant_paged_attention(x, c, c, table, pos).shape == x.shape
    table, pos = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    x = torch.zeros(2, 2, 0, 64, device="cuda")
    ops.quant_paged_append(x, None, c, None, table, pos)
    assert ops.quant_paged_read(c, None, table, pos, 0)[0].shape == (2, 2, 0, 64)
    assert ops.quant_paged_attention(x, c, c, table, pos).shape == x.shape
    assert torch.equal(before, c.pool)
    # a table without pages: no key for any query
    table = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    out = ops.quant_paged_attention(torch.ones(2, 4, 3, 64, device="cuda"), c, c, table, pos, out=torch.full((2, 4, 3, 64), 7.0, device="cuda"))
    assert not out.any()
    ops.check_device_errors()


# ------------------------------------------------------------------ attention
def filled(ops, r, lengths, heads, dim, rows, fmt, seed, width=0):
    """Two caches of random blocks (scales of a few octaves), a block table."""
    table, pages = make_table(r, lengths, rows)
    if width:
        table = np.concatenate([table, np.full((len(lengths), width - table.shape[1]), -1, np.int32)], 1)
    caches = []
    for i in range(2):
        c = empty(ops, pages, heads, rows, dim, fmt, seed + i)
        if fmt == "e4m3":  # bit patterns spread over all exponents: most are tiny
            c.pool.copy_((torch.randn(c.pool.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed + i)) * 100)
                         .clamp(-448, 448).to(torch.float8_e4m3fn))
        base = 120 if fmt == "int8" else 118
        c.scales.copy_(cuda(r.integers(base - 2, base + 2, c.scales.shape, dtype=np.uint8)))
        caches.append(c)
    return table, caches[0], caches[1]


def check(ops, q, kc, vc, table, pos, counts=None, window=0, scale=-1.0, what=""):
    out = torch.full(q.shape, 99.0, dtype=q.dtype, device="cuda")
    got = ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array(pos)),
                                    counts=None if counts is None else cuda(np.array(counts)), window=window, scale=scale,
                                    out=out)
    ops.check_device_errors()
    assert got is out
    cnt = counts if counts is not None else [q.shape[2]] * q.shape[0]
    # bf16: weights may be two bf16 numbers, the first cut (what is left is below
    # 2^-7 of the weight), the second rounded (2^-8 of that)
    want, slack = R.attention(f64(q), R.Cache.of(kc), R.Cache.of(vc), table, pos, cnt, window, scale,
                              WEIGHT if q.dtype == BF16 else 0.0)
    R.assert_attention(got, want, slack, what)
    return got


CTX = [1, 2, 15, 16, 17, 31, 33, 64, 129, 300, 513]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hq,heads,dim,rows", [(32, 4, 64, 16), (8, 2, 256, 16), (16, 2, 128, 32), (12, 12, 64, 16),
                                               (10, 2, 96, 64), (6, 3, 80, 16), (32, 1, 64, 16), (5, 1, 112, 128),
                                               (4, 2, 64, 2), (3, 3, 20, 16), (2, 1, 320, 16), (34, 2, 192, 16)])
def test_decode(ops, hq, heads, dim, rows, fmt, dtype):
    r = rng(hq + dim)
    table, kc, vc = filled(ops, r, CTX, heads, dim, rows, fmt, hq)
    q = from_f32(r.standard_normal((len(CTX), hq, 1, dim)).astype(np.float32), dtype)
    check(ops, q, kc, vc, table, [c - 1 for c in CTX])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [1, 7, 64, 500, 10 ** 12])
def test_decode_window(ops, window, dtype):
    """Pages before every window have left the table."""
    r = rng(window % 1000)
    ctx = [5, 100, 700, 1200]
    table, kc, vc = filled(ops, r, ctx, 2, 64, 16, "int8", 3)
    for b, c in enumerate(ctx):
        table[b, :max(0, (c - window) // 16)] = -1
    q = from_f32(r.standard_normal((4, 16, 1, 64)).astype(np.float32), dtype)
    check(ops, q, kc, vc, table, [c - 1 for c in ctx], window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_decode_long(ops, fmt, dtype):
    """Contexts of many splits beside short ones, under a table wide enough for more."""
    r = rng(11)
    ctx = [9000, 1, 33, 4097]
    table, kc, vc = filled(ops, r, ctx, 2, 64, 16, fmt, 5, width=700)
    q = from_f32(2 * r.standard_normal((4, 8, 1, 64)).astype(np.float32), dtype)
    check(ops, q, kc, vc, table, [c - 1 for c in ctx])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hq,heads,dim,rows,T,window", [
    (32, 4, 64, 16, 2, 0), (32, 4, 64, 16, 37, 0), (8, 2, 256, 16, 21, 16), (16, 2, 128, 32, 70, 50), (12, 12, 64, 16, 9, 3),
    (10, 2, 96, 64, 33, 0), (6, 3, 80, 16, 65, 40), (4, 2, 64, 2, 5, 0), (2, 1, 20, 16, 6, 4), (4, 4, 64, 16, 130, 0)])
def test_chunks(ops, hq, heads, dim, rows, T, window, fmt, dtype):
    """Ragged chunks after contexts of several lengths; one sequence has no query."""
    r = rng(T + dim)
    pos, counts = [0, 3, 100, 257, 40], [T, max(1, T - 5), T, (T + 1) // 2, 0]
    table, kc, vc = filled(ops, r, [max(p + c, 1) for p, c in zip(pos, counts)], heads, dim, rows, fmt, T)
    # queries as the projection leaves them
    q = from_f32(r.standard_normal((5, T, hq, dim)).astype(np.float32), dtype).transpose(1, 2)
    check(ops, q, kc, vc, table, pos, counts, window)


@pytest.mark.parametrize("hq,heads,dim", [(32, 4, 64), (16, 2, 128), (8, 2, 256)])
@pytest.mark.parametrize("fmt,dtype", [("int8", BF16), ("e4m3", F32), ("e4m3", BF16)])
def test_long_chunks(ops, hq, heads, dim, fmt, dtype):
    """Enough rows for the prompt tiles, from the first key and behind a context."""
    r = rng(dim)
    T = 300
    table, kc, vc = filled(ops, r, [T, 777], heads, dim, 16, fmt, 3)
    q = from_f32(r.standard_normal((2, hq, T, dim)).astype(np.float32), dtype)
    check(ops, q, kc, vc, table, [0, 777 - T], scale=0.07)
    check(ops, q, kc, vc, table, [0, 777 - T], window=100)


def test_attention_strides_and_outputs(ops):
    """Rows that are not 16-byte aligned, element strides, an output view, out = q."""
    r = rng(21)
    table, kc, vc = filled(ops, r, [40, 70], 2, 64, 16, "int8", 3)
    x = r.standard_normal((2, 4, 3, 64)).astype(np.float32)
    pos = [37, 67]
    for dtype in (BF16, F32):
        want = check(ops, from_f32(x, dtype), kc, vc, table, pos)
        wide = torch.zeros(2, 4, 3, 67, dtype=dtype, device="cuda")
        wide[..., 1:65] = from_f32(x, dtype)
        off = check(ops, wide[..., 1:65], kc, vc, table, pos)
        every = torch.zeros(2, 4, 3, 128, dtype=dtype, device="cuda")
        every[..., ::2] = from_f32(x, dtype)
        check(ops, every[..., ::2], kc, vc, table, pos)
        out = torch.full((2, 3, 4, 70), 5.0, dtype=dtype, device="cuda")
        view = out.transpose(1, 2)[..., 3:67]
        ops.quant_paged_attention(from_f32(x, dtype), kc, vc, cuda(table), cuda(np.array(pos)), out=view)
        assert (out[..., :3] == 5).all() and (out[..., 67:] == 5).all()
        np.testing.assert_allclose(f64(view), f64(want), rtol=2 ** -7, atol=1e-6)
        q = from_f32(x, dtype)
        ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array(pos)), out=q)
        assert torch.equal(q, want)
        del off
    ops.check_device_errors()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("T,dim", [(1, 64), (5, 64), (40, 128), (4, 36)])
def test_not_finite_reaches_its_readers_only(ops, fmt, dtype, T, dim):
    """A NaN block, a NaN query and bytes behind the last key: only the queries
    that see them are NaN."""
    r = rng(31)
    n = 90
    table, kc, vc = filled(ops, r, [n, n], 2, dim, 16, fmt, 3)
    for c in (kc, vc):  # bytes behind the last row: NaN in e4m3
        c.pool.view(torch.uint8)[int(table[0, 5]), :, n - 80:] = 0x7f
        c.pool.view(torch.uint8)[int(table[1, 5]), :, n - 80:] = 0xff
        c.scales[int(table[1, 5])] = 120
    q = from_f32(r.standard_normal((2, 4, T, dim)).astype(np.float32), dtype)
    pos = [n - T, n - T]
    clean = check(ops, q, kc, vc, table, pos)
    assert torch.isfinite(clean).all()
    kc.scales[int(table[0, 4]), 1] = 255   # keys 64..79 of the second kv head
    vc.scales[int(table[1, 0]), 0] = 255   # keys 0..15 of the first
    got = check(ops, q, kc, vc, table, pos)
    assert torch.equal(torch.isnan(got[0, :2]), torch.zeros_like(got[0, :2], dtype=torch.bool))
    window = 10  # the second sequence's block is out of sight; the first's may be seen by some
    check(ops, q, kc, vc, table, pos, window=window)
    q = q.clone()
    q[0, 1, T - 1, 5] = float("nan")
    want = torch.zeros_like(got, dtype=torch.bool)
    got = check(ops, q[:1], kc, vc, table[:1], pos[:1], window=window)
    want = torch.isnan(got[0, 0])
    assert not want.any() and torch.isnan(got[0, 1, T - 1]).all() and not torch.isnan(got[0, 1, :T - 1]).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("T,dim", [(1, 64), (70, 64), (33, 128), (3, 36)])
def test_blocks_of_far_scales(ops, fmt, dtype, T, dim):
    """Blocks of zeros (the smallest scale) and of very small and large numbers
    beside ordinary ones: their weights count in the sum all the same."""
    r = rng(33)
    n = 150
    table, pages = make_table(r, [n], 16)
    kc, vc = (empty(ops, pages, 2, 16, dim, fmt, i) for i in (1, 2))
    k, v = (r.standard_normal((1, 2, n, dim)) for _ in range(2))
    v[:, :, 16:32] = 0
    v[:, 0, 64:80] *= 1e-36
    v[:, 1, 80:96] *= 1e30
    k[:, :, 96:112] = 0
    k[:, :, 112:128] *= 1e-37
    k, v = (from_f32(x.astype(np.float32), dtype) for x in (k, v))
    ops.quant_paged_append(k, v, kc, vc, cuda(table), cuda(np.zeros(1, np.int64)))
    assert (vc.scales[int(table[0, 1])] == 1).all() and (kc.scales[int(table[0, 6])] == 1).all()
    q = from_f32(r.standard_normal((1, 8, T, dim)).astype(np.float32), dtype)
    check(ops, q, kc, vc, table, [n - T])


def test_attention_records(ops):
    from sandyrt_amd._lib import SandyError
    r = rng(41)
    table, kc, vc = filled(ops, r, [40, 40, 40], 2, 64, 16, "int8", 3)
    for T in (1, 20):
        q = from_f32(r.standard_normal((3, 4, T, 64)).astype(np.float32), BF16)
        good = ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array([20, 20, 20])))
        ops.check_device_errors()
        got = ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array([20, -1, 20])))
        with pytest.raises(SandyError, match="position_offsets must be non-negative"):
            ops.check_device_errors()
        assert not got[1].any() and torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
        bad = table.copy()
        bad[1, 1] = 10 ** 6
        got = ops.quant_paged_attention(q, kc, vc, cuda(bad), cuda(np.array([20, 20, 20])))
        with pytest.raises(SandyError, match="block id outside the pool"):
            ops.check_device_errors()
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2]) and torch.isfinite(got).all()
        got = ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array([20, 20, 20])), counts=cuda(np.array([T, T + 1, -3])))
        with pytest.raises(SandyError, match="counts out of range"):
            ops.check_device_errors()
        assert torch.equal(got[:2], good[:2]) and not got[2].any()
        # past the table's last key: every key it has
        check(ops, q, kc, vc, table, [20, 20, 100])


@pytest.mark.parametrize("merge_kernel", [0, 1])
@pytest.mark.parametrize("splits", [1, 2, 5, 17, 40, 256])
def test_splits(ops, monkeypatch, splits, merge_kernel):
    """Every number of splits, joined by the last workgroup (in one group of 16 or
    several) or by the merge kernel; a second call finds the counters as the first."""
    ops._quant_workspace.cache_clear()
    monkeypatch.setenv("SANDY_QUANT_SPLITS", str(splits))
    monkeypatch.setenv("SANDY_QUANT_MERGE_KERNEL", str(merge_kernel))
    r = rng(splits)
    ctx = [9000, 3, 1100, 40]
    for dim, T, dtype in ((64, 1, BF16), (256, 1, BF16), (128, 5, BF16), (64, 2, F32)):
        table, kc, vc = filled(ops, r, ctx, 2, dim, 16, "int8", 5)
        q = from_f32(r.standard_normal((4, 8, T, dim)).astype(np.float32), dtype)
        pos = [max(0, c - T) for c in ctx]
        first = check(ops, q, kc, vc, table, pos, counts=[T, min(T, 3), T, T])
        assert torch.equal(first, check(ops, q, kc, vc, table, pos, counts=[T, min(T, 3), T, T]))
    ops._quant_workspace.cache_clear()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hq,heads,dim,rows,T,window", [(32, 4, 64, 16, 37, 0), (8, 2, 256, 16, 21, 16), (16, 2, 128, 32, 70, 50),
                                                        (10, 2, 96, 64, 33, 0), (6, 3, 80, 16, 65, 40), (34, 2, 192, 16, 3, 9),
                                                        (4, 4, 64, 16, 130, 0), (3, 1, 16, 16, 11, 0)])
def test_prompt_tiles_of_short_chunks(ops, monkeypatch, hq, heads, dim, rows, T, window, fmt, dtype):
    """The prompt kernel on rows that do not fill a tile, ragged and windowed."""
    ops._quant_workspace.cache_clear()
    monkeypatch.setenv("SANDY_QUANT_PROMPT_WGS", "1")
    r = rng(T + dim)
    pos, counts = [0, 3, 100, 257, 40], [T, max(1, T - 5), T, (T + 1) // 2, 0]
    table, kc, vc = filled(ops, r, [max(p + c, 1) for p, c in zip(pos, counts)], heads, dim, rows, fmt, T)
    kc.scales[int(table[2, 1])] = 255  # keys the later queries of the third sequence see
    q = from_f32(r.standard_normal((5, T, hq, dim)).astype(np.float32), dtype).transpose(1, 2)
    check(ops, q, kc, vc, table, pos, counts, window)
    ops._quant_workspace.cache_clear()


@pytest.mark.parametrize("T,dim", [(1, 64), (300, 64), (3, 128), (2, 36)])
def test_far_positions_and_windows(ops, T, dim):
    """Positions past the block table see what it covers, windows of any size."""
    r = rng(47)
    table, kc, vc = filled(ops, r, [64, 64], 2, dim, 16, "int8", 3)
    q = from_f32(r.standard_normal((2, 8, T, dim)).astype(np.float32), BF16)
    far = 2 ** 63 - 1
    whole = check(ops, q, kc, vc, table, [63, 64])
    for pos, window in (([far, far], far), ([far, 70], 0), ([2 ** 31, 2 ** 40], 2 ** 40 + 1), ([63, 64], far), ([70, 64], 2 ** 31)):
        got = ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array(pos)), window=window)
        ops.check_device_errors()
        for b in range(2):
            for i in sorted({0, T // 2, min(63, T - 1), min(64, T - 1), T - 1}):
                last = min(pos[b] + i, 63)
                first = max(0, pos[b] + i + 1 - window) if window else 0
                if first > last:
                    assert not got[b, :, i].any()
                    continue
                want, slack = R.attention(f64(q)[b:b + 1, :, i:i + 1], R.Cache.of(kc), R.Cache.of(vc), table[b:b + 1], [last], [1],
                                          last - first + 1, -1.0, WEIGHT)
                R.assert_attention(got[b:b + 1, :, i:i + 1], want, slack, f"{pos} {window} {b} {i}")
        if pos == [63, 64]:
            assert torch.equal(got, whole)
    # windows that leave the table nothing
    got = ops.quant_paged_attention(q, kc, vc, cuda(table), cuda(np.array([200, far])), window=100)
    assert not got.any()
    ops.check_device_errors()


@pytest.mark.parametrize("merge_kernel", [0, 1])
@pytest.mark.parametrize("hq,heads,dim,T,dtype", [(8, 2, 64, 1, BF16), (8, 2, 128, 1, F32), (4, 2, 256, 1, BF16), (16, 2, 64, 2, BF16),
                                                  (10, 2, 96, 4, F32)])
def test_splits_of_mixed_contexts(ops, monkeypatch, hq, heads, dim, T, dtype, merge_kernel):
    """More row tiles than half the CUs: sequences of a piece each beside long ones
    that take several, at the lengths where their number changes."""
    monkeypatch.setenv("SANDY_QUANT_MERGE_KERNEL", str(merge_kernel))
    r = rng(dim + T)
    long = [1024, 1025, 2048, 2049, 2080, 3073, 4097, 6000]
    ctx = [long[b // 9] if b % 9 == 0 else int(r.integers(T, 400)) for b in range(72)]
    table, kc, vc = filled(ops, r, ctx, heads, dim, 16, "e4m3", 5)
    q = from_f32(r.standard_normal((72, hq, T, dim)).astype(np.float32), dtype)
    pos = [c - T for c in ctx]
    first = check(ops, q, kc, vc, table, pos)
    assert torch.equal(first, check(ops, q, kc, vc, table, pos))
    check(ops, q, kc, vc, table, pos, window=2500)


def test_many_sequences(ops):
    """More row tiles than 2^16."""
    r = rng(91)
    B, hq, heads, dim, T = 9000, 16, 8, 64, 9
    table, kc, vc = filled(ops, r, [T] * 16, heads, dim, 16, "e4m3", 3)
    gt = cuda(table).repeat(B // 16 + 1, 1)[:B].contiguous()
    q = torch.randn(B, hq, T, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF16)
    got = ops.quant_paged_attention(q, kc, vc, gt, torch.zeros(B, dtype=torch.int32, device="cuda"))
    ops.check_device_errors()
    pick = [0, 15, 4097, B - 1]
    want, slack = R.attention(f64(q[pick]), R.Cache.of(kc), R.Cache.of(vc), table[[b % 16 for b in pick]], [0] * 4, [T] * 4, 0, -1.0, WEIGHT)
    R.assert_attention(got[pick], want, slack)


def test_deterministic(ops):
    r = rng(51)
    table, kc, vc = filled(ops, r, [4000, 900], 4, 64, 16, "e4m3", 3)
    for T in (1, 64):
        q = from_f32(r.standard_normal((2, 32, T, 64)).astype(np.float32), BF16)
        args = (q, kc, vc, cuda(table), cuda(np.array([4000 - T, 900 - T])))
        first = ops.quant_paged_attention(*args)
        for _ in range(5):
            assert torch.equal(first, ops.quant_paged_attention(*args))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("fmt,dtype", [("int8", BF16), ("e4m3", F32)])
def test_prompt_then_steps_in_a_graph(ops, fmt, dtype):
    """A ragged prompt, then decode steps replayed from one captured graph whose
    positions advance on the device; every step against the reference."""
    r = rng(61)
    B, heads, hq, dim, rows, steps = 3, 2, 8, 64, 16, 20
    counts = [50, 1, 33]
    table, pages = make_table(r, [c + steps + 2 for c in counts], rows)
    kc, vc = (empty(ops, pages, heads, rows, dim, fmt, i) for i in (1, 2))
    kr, vr = R.Cache.of(kc), R.Cache.of(vc)
    T = max(counts)
    gt, pos = cuda(table), torch.zeros(B, dtype=torch.int64, device="cuda")
    k, v, q = (from_f32(r.standard_normal((B, h, T, dim)).astype(np.float32), dtype) for h in (heads, heads, hq))
    cnt = cuda(np.array(counts))
    ops.quant_paged_append(k, v, kc, vc, gt, pos, counts=cnt)
    out = ops.quant_paged_attention(q, kc, vc, gt, pos, counts=cnt)
    kr.append(f64(k), table, [0] * B, counts)
    vr.append(f64(v), table, [0] * B, counts)
    weight = WEIGHT if dtype == BF16 else 0.0
    R.assert_attention(out, *R.attention(f64(q), kr, vr, table, [0] * B, counts, 0, -1.0, weight), "prompt")
    pos.copy_(cnt)

    k1, v1, q1 = (torch.zeros(B, h, 1, dim, dtype=dtype, device="cuda") for h in (heads, heads, hq))
    one = torch.ones_like(pos)

    def step():
        ops.quant_paged_append(k1, v1, kc, vc, gt, pos)
        o = ops.quant_paged_attention(q1, kc, vc, gt, pos)
        pos.add_(one)
        return o

    at = list(counts)
    graph = torch.cuda.CUDAGraph()
    for i in range(steps):
        for t in (k1, v1, q1):
            t.copy_(from_f32((r.standard_normal(t.shape) * 1.3 ** (i % 7)).astype(np.float32), dtype))
        if i == 1:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                out = step()
        if i == 0:
            out = step()
        else:
            graph.replay()
        kr.append(f64(k1), table, at, [1] * B)
        vr.append(f64(v1), table, at, [1] * B)
        R.assert_attention(out, *R.attention(f64(q1), kr, vr, table, at, [1] * B, 0, -1.0, weight), f"step {i}")
        at = [a + 1 for a in at]
    ops.check_device_errors()
    assert_same(kc, kr)
    assert_same(vc, vr)


def test_two_graphs_and_streams(ops):
    """Two captured steps replayed at once on two streams share no memory."""
    r = rng(71)
    cases = []
    for n in (6000, 5000):
        table, kc, vc = filled(ops, r, [n, n // 3], 4, 64, 16, "int8", n)
        q = from_f32(r.standard_normal((2, 32, 1, 64)).astype(np.float32), BF16)
        args = (q, kc, vc, cuda(table), cuda(np.array([n - 1, n // 3 - 1])))
        want = ops.quant_paged_attention(*args)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = ops.quant_paged_attention(*args)
        cases.append((args, want, stream, graph, out))
    for _ in range(10):
        for args, want, stream, graph, out in cases:
            out.zero_()
        torch.cuda.synchronize()
        eager = []
        for args, want, stream, graph, out in cases:
            with torch.cuda.stream(stream):
                graph.replay()
                eager.append(ops.quant_paged_attention(*args))
        torch.cuda.synchronize()
        for (args, want, stream, graph, out), e in zip(cases, eager):
            assert torch.equal(out, want) and torch.equal(e, want)


def test_offsets_past_32_bits(ops):
    """Pages beyond 4 GiB of a pool."""
    heads, rows, dim = 8, 64, 256
    pages = (1 << 32) // (heads * rows * dim) + 40
    c = [ops.QuantPagedCache(torch.empty(pages, heads, rows, dim, dtype=torch.int8, device="cuda"),
                             torch.empty(pages, heads, dtype=torch.uint8, device="cuda")) for _ in range(2)]
    r = rng(81)
    table = np.array([[pages - 1, 3, pages - 7, pages - 30]], np.int32)
    n = 200
    k, v = (loud_rows(r, (1, heads, n, dim), BF16) for _ in range(2))
    pos = cuda(np.zeros(1, np.int64))
    ops.quant_paged_append(k, v, *c, cuda(table), pos)
    refs = []
    for x in (k, v):
        ref = R.Cache(4, heads, rows, dim, "int8")
        ref.append(f64(x), [[0, 1, 2, 3]], [0], [n])
        refs.append(ref)
    for got, ref in zip(ops.quant_paged_read(*c, cuda(table), pos, n, dtype=F32), refs):
        np.testing.assert_array_equal(f64(got[0]), ref.rows_of([0, 1, 2, 3], 0, n))
    for T in (1, 24):
        q = from_f32(r.standard_normal((1, 16, T, dim)).astype(np.float32), BF16)
        got = ops.quant_paged_attention(q, *c, cuda(table), cuda(np.array([n - T])))
        R.assert_attention(got, *R.attention(f64(q), *refs, [[0, 1, 2, 3]], [n - T], [T], 0, -1.0, WEIGHT))
    ops.check_device_errors()
