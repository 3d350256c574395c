"""What the products of matrices in 8 bits promise of NaN, of scale bytes near both ends and of their sums, for either output
type in every kernel form, dense and by expert."""
import numpy as np
import pytest
import torch

from sandyrt_amd import ops
from tests import block_quant_reference as R
from tests.test_gpu_block_quant import NAN8, f64, grouped, offsets_of, product, same

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]
K = 128 * 9 + 44  # blocks of every group of waves, and a short last one
forms = pytest.mark.parametrize("form", [None, *range(9)])  # as chosen; the stream, the tile forms


@pytest.fixture(autouse=True)
def _form(request, monkeypatch):
    form = request.node.callspec.params.get("form")
    if form is not None:
        monkeypatch.setenv("SANDY_QUANT_FORM", str(form))


def spoil_rows(x):
    """NaN by scale byte or payload in the first, a late and the short last block; -> rows that become NaN."""
    last = x.scales.shape[1] - 1
    bits = x.payload.view(torch.uint8)
    for row, block in ((1, last), (2, 7), (3, 0), (4, 5)):
        x.scales[row, block] = 255
        if row % 2:  # as block_quant leaves such a block
            bits[row, 128 * block:128 * (block + 1)] = 0
    bits[5, 5], bits[6, K - 1], bits[7, 128 * 8] = NAN8, NAN8 | 0x80, NAN8
    return [1, 2, 3, 4, 5, 6, 7]


@forms
@pytest.mark.parametrize("dtype", TYPES)
def test_nan_of_rows_and_weights(form, dtype):
    rng = np.random.default_rng(1)
    x, w, each = R.whole(rng, (70, K), 1), R.whole(rng, (300, K), 128), R.whole(rng, (300, K), 1)
    want = product(x, w)
    rows = spoil_rows(x)
    w.scales[1, 9] = 255  # weight rows 128 .. 255
    each.scales[9, 6] = each.scales[201, 9] = 255
    each.payload.view(torch.uint8)[40, 700] = NAN8
    lost = product(x, w)
    assert np.isnan(lost[rows]).all() and np.isnan(lost[:, 128:256]).all() and np.isnan(lost).sum() == 70 * 128 + len(rows) * 172
    keep = ~np.isnan(lost)
    np.testing.assert_array_equal(lost[keep], want[keep])
    same(ops.quant_linear(x, w, dtype=dtype), lost, dtype)
    lost = product(x, each)
    assert np.isnan(lost[0]).sum() == 3
    same(ops.quant_linear(x, each, dtype=dtype), lost, dtype)


@pytest.mark.parametrize("rows", [1, 3, 17, 70, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_nan_of_quantised_rows_that_are_not_finite(rows, dtype):
    """block_quant marks their blocks 255 over payloads 0."""
    rng = np.random.default_rng(rows)
    v = torch.from_numpy(rng.integers(-8, 9, (rows, K))).float().cuda()
    v[0, K - 1] = float("inf")
    v[-1, 300] = float("nan")
    w = R.whole(rng, (200, K), 128)
    x = ops.block_quant(v)
    assert x.scales[0, 9] == 255 and x.scales[-1, 2] == 255
    want = product(x, w)
    assert np.isnan(want[[0, -1]]).all() and not np.isnan(want[1:-1]).any()
    same(ops.quant_linear(x, w, dtype=dtype), want, dtype)
    m = torch.from_numpy(rng.integers(-8, 9, (200, K))).float().cuda()
    m[150, 1000] = -float("inf")
    q = ops.block_quant(m, 128)
    want = product(x, q)
    assert np.isnan(want[:, 128:]).all()
    same(ops.quant_linear(x, q, dtype=dtype), want, dtype)


@forms
@pytest.mark.parametrize("dtype", TYPES)
def test_nan_by_expert(form, dtype):
    rng = np.random.default_rng(2)
    counts = [3, 0, 70, 1, 9]
    x, w = R.whole(rng, (sum(counts), K), 1), R.whole(rng, (5, 300, K), 128)
    rows = spoil_rows(x)
    w.scales[2, 2, 9] = w.scales[1] = w.scales[3, 0, 4] = 255
    want = grouped(x, counts, w)
    assert np.isnan(want[rows]).all() and np.isnan(want[3:73, 256:]).all() and np.isnan(want[73, :128]).all()
    assert np.isnan(want).sum() == len(rows) * 300 + 65 * 44 + 128  # 5 of the 70 rows whose last 44 columns are NaN are lost as a whole
    same(ops.quant_moe_matmul(x, offsets_of(counts), w, dtype=dtype), want, dtype)


# scale bytes of x and the weight; a payload of 8 with 246 is 2^122, with 0 it is 2^-124, and with 254 2^130
ENDS = [(0, 254), (0, 246), (0, 200), (1, 253), (1, 246), (1, 150), (246, 0), (246, 1), (246, 90), (246, 8), (8, 246), (20, 230), (200, 0), (127, 60), (60, 127)]


@forms
@pytest.mark.parametrize("dtype", TYPES)
def test_scale_bytes_near_both_ends(form, dtype):
    """Sums of whole multiples of 2^(a + b - 254) stay exact; f32 outputs widen payloads to bf16, which holds all of these
    but those of 2^128 and more."""
    rng = np.random.default_rng(3)
    x, w = R.whole(rng, (70, K), 1), R.whole(rng, (200, K), 128)
    for a, b in ENDS:
        if dtype == torch.float32 and max(a, b) > 246:
            continue
        x.scales.fill_(a)
        w.scales.fill_(b)
        same(ops.quant_linear(x, w, dtype=dtype), product(x, w), dtype)


@pytest.mark.parametrize("rows", [1, 16, 70])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_different_ends(rows, dtype):
    """Each row and each 128 weight rows with their own scale, through experts too."""
    rng = np.random.default_rng(rows)
    x, w = R.whole(rng, (rows, K), 1), R.whole(rng, (3, 300, K), 128)
    x.scales.copy_(torch.from_numpy(rng.choice([20, 60, 127, 200, 220], (rows, 1)).repeat(10, 1)))
    for low, high in ((120, 128), (130, 141)):
        w.scales.copy_(torch.from_numpy(rng.integers(low, high, (3, 3, 1)).repeat(10, 2)))
        one = ops.QuantMatrix(w.payload[1], w.scales[1])
        inside = np.abs(want := product(x, one))
        assert ((inside == 0) | ((inside > 2.0 ** -120) & (inside < 2.0 ** 127))).all()
        same(ops.quant_linear(x, one, dtype=dtype), want, dtype)
        counts = [rows // 3, 0, rows - rows // 3]
        same(ops.quant_moe_matmul(x, offsets_of(counts), w, dtype=dtype), grouped(x, counts, w), dtype)


@forms
def test_values_past_the_largest_float(form):
    """Infinite in f32 outputs and read back; bf16 outputs, whose instruction takes the bytes, hold their products."""
    x = ops.QuantMatrix(torch.zeros(3, 144, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :130],
                        torch.tensor([[254, 127], [247, 127], [254, 127]], dtype=torch.uint8, device="cuda"))
    w = ops.QuantMatrix(torch.zeros(2, 144, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :130],
                        torch.tensor([[7, 127]], dtype=torch.uint8, device="cuda"))
    for q, column in ((x, [2.0, 448.0, -1.875]), (w, [1.0, -2.0])):
        q.payload[:, 3] = torch.tensor(column, device="cuda").to(torch.float8_e4m3fn)
        q.payload[:, 129] = torch.ones(len(column), device="cuda").to(torch.float8_e4m3fn)
    inf, row = float("inf"), 2.0 ** 7
    for dtype in TYPES:
        back = ops.block_dequant(x, dtype)[:, [3, 129]].float()
        assert back.tolist() == [[inf, 1.0], [inf, 1.0], [-1.875 * 2.0 ** 127, 1.0]]
    assert ops.quant_linear(x, w, dtype=torch.float32).tolist() == [[inf, -inf], [inf, -inf], [-1.875 * row + 1, 3.75 * row + 1]]
    exact = torch.tensor([[2 * row + 1, -4 * row + 1], [449.0, -895.0], [-1.875 * row + 1, 3.75 * row + 1]])
    assert torch.equal(ops.quant_linear(x, w).cpu(), exact.bfloat16())


# ------------------------------------------------------------------ what the sums of bf16 outputs hold
def cut_off(x, w):
    """(sums of magnitudes, roots of sums of squares) of what an output x [k] . w [n, k]^T may lose, where within eight
    neighbouring products the instruction keeps multiples of 2^-13 of the largest one's power of two."""
    p = np.pad(w * x, ((0, 0), (0, -w.shape[1] % 8))).reshape(len(w), -1, 8)
    top = np.abs(p).max(-1, keepdims=True)
    lost = np.fmod(p, np.exp2(np.floor(np.log2(np.where(top == 0, 1, top))) - 13))
    return np.abs(lost).sum((1, 2)), np.sqrt((lost ** 2).sum((1, 2)))


@forms
@pytest.mark.parametrize("kind", ["normal", "payloads"])
@pytest.mark.parametrize("k", [520, 2048])
def test_what_bf16_outputs_leave_out(form, kind, k):
    """A bias of minus the result, rounded to bf16, is added before the output's rounding and leaves what that would hide
    (measured: 1.5e-5 of the norm for normal values, 5.1e-5 for payloads of all kinds, in every form)."""
    rng = np.random.default_rng(k)
    n = 400
    if kind == "normal":
        x = ops.block_quant(torch.from_numpy(rng.standard_normal((1, k))).float().cuda())
        w = ops.block_quant(torch.from_numpy(rng.standard_normal((n, k)) / k ** 0.5).float().cuda(), 128)
    else:
        finite = np.flatnonzero(np.arange(256) & 0x7f != 0x7f)
        x, w = (ops.QuantMatrix(torch.from_numpy(rng.choice(finite, s)).byte().cuda().view(torch.float8_e4m3fn),
                                torch.full((s[0], -(-k // 128)), 127, dtype=torch.uint8, device="cuda")) for s in ((1, k), (n, k)))
        x, w = (ops.QuantMatrix(torch.nn.functional.pad(q.payload.view(torch.uint8), (0, -k % 16)).view(torch.float8_e4m3fn)[:, :k], q.scales) for q in (x, w))
    xv, wv = R.held(x)[0], R.held(w)
    want, terms = wv @ xv, np.abs(wv) @ np.abs(xv)
    bias = torch.from_numpy(-want).bfloat16()
    left = want + f64(bias)
    lost, root = cut_off(xv, wv)
    # f32 sums: k / 8 of eights, and their groups', each off by 2^-23 of a partial sum at most (should the adder cut off).
    # The sum with the bias is exact; what is left is below 2^-8 of the result, and its rounding 2^-16 of that.  A root mean
    # square over 400 outputs is within an eighth of what is expected, and partial sums are on average two thirds of whole ones.
    bound = (lost + (k / 8 + 16) * 2.0 ** -23 * terms) * 1.01 + 2.0 ** -16 * np.abs(want)
    norm = 1.125 * np.linalg.norm(root) + ((k / 8 + 16) * 2.0 ** -23 * 2 / 3 + 2.0 ** -16) * np.linalg.norm(want)
    for rows in (1, 70, 300):
        many = ops.QuantMatrix(x.payload.view(torch.uint8).expand(rows, k), x.scales.expand(rows, -1).contiguous())
        wide = torch.zeros(rows, (k + 15) // 16 * 16, dtype=torch.uint8, device="cuda")
        wide[:, :k] = many.payload
        got = f64(ops.quant_linear(ops.QuantMatrix(wide.view(torch.float8_e4m3fn)[:, :k], many.scales), w, bias.cuda()))
        error = np.abs(got - left)
        assert (error <= bound).all()
        assert (np.linalg.norm(error, axis=1) <= norm).all()
