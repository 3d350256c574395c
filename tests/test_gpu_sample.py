"""Drawing tokens on the GPU against plain whole-number arithmetic: ids equal, shares as floats."""
import numpy as np
import pytest
import torch

from sandyrt_amd import ops
from tests import sample_reference as R

pytestmark = pytest.mark.gpu


def f32(v):
    return torch.tensor(np.asarray(v, np.float32), device="cuda")


def check(logits, u, t=None, k=None, p=None, least=None, k_dtype=torch.int32, **kw):
    """sample() of these rows against the plain form; settings are lists, one a row."""
    ids, probs = ops.sample(logits, f32(u), temperature=None if t is None else f32(t),
                            top_k=None if k is None else torch.tensor(k, dtype=k_dtype, device="cuda"),
                            top_p=None if p is None else f32(p), min_p=None if least is None else f32(least), **kw)
    rows = logits.float().cpu().double().numpy()
    want = []
    for r, row in enumerate(rows):
        s = {name: float(np.float32(v[r])) if name != "k" else v[r]
             for name, v in (("t", t), ("k", k), ("p", p), ("least", least)) if v is not None}
        want.append(R.draw(row, float(np.float32(u[r])), **s))
    assert ids.tolist() == [i for i, _ in want]
    # a share is rounded once from f64 to f32; whole weights may differ by one where 80 bits and 53 round apart
    np.testing.assert_allclose(probs.cpu().double().numpy(), [v for _, v in want], rtol=2.0 ** -23, atol=2.0 ** -30)
    return ids, probs


def model_logits(rng, rows, vocab, dtype):
    x = 2.0 * rng.standard_normal((rows, vocab))
    x[:, rng.integers(0, vocab, 20)] += rng.uniform(3, 9, 20)
    return torch.from_numpy(x).float().to(dtype).cuda()


def settings(rng, rows):
    return dict(t=rng.choice([0.0, 0.5, 0.8, 1.0, 1.3, 2.5], rows), k=rng.choice([0, 1, 2, 7, 50, 1000, 5000], rows).tolist(),
                p=rng.choice([1.0, 0.3, 0.8, 0.9, 0.95, 0.999], rows), least=rng.choice([0.0, 0.01, 0.1, 0.7], rows))


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (7, 100), (4, 2047), (3, 4095), (5, 4096), (3, 4097), (6, 8193), (8, 32000),
                                        (4, 50257), (2, 65536), (2, 65537), (3, 131075), (200, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_settings(rows, vocab, dtype):
    rng = np.random.default_rng(vocab + rows)
    x = model_logits(rng, rows, vocab, dtype)
    for _ in range(2):
        check(x, rng.random(rows, np.float32), **settings(rng, rows))


@pytest.mark.parametrize("only", ["t", "k", "p", "least", None])
def test_each_setting_alone(only):
    rng = np.random.default_rng(8)
    x = model_logits(rng, 40, 3000, torch.float32)
    s = settings(rng, 40)
    check(x, rng.random(40, np.float32), **{n: v for n, v in s.items() if n == only}, k_dtype=torch.int64, index_dtype=torch.int32)


def test_edges_of_the_settings():
    rng = np.random.default_rng(9)
    last = 1 - 2.0 ** -24
    k = [-3, 0, 1, 299, 300, 301, 1 << 30, 2]
    for u in (0.0, last, 0.5, 2.0 ** -24):
        check(model_logits(rng, 8, 300, torch.float32), [u] * 8, k=k)
        check(model_logits(rng, 8, 300, torch.float32), [u] * 8, p=[-1.0, 0.0, 1e-40, 1e-30, 1e-3, last, 1.0, 7.0])
        check(model_logits(rng, 8, 300, torch.float32), [u] * 8, least=[-1.0, 0.0, 1e-40, 1e-5, 0.5, last, 1.0, 0.999])
        check(model_logits(rng, 8, 300, torch.float32), [u] * 8, t=[0.0, 1e-40, 1e-30, 1e-3, 0.1, 30.0, 1e20, np.inf])
        check(model_logits(rng, 8, 300, torch.float32), [u] * 8, k=k, p=[0.0, 1e-30, 0.5, last] * 2, least=[0.0, 1.0, 0.1, 0.2] * 2)


@pytest.mark.parametrize("vocab", [40, 3000, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_further_apart_than_f32_reaches(vocab, dtype):
    """Temperatures so high that tokens weigh something whose distance from the maximum no f32 holds."""
    rng = np.random.default_rng(vocab + 7)
    x = torch.from_numpy(rng.uniform(-3.3e38, 3.3e38, (6, vocab))).to(dtype).cuda()
    t = [1e37, 3e37, 1e38, 1e38, 3e38, 3e38]
    for u in (0.2, 0.9, 1 - 2.0 ** -24):
        check(x, [u] * 6, t=t)
        check(x, [u] * 6, t=t, k=[3, 20, vocab - 1, vocab - 5, vocab * 4 // 5, vocab - 2])
        check(x, [u] * 6, t=t, p=[0.5, 0.9, 0.95, 0.99, 0.999, 0.9999])
        check(x, [u] * 6, t=t, k=[0, 0, vocab - 2, vocab - 1, 0, 30], p=[1.0, 0.99, 0.999, 0.9, 0.99, 0.9], least=[0.1, 0.3, 0.15, 0.01, 0.12, 0.2])


@pytest.mark.parametrize("vocab", [5, 5000, 20000, 70000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits(vocab, dtype):
    """Cuts inside runs of equals, more of them than a list holds: the lowest ids stay."""
    rng = np.random.default_rng(vocab)
    same = torch.full((6, vocab), 1.5, dtype=dtype, device="cuda")
    few = torch.from_numpy(rng.integers(-3, 3, (6, vocab))).to(dtype).cuda()
    k = [1, 3, vocab // 2, vocab - 1, vocab, 0]
    p = [0.5, 1.0, 0.25, 0.75, 0.9, 0.3]
    for x in (same, few, few * 0):
        for u in ([0.0] * 6, [1 - 2.0 ** -24] * 6, rng.random(6, np.float32)):
            check(x, u, k=k)
            check(x, u, p=p)
            check(x, u, k=k, p=p, least=[0.0, 0.05, 0.0, 0.3, 0.0, 0.1])
    if vocab > 5:  # the shares are 1 / kept exactly: every id in turn
        n = 64
        ids, probs = ops.sample(same[:1].expand(n, vocab), f32((np.arange(n) + 0.5) / n), top_k=torch.full((n,), n, device="cuda"))
        assert ids.tolist() == list(range(n)) and torch.equal(probs, torch.full_like(probs, 1 / n))


@pytest.mark.parametrize("vocab", [4, 4100, 30000, 66000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks(vocab, dtype):
    rng = np.random.default_rng(vocab + 1)
    x = model_logits(rng, 9, vocab, dtype)
    low = torch.finfo(dtype).min
    x[0, :] = -np.inf                       # nothing left
    x[1, :] = float("nan")
    x[2, 1:] = -np.inf                      # one token
    x[3, ::2] = -np.inf
    x[4, 1::2] = low                        # the type's lowest value is a logit like another
    x[5, :] = low
    x[6, 0] = float("nan")
    x[6, vocab - 1] = np.inf                # likelier than anything
    x[7, [0, vocab // 2]] = np.inf
    x[8, :-1] = -np.inf
    for u in (0.0, 0.3, 1 - 2.0 ** -24):
        check(x, [u] * 9)
        check(x, [u] * 9, t=[0.7] * 9, k=[3] * 9, p=[0.9] * 9, least=[0.05] * 9)
        check(x, [u] * 9, t=[0.0] * 9)
        check(x, [u] * 9, t=[50.0] * 9, p=[0.6] * 9)


def test_wide_and_narrow_ranges():
    """Logits far apart, next to one another, at the ends of the type; zeros of both signs rank alike."""
    rng = np.random.default_rng(3)
    n = 12000
    rows = [rng.standard_normal(n) * 1e30, rng.standard_normal(n) * 1e-30, 5.0 + rng.integers(0, 4, n) * 2.0 ** -21, rng.standard_normal(n) * 1e3,
            np.where(rng.random(n) < 0.5, -0.0, 0.0), np.where(rng.random(n) < 0.5, 3.4e38, -3.4e38), np.linspace(-1, 1, n), -np.abs(rng.standard_normal(n)) - 80]
    x = torch.from_numpy(np.stack(rows)).float().cuda()
    for t in (1.0, 1e-3, 1e4, 1e28, 1e-33):
        check(x, rng.random(8, np.float32), t=[t] * 8, k=[0, 5, 700, 0, 33, 9000, 0, 20], p=[0.9, 1.0, 0.5, 0.99, 0.9, 0.95, 0.3, 0.9])


def test_layouts():
    rng = np.random.default_rng(4)
    for dtype in (torch.float32, torch.bfloat16):
        wide = model_logits(rng, 7, 5003, dtype)
        for x in (wide[:, 3:4990], wide[::2, 1:], wide[2:3], wide[:1].expand(5, 5003), wide[:, :1]):
            check(x, rng.random(x.shape[0], np.float32), p=[0.9] * x.shape[0], k=[300] * x.shape[0])
    ids, probs = torch.empty(7, dtype=torch.int32, device="cuda"), torch.empty(7, device="cuda")
    out = check(wide, rng.random(7, np.float32), ids=ids, probs=probs)
    assert out[0] is ids and out[1] is probs
    assert ops.sample(wide[:0], f32([]))[0].shape == (0,)


def test_settings_out_of_range():
    """Recorded, and such a row gives -1; its neighbours their tokens."""
    rng = np.random.default_rng(5)
    x = model_logits(rng, 3, 5000, torch.float32)
    good = dict(t=1.0, p=0.9, least=0.1, u=0.25)
    for name, value in [("t", -1.0), ("t", np.nan), ("p", np.nan), ("least", 1.5), ("least", np.nan), ("u", 1.0), ("u", -0.1), ("u", np.nan)]:
        s = {n: [v, value if n == name else v, v] for n, v in good.items()}
        ids, probs = ops.sample(x, f32(s["u"]), temperature=f32(s["t"]), top_p=f32(s["p"]), min_p=f32(s["least"]))
        with pytest.raises(ops.SandyError, match="sample temperature"):
            ops.check_device_errors()
        ops.check_device_errors()
        want = [R.draw(x[r].cpu().double().numpy(), 0.25, t=1.0, p=float(np.float32(0.9)), least=float(np.float32(0.1))) for r in (0, 2)]
        assert ids.tolist() == [want[0][0], -1, want[1][0]] and probs[1].item() == 0.0


def test_streams_and_graphs():
    rng = np.random.default_rng(6)
    x, u = model_logits(rng, 16, 20000, torch.bfloat16), f32(rng.random(16))
    s = dict(temperature=f32([0.8] * 16), top_k=torch.full((16,), 500, device="cuda"), top_p=f32([0.9] * 16))
    want = ops.sample(x, u, **s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.sample(x, u, **s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs over the same inputs share no workspace
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.sample(x, u, **s))
    for i in range(3):
        x.add_(torch.randn_like(x) * i)
        u.copy_(torch.rand_like(u))
        now = ops.sample(x, u, **s)
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], now[0]) and torch.equal(out[1], now[1])
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])


def test_more_rows_than_are_done_at_a_time():
    rng = np.random.default_rng(7)
    rows, vocab = 2100, 9000
    x = torch.full((rows, vocab + 3), -np.inf)
    for r in range(rows):
        x[r, rng.integers(0, vocab, 12)] = torch.from_numpy(3 * rng.standard_normal(12)).float()
    s = settings(rng, rows)
    for index in (torch.int32, torch.int64):
        check(x.cuda()[:, :vocab], rng.random(rows, np.float32), **s, k_dtype=index, index_dtype=index)


def test_largest_vocabulary():
    """Ids of 24 bits, at either end and where parts meet."""
    vocab = 1 << 24
    at = torch.tensor([0, 1, 262143, 262144, 1 << 23, vocab - 2, vocab - 1])
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.full((2, vocab), -np.inf, dtype=dtype)
        x[:, at] = torch.tensor([1.0, 0.5, 0.5, -1.0, 1.0, 0.25, 1.0], dtype=dtype)
        for u in (0.0, 0.4, 0.7, 1 - 2.0 ** -24):
            check(x.cuda(), [u] * 2, k=[0, 5], p=[1.0, 0.9])
