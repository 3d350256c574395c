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


# Two logits 0 and l: exp(l / T) is above min_p by 1.5e-15 to 5.8e-15 of itself.  All are near half a power of two, where a series
# of 2^f is worst; the comparison is in 64 bits, whose roundings (2.3e-16 of the exponent, 2.5 at most here, in base 2, and of the
# sum) are below 1e-15 together.
BARELY = [("-0x1.1ecd28p+1", "0x1.15aca4p+1", "0x1.6c8712p-2"), ("-0x1.6a9f24p-1", "0x1.028444p+1", "0x1.688e86p-1"),
          ("-0x1.284cc2p-2", "0x1.1b3b8ep-2", "0x1.67b93cp-2"), ("-0x1.d7620cp-1", "0x1.5cf878p+1", "0x1.6d446ap-1"),
          ("-0x1.0b6424p+2", "0x1.34d0dcp+1", "0x1.6a746ep-3"), ("-0x1.563dbcp+0", "0x1.f26944p+1", "0x1.6b36d0p-1"),
          ("-0x1.f2141ap+1", "0x1.e3a5fep+1", "0x1.6da296p-2"), ("-0x1.be7df6p-2", "0x1.3ba932p+0", "0x1.677f6ap-1"),
          ("-0x1.4e4fbcp+1", "0x1.427730p+1", "0x1.6b1f02p-2"), ("-0x1.26bc6cp+1", "0x1.541c6ap+0", "0x1.69ed66p-3"),
          ("-0x1.526524p+1", "0x1.458eeap+1", "0x1.6a24d6p-2"), ("-0x1.b07b96p-3", "0x1.33afd0p-1", "0x1.684bcap-1"),
          ("-0x1.26688cp+0", "0x1.ac9654p+1", "0x1.6b2a92p-1"), ("-0x1.581180p+1", "0x1.4ab5dep+1", "0x1.69cbbep-2"),
          ("-0x1.674756p-1", "0x1.ff4bc0p+0", "0x1.685114p-1"), ("-0x1.a1a680p-3", "0x1.30cf92p-1", "0x1.6b7facp-1"),
          ("-0x1.9ce10cp-2", "0x1.300482p+0", "0x1.6c9a0ap-1"), ("-0x1.c0f51ep-2", "0x1.44e9eap+0", "0x1.6a72b0p-1"),
          ("-0x1.e535c6p-2", "0x1.5fd2aap+0", "0x1.6ab004p-1")]
# A logit 0 and `n` logits l: the first token's share is below u, so that a later one is drawn, by two to four and a half multiples
# of 2^-50 in the weight of each, which the whole weights, off by one at most, leave room for.
SHARES = [("-0x1.5c1c88p-2", 2297, "0x1.40777ap-11"), ("-0x1.5c2240p-2", 2929, "0x1.f6b6e0p-12"), ("-0x1.62866cp-2", 3726, "0x1.8db25ap-12"),
          ("-0x1.5fc9bap-2", 3658, "0x1.940180p-12"), ("-0x1.6a50cep-2", 2411, "0x1.3595c4p-11"), ("-0x1.614f26p-2", 2975, "0x1.f1739cp-12"),
          ("-0x1.5c1e04p-2", 174, "0x1.0673c4p-7"), ("-0x1.615f8ap-2", 1935, "0x1.7e5594p-11")]


@pytest.mark.parametrize("padding", [0, 8200])
def test_weights_next_to_min_p(padding):
    """What is kept by a few parts in 10^15."""
    l, t, least = (np.array([float.fromhex(v) for v in column]) for column in zip(*BARELY))
    x = torch.full((len(l), 2 + padding), -np.inf)
    x[:, 0], x[:, 1] = 0.0, torch.from_numpy(l).float()
    assert (x[:, 1].double().numpy() == l).all() and (t.astype(np.float32) == t).all() and (least.astype(np.float32) == least).all()
    ids, _ = check(x.cuda(), [1 - 2.0 ** -24] * len(l), t=t, least=least)
    assert ids.tolist() == [1] * len(l)


@pytest.mark.parametrize("l,n,u", SHARES)
def test_weights_next_to_a_share(l, n, u):
    x = torch.full((1, n + 1), float.fromhex(l))
    x[0, 0] = 0.0
    ids, _ = check(x.cuda(), [float.fromhex(u)])
    assert ids.item() == 1


BAD = [("t", -1.0), ("t", np.nan), ("t", -np.inf), ("p", np.nan), ("least", 1.5), ("least", np.nan), ("u", 1.0), ("u", -0.1), ("u", np.nan),
       ("u", -2.0 ** -149), ("u", np.inf)]


@pytest.mark.parametrize("cuts", [True, False])
@pytest.mark.parametrize("rows,vocab,bad", [(4, 8193, (1, 3)), (5, 60000, (0, 2)), (2060, 8200, (2, 1023, 1024, 1030, 2048, 2059))])
def test_settings_out_of_range_of_rows_in_parts(rows, vocab, bad, cuts):
    """Recorded, and such a row gives -1; its neighbours their tokens, also behind the rows that are done at a time."""
    rng = np.random.default_rng(rows)
    x = torch.full((rows, vocab), -np.inf)
    at = torch.from_numpy(rng.integers(0, vocab, (rows, 12)))
    x.scatter_(1, at, torch.from_numpy(3 * rng.standard_normal((rows, 12))).float())
    x = x.cuda()
    good = dict(t=0.8, p=0.9 if cuts else 1.0, least=0.01, u=0.25)

    def draw(s):
        return ops.sample(x, f32(s["u"]), temperature=f32(s["t"]), top_p=f32(s["p"]), min_p=f32(s["least"]))

    fine = check(x, [good["u"]] * rows, **{n: [v] * rows for n, v in good.items() if n != "u"})
    ops.check_device_errors()
    for name, value in BAD:
        s = {n: np.full(rows, v, np.float32) for n, v in good.items()}
        s[name][list(bad)] = value
        ids, probs = draw(s)
        with pytest.raises(ops.SandyError, match="sample temperature"):
            ops.check_device_errors()
        ops.check_device_errors()
        want, share = fine[0].clone(), fine[1].clone()
        want[list(bad)] = -1
        share[list(bad)] = 0.0
        assert torch.equal(ids, want) and torch.equal(probs, share), (name, value)


@pytest.mark.parametrize("vocab", [700, 9000])
def test_subnormal_logits_and_temperatures(vocab):
    """Distances that are subnormal floats, one bin for all of them."""
    rng = np.random.default_rng(vocab + 2)
    x = torch.from_numpy(rng.integers(-70000, 70000, (6, vocab)) * 2.0 ** -149).float().cuda()
    assert x.abs().max() < 2.0 ** -126 and x.unique().numel() > 600
    for t in (2.0 ** -149, 1e-42, 1e-41, 1e-40, 1e-38, 1.0):
        check(x, rng.random(6, np.float32), t=[t] * 6)
        check(x, rng.random(6, np.float32), t=[t] * 6, k=[1, 7, 300, vocab - 1, 0, 0], p=[1.0, 0.9, 0.5, 1.0, 0.8, 0.99], least=[0.0, 0.1, 0.0, 0.0, 0.3, 0.0])


@pytest.mark.parametrize("vocab", [900, 9000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_logits_at_every_temperature(vocab, dtype):
    """The likeliest at inf share all of the weight, however hot."""
    rng = np.random.default_rng(vocab + 3)
    x = model_logits(rng, 6, vocab, dtype)
    for r in range(6):
        x[r, torch.from_numpy(rng.permutation(vocab)[:r + 1])] = np.inf
    top = torch.isinf(x)
    for t in (1e-30, 1.0, 1e30, np.inf):
        for s in ({}, dict(k=[1, 1, 2, 9, 300, vocab - 1]), dict(p=[0.5] * 6), dict(k=[3] * 6, p=[0.9] * 6, least=[0.2] * 6)):
            for u in (0.0, 0.6, 1 - 2.0 ** -24):
                finite = min(t, 1e30)  # inf / inf has no value in the plain form; every finite temperature has the same result
                ids, probs = check(x, [u] * 6, t=[finite] * 6, **s)
                if t != finite:
                    names = dict(k="top_k", p="top_p", least="min_p")
                    kw = {names[n]: torch.tensor(v, dtype=torch.int32, device="cuda") if n == "k" else f32(v) for n, v in s.items()}
                    hot = ops.sample(x, f32([u] * 6), temperature=f32([t] * 6), **kw)
                    assert torch.equal(hot[0], ids) and torch.equal(hot[1], probs)
                assert bool(top[torch.arange(6, device="cuda"), ids].all())
