"""The 8-bit products and sampling together, as a model would use them: norm, rows into 8 bits, products, experts, the head's
f32 logits and a token, against 64-bit numpy that begins each stage from what the GPU had; eagerly and as a replayed graph."""
import numpy as np
import pytest
import torch

from sandyrt_amd import ops
from tests import block_quant_reference as R
from tests import sample_reference as S

pytestmark = pytest.mark.gpu
HIDDEN, FFN, MOE_FFN, EXPERTS, TOP, VOCAB = 320, 700, 192, 6, 2, 9001  # one vocabulary of rows in parts, ffn no multiple of 128
HALF = 2.0 ** -8  # half a step of bf16, relative


def f64(t):
    return t.detach().cpu().double().numpy()


class Model:
    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            return ops.block_quant(torch.randn(*shape, generator=g, device="cuda") / shape[-1] ** 0.5, 128)

        self.norm = torch.ones(HIDDEN, dtype=torch.bfloat16, device="cuda")
        self.gate_up, self.down = weight(2 * FFN, HIDDEN), weight(HIDDEN, FFN)
        self.router = torch.randn(EXPERTS, HIDDEN, generator=g, device="cuda").bfloat16()
        self.expert_up, self.expert_down = weight(EXPERTS, 2 * MOE_FFN, HIDDEN), weight(EXPERTS, HIDDEN, MOE_FFN)
        self.head = weight(VOCAB, HIDDEN)

    def step(self, h, settings):
        """h [rows, HIDDEN] bf16 -> (token ids, what every stage began and ended with)."""
        nodes, result = ops.silu_mul_nodes()
        seen = {}

        def act(gate_up, ffn):
            return ops.elementwise(nodes, result, [gate_up[:, :ffn].contiguous(), gate_up[:, ffn:].contiguous()])

        def linear(name, x, w, **kw):
            q = ops.block_quant(x)
            y = ops.quant_linear(q, w, **kw)
            seen[name] = (x, q, w, y)
            return y

        def experts(name, x, offsets, w):
            q = ops.block_quant(x)
            y = ops.quant_moe_matmul(q, offsets, w)
            seen[name] = (x, q, w, y, offsets)
            return y

        y = act(linear("gate_up", ops.rms_norm(h, self.norm, 1e-6), self.gate_up), FFN)
        h = h + linear("down", y, self.down)
        x = ops.rms_norm(h, self.norm, 1e-6)
        share, chosen = ops.topk(ops.softmax(ops.matmul(x, self.router, transpose_rhs=True)), TOP)
        packed, shares, tokens, offsets = ops.moe_gather(x, chosen, share, EXPERTS)
        y = experts("expert_down", act(experts("expert_up", packed, offsets, self.expert_up), MOE_FFN), offsets, self.expert_down)
        h = h + ops.moe_scatter_sum(y, shares, tokens, h.shape[0])
        logits = linear("head", ops.rms_norm(h, self.norm, 1e-6), self.head, dtype=torch.float32)
        ids, probs = ops.sample(logits, **settings)
        seen["sample"] = (logits, ids, probs)
        return ids, seen


def settings_of(rows, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def pick(*values):
        return torch.tensor(values, device="cuda")[torch.randint(len(values), (rows,), generator=g, device="cuda")]

    return dict(uniforms=torch.rand(rows, generator=g, device="cuda"), temperature=pick(0.0, 0.7, 1.0, 1.2), top_k=pick(0, 5, 40, 2000),
                top_p=pick(1.0, 0.9, 0.5), min_p=pick(0.0, 0.02))


@pytest.mark.parametrize("rows", [1, 3, 40, 150])
def test_run(rows):
    model, settings = Model(rows), settings_of(rows, rows)
    h = torch.randn(rows, HIDDEN, device="cuda").bfloat16()
    _, seen = model.step(h, settings)
    for name, (x, q, w, y, *offsets) in ((n, v) for n, v in seen.items() if n != "sample"):
        payload, code = R.quantise(f64(x), 1)
        np.testing.assert_array_equal(f64(q.payload.float()), payload)
        np.testing.assert_array_equal(q.scales.cpu().numpy(), code)
        xv, got = R.held(q), f64(y)
        parts = [(0, len(xv), w)]
        if offsets:
            at = offsets[0].tolist()
            assert at[0] == 0 and at[-1] == len(xv) == rows * TOP
            parts = [(a, b, ops.QuantMatrix(w.payload[e], w.scales[e])) for e, (a, b) in enumerate(zip(at, at[1:]))]
        for a, b, each in parts:
            wv = R.held(each)
            want = xv[a:b] @ wv.T
            # as the products' own tests: bf16 outputs drop less than 2^-10 of the terms' magnitudes and round once;
            # f32 sums of k exact terms are off by less than k steps of them
            terms = np.abs(xv[a:b]) @ np.abs(wv).T
            bound = terms * 2.0 ** -10 + HALF * np.abs(want) if y.dtype == torch.bfloat16 else terms * xv.shape[1] * 2.0 ** -23
            assert (np.abs(got[a:b] - want) <= bound * 1.01).all(), name
    logits, ids, probs = seen["sample"]
    for r, row in enumerate(f64(logits)):
        s = {n: float(settings[m][r]) for n, m in (("t", "temperature"), ("p", "top_p"), ("least", "min_p"))}
        token, share = S.draw(row, float(settings["uniforms"][r]), k=int(settings["top_k"][r]), **s)
        assert ids[r].item() == token
        np.testing.assert_allclose(probs[r].item(), share, rtol=2.0 ** -23, atol=2.0 ** -30)


@pytest.mark.parametrize("rows", [1, 40])
def test_run_in_a_graph(rows):
    model, settings = Model(7), settings_of(rows, 7)
    h = torch.randn(rows, HIDDEN, device="cuda").bfloat16()
    model.step(h, settings)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, seen = model.step(h, settings)
    for _ in range(3):
        h.copy_(torch.randn_like(h))
        settings["uniforms"].copy_(torch.rand(rows, device="cuda"))
        now, eager = model.step(h, settings)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, now) and torch.equal(seen["sample"][2], eager["sample"][2])
        assert all(torch.equal(seen[n][3], eager[n][3]) for n in seen if n != "sample")


def test_two_streams_at_once():
    """Two runs side by side share no workspace: each has the tokens it has alone."""
    model = Model(8)
    hs = [torch.randn(30, HIDDEN, device="cuda").bfloat16() for _ in range(2)]
    sets = [settings_of(30, i) for i in range(2)]
    want = [model.step(h, s)[0] for h, s in zip(hs, sets)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(model.step(hs[i], sets[i])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(ids, want[i]) for i in range(2) for ids in got[i])
