"""Performance cases of the paged K/V cache held in 8 bits: writing it, reading it back, attending to it.

A pool is [pages, kv heads, page rows, head dim] of int8 or e4m3 payloads.  Each block (a page of one head) has one
scale 2^(c - 127), its byte c in [pages, kv heads]; c = 255 stands for NaN.  Kinds:

  append   quantise new K and V rows as they are written behind each sequence's rows, and read the touched pages back
           as what they stand for (the rows already there among them: a block whose scale grows is rescaled)
  read     a context's K and V rows back in bf16 or f32
  attend   causal attention of one query a sequence (a decode step) or of several (a prompt chunk) over the cache

Head layouts are those this repository runs (TinyLlama 32 / 4 of 64, a Gemma-style layer 8 / 2 of 256, GPT-2 12 / 12
of 64, 16 / 2 of 128) and two odd head dims.  Sequences of a batch have contexts spread over the case's range; the
last of a chunked batch is the shortest.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "f32": F32}
# payload type, exponent of the largest payload's frexp, its mantissa, the largest payload
FORMATS = {"int8": (torch.int8, 7, 127.0 / 128.0), "e4m3": (torch.float8_e4m3fn, 9, 0.875)}


def listed():
    return [
        # one sequence's decode step: launches and latency
        {"name": "append_step_1", "kind": "append", "batch": 1, "heads": 4, "dim": 64, "page": 16, "tokens": 1,
         "low": 777, "high": 777, "format": "int8", "dtype": "bf16"},
        # a batched step of a sliding-window layer's wide heads
        {"name": "append_step_64", "kind": "append", "batch": 64, "heads": 2, "dim": 256, "page": 16, "tokens": 1,
         "low": 512, "high": 4096, "format": "e4m3", "dtype": "bf16"},
        # long prompts of a batch, from the first row: memory streams
        {"name": "append_prompts_4096", "kind": "append", "batch": 8, "heads": 8, "dim": 128, "page": 32, "tokens": 4096,
         "low": 0, "high": 0, "format": "e4m3", "dtype": "bf16"},
        # ragged fp32 chunks that begin and end inside a page
        {"name": "append_ragged_f32", "kind": "append", "batch": 7, "heads": 12, "dim": 64, "page": 16, "tokens": 333,
         "low": 5, "high": 700, "format": "int8", "dtype": "f32"},
        # a short context back
        {"name": "read_short", "kind": "read", "batch": 1, "heads": 4, "dim": 64, "page": 16, "low": 100, "high": 100,
         "format": "e4m3", "dtype": "f32"},
        # a batch's whole contexts back
        {"name": "read_contexts", "kind": "read", "batch": 32, "heads": 4, "dim": 64, "page": 16, "low": 512, "high": 4096,
         "format": "int8", "dtype": "bf16"},
        # one sequence's decode step at a long context
        {"name": "decode_long_1", "kind": "attend", "batch": 1, "q_heads": 32, "heads": 4, "dim": 64, "page": 16,
         "tokens": 1, "low": 32749, "high": 32749, "window": 0, "format": "int8", "dtype": "bf16"},
        # a batched decode step of mixed contexts
        {"name": "decode_32", "kind": "attend", "batch": 32, "q_heads": 32, "heads": 4, "dim": 64, "page": 16, "tokens": 1,
         "low": 512, "high": 4096, "window": 0, "format": "e4m3", "dtype": "bf16"},
        # wide heads, a sliding window, many sequences
        {"name": "decode_window_64", "kind": "attend", "batch": 64, "q_heads": 8, "heads": 2, "dim": 256, "page": 16,
         "tokens": 1, "low": 512, "high": 4096, "window": 1024, "format": "int8", "dtype": "bf16"},
        # fp32 heads without groups, short contexts
        {"name": "decode_f32", "kind": "attend", "batch": 3, "q_heads": 12, "heads": 12, "dim": 64, "page": 16, "tokens": 1,
         "low": 9, "high": 1000, "window": 0, "format": "e4m3", "dtype": "f32"},
        # the prompt chunk of the engine's default length
        {"name": "prompt_2048", "kind": "attend", "batch": 1, "q_heads": 32, "heads": 4, "dim": 64, "page": 16,
         "tokens": 2048, "low": 2048, "high": 2048, "window": 0, "format": "e4m3", "dtype": "bf16"},
        # later, ragged chunks of a batch over larger pages
        {"name": "prompt_ragged", "kind": "attend", "batch": 3, "q_heads": 16, "heads": 2, "dim": 128, "page": 64,
         "tokens": 203, "low": 300, "high": 1700, "window": 0, "format": "int8", "dtype": "bf16"},
    ]


LAYOUTS = [(32, 4, 64), (32, 4, 64), (8, 2, 256), (16, 2, 128), (12, 12, 64), (10, 2, 96), (6, 3, 80)]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
    q_heads, heads, dim = rng.choice(LAYOUTS)
    case = {"kind": kind, "heads": heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128]),
            "format": rng.choice(["int8", "e4m3"]), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "attend":
        case |= {"q_heads": q_heads, "window": rng.choice([0, 0, rng.randrange(1, 2000)])}
        if rng.random() < 0.4:  # chunks
            batch = rng.choice([1, 1, 2, 5])
            tokens = _log_int(rng, 2, 2000 // batch)
            low = tokens + rng.choice([0, rng.randrange(1, 1500 // batch)])
            high = low + rng.randrange(0, 300)
            # no more products than the listed chunk of 2048
            most = 2048 * 960 * 32 * 64 // (batch * (high - tokens // 2) * q_heads * dim)
            tokens = min(tokens, max(2, most), 300 if case["dtype"] == "f32" else 2000)
            return case | {"batch": batch, "tokens": tokens, "low": low, "high": high}
        low = _log_int(rng, 1, 1500) if rng.random() < 0.8 else _log_int(rng, 1500, 60000)
        high = low + _log_int(rng, 1, 4000)
        batch = min(_log_int(rng, 1, 64), max(1, 64 * 4096 * 2 * 256 // (high * heads * dim)))
        return case | {"batch": batch, "tokens": 1, "low": low, "high": high}
    low = _log_int(rng, 1, 1500)
    if kind == "read":
        high = low + _log_int(rng, 1, 2500)
        batch = min(_log_int(rng, 1, 32), max(1, 32 * 4096 * 4 * 64 // (high * heads * dim)))
        return case | {"batch": batch, "low": low, "high": high}
    if rng.random() < 0.5:
        return case | {"batch": _log_int(rng, 1, 128), "tokens": 1, "low": low, "high": low + _log_int(rng, 1, 2500)}
    batch = _log_int(rng, 1, 8)
    low = rng.choice([0, low])
    return case | {"batch": batch, "tokens": _log_int(rng, 2, 4000 // batch), "low": low, "high": low + rng.randrange(0, 500)}


# ------------------------------------------------------------------ inputs
def _spread(case):
    """One length a sequence, spread over the case's range, the last the shortest."""
    low, high, n = case["low"], case["high"], case["batch"]
    return [low + int((high - low) * (((n - 1 - b) * 0.6180339887498949) % 1.0) + 0.5) for b in range(n)]


def _counts(case):
    """Valid new rows (or queries) of each sequence: all of them, or a ragged batch of chunks."""
    t = case.get("tokens", 0)
    if t < 2 or case["batch"] < 2:
        return [t] * case["batch"]
    return [t - (b * 37) % max(1, t // 2) for b in range(case["batch"])]


def _rows(case):
    """Per sequence: (first new row or query, rows in the cache after the call)."""
    if case["kind"] == "append":
        return [(p, p + n) for p, n in zip(_spread(case), _counts(case))]
    if case["kind"] == "read":
        return [(0, n) for n in _spread(case)]
    return [(max(0, n - c), max(n, c)) for n, c in zip(_spread(case), _counts(case))]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    heads, dim, page, batch = case["heads"], case["dim"], case["page"], case["batch"]
    rows = _rows(case)
    blocks = [-(-last // page) for _, last in rows]
    width, total = max(blocks), sum(blocks)
    perm = torch.randperm(total + 3, generator=g, device="cuda").to(torch.int32)
    # entries past a sequence's pages name none; the pool's last page stays unused
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = perm[at:at + n]
        at += n
    s = {"case": case, "table": table, "format": case["format"], "page": page, "dtype": DTYPES[case["dtype"]]}
    kind, pages = FORMATS[case["format"]][0], total + 4
    for name in ("k", "v"):
        # what earlier appends left: N(0, 1) rows, some pages louder than others
        loud = torch.exp(torch.randn(pages, heads, 1, 1, generator=g, device="cuda"))
        x = torch.randn(pages, heads, page, dim, generator=g, device="cuda") * loud
        code = _code(x.abs().amax((2, 3)), case["format"])
        s[name + "_pool"] = _round(x * _pow2(127 - code)[..., None, None], case["format"])
        s[name + "_scales"] = code.to(torch.uint8)
        assert s[name + "_pool"].dtype == kind
        del x, loud
    s["positions"] = torch.tensor([p for p, _ in rows], dtype=torch.int64, device="cuda")
    counts = _counts(case)
    s["counts"] = torch.tensor(counts, dtype=torch.int64, device="cuda") if len(set(counts)) > 1 else None
    t = case.get("tokens", 0)
    if case["kind"] == "append":
        # K and V as the projection leaves them: heads side by side in a token's row
        kv = torch.randn(batch, t, 2, heads, dim, generator=g, device="cuda")
        kv = (kv * torch.exp(0.5 * torch.randn(batch, t, 1, 1, 1, generator=g, device="cuda"))).to(s["dtype"])
        s["k"], s["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        # the rows read back: from the start of the first touched page
        s["back_at"] = s["positions"] // page * page
        s["back_counts"] = torch.tensor([last - p // page * page for p, last in rows], dtype=torch.int64, device="cuda")
        s["back"] = max(last - p // page * page for p, last in rows)
    elif case["kind"] == "read":
        s["back_at"] = s["positions"]
        s["back_counts"] = torch.tensor([last for _, last in rows], dtype=torch.int64, device="cuda")
        s["back"] = max(last for _, last in rows)
    else:
        q = torch.randn(batch, t, case["q_heads"], dim, generator=g, device="cuda").to(s["dtype"])
        s["q"] = q.transpose(1, 2)
    return s


# ------------------------------------------------------------------ plain forms
def _pow2(e):
    """2^e as f32, e whole: the smallest normal number at the least, 0 at e = -127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _code(amax, format):
    """The scale byte of a block whose largest magnitude is amax."""
    _, bits, top = FORMATS[format]
    m, ex = torch.frexp(amax)
    e = torch.where(amax > 0, ex - bits + (m > top), -126).clamp(min=-126)
    return torch.where(torch.isfinite(amax), e + 127, 255).to(torch.int32)


def _round(y, format):
    return torch.round(y).to(torch.int8) if format == "int8" else y.to(torch.float8_e4m3fn)


def _values(pool, index):
    """Payloads of the pages named, as f32."""
    return pool.view(torch.uint8)[index].view(pool.dtype).float()


def _plain_append(s, x, pool, scales):
    page, table, pos, fmt = s["page"], s["table"], s["positions"], s["format"]
    batch, heads, t, dim = x.shape
    count = s["counts"] if s["counts"] is not None else torch.full_like(pos, t)
    n = (t + page - 2) // page + 1
    ordinal = pos[:, None] // page + torch.arange(n, device=pos.device)
    slot = ordinal[..., None] * page + torch.arange(page, device=pos.device)  # [batch, n, page] positions
    first, end = pos[:, None, None], (pos + count)[:, None, None]
    new, old = (slot >= first) & (slot < end), slot < first
    touched = new.any(-1)
    blocks = table.gather(1, ordinal.clamp(max=table.shape[1] - 1)).long()
    blocks = torch.where(touched, blocks, pool.shape[0] - 1)  # the page that no sequence has
    index = (slot - first).clamp(0, t - 1)
    rows = x.transpose(1, 2)[torch.arange(batch, device=pos.device)[:, None, None], index].float()
    rows = rows.transpose(2, 3)  # [batch, n, heads, page, dim]
    new, old = new[:, :, None, :, None], old[:, :, None, :, None]
    code = _code((rows.abs() * new).amax((3, 4)), fmt)
    was = torch.where(old.any(3)[..., 0], scales[blocks].int(), 0)
    code = torch.maximum(code, was)
    kept = _values(pool, blocks)
    kept = torch.where(old, _round(kept * _pow2((was - code).clamp(min=-126))[..., None, None], fmt).float(), kept)
    fresh = _round(rows * _pow2(127 - code)[..., None, None], fmt).float()
    out = torch.where(new, torch.where((code == 255)[..., None, None], 0.0, fresh), kept)
    pool.view(torch.uint8)[blocks] = out.to(pool.dtype).view(torch.uint8)
    scales[blocks] = code.to(torch.uint8)


def _plain_read(s, pool, scales, first, count, tokens, dtype):
    """Rows first .. first + tokens of each sequence [batch, heads, tokens, dim], zero from count on."""
    page, table = s["page"], s["table"]
    at = first[:, None] + torch.arange(tokens, device=first.device)
    block = table.gather(1, (at // page).clamp(max=table.shape[1] - 1)).clamp(min=0).long()
    payload = pool.view(torch.uint8).transpose(1, 2)[block, at % page].view(pool.dtype).float()
    code = scales[block].int()
    value = payload * torch.where(code == 255, math.nan, _pow2(code - 127))[..., None]
    value = torch.where((torch.arange(tokens, device=first.device) < count[:, None])[..., None, None], value, 0.0)
    return value.transpose(1, 2).to(dtype).contiguous()


def _plain_attend(s):
    case, q, pos = s["case"], s["q"], s["positions"]
    batch, hq, t, dim = q.shape
    heads, window = case["heads"], case["window"]
    keys = s["table"].shape[1] * s["page"]
    all_keys, zero = torch.full_like(pos, keys), torch.zeros_like(pos)
    last = pos[:, None] + torch.arange(t, device=pos.device)
    if s["counts"] is not None:
        last = torch.where(torch.arange(t, device=pos.device) < s["counts"][:, None], last, -1)
    key = torch.arange(keys, device=pos.device)
    seen = key <= last[..., None]
    if window > 0:
        seen &= key > last[..., None] - window
    seen = seen[:, None, None]  # [batch, 1, 1, t, keys]
    k = _plain_read(s, s["k_pool"], s["k_scales"], zero, all_keys, keys, F32)
    score = q.float().reshape(batch, heads, hq // heads * t, dim) @ k.transpose(2, 3) * (1.0 / math.sqrt(dim))
    del k
    score = torch.where(seen, score.view(batch, heads, hq // heads, t, keys), -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=torch.finfo(F32).min))
    del score
    total = p.sum(-1, keepdim=True)
    v = _plain_read(s, s["v_pool"], s["v_scales"], zero, all_keys, keys, F32)
    out = p.reshape(batch, heads, hq // heads * t, keys) @ v
    out = out.view(batch, heads, hq // heads, t, dim) / torch.where(total > 0, total, 1.0)
    return out.reshape(batch, hq, t, dim).to(q.dtype)


# ------------------------------------------------------------------ one pass
def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        from sandyrt_amd import ops
        caches = ops.QuantPagedCache(s["k_pool"], s["k_scales"]), ops.QuantPagedCache(s["v_pool"], s["v_scales"])
        if kind == "attend":
            return ops.quant_paged_attention(s["q"], *caches, s["table"], s["positions"], counts=s["counts"],
                                             window=s["case"]["window"])
        if kind == "append":
            ops.quant_paged_append(s["k"], s["v"], *caches, s["table"], s["positions"], counts=s["counts"])
        k, v = ops.quant_paged_read(*caches, s["table"], s["back_at"], s["back"], counts=s["back_counts"],
                                    dtype=s["dtype"])
        return {"k": k, "v": v}
    if kind == "attend":
        return _plain_attend(s)
    if kind == "append":
        _plain_append(s, s["k"], s["k_pool"], s["k_scales"])
        _plain_append(s, s["v"], s["v_pool"], s["v_scales"])
    return {n: _plain_read(s, s[n + "_pool"], s[n + "_scales"], s["back_at"], s["back_counts"], s["back"], s["dtype"])
            for n in ("k", "v")}


def work(case):
    dim, heads, page = case["dim"], case["heads"], case["page"]
    size = 2 if case["dtype"] == "bf16" else 4
    rows, counts = _rows(case), _counts(case)
    if case["kind"] == "attend":
        t, hq, window = case["tokens"], case["q_heads"], case["window"]
        read = seen = 0
        for (first, _), n in zip(rows, counts):
            lowest = max(0, first + 1 - window) if window > 0 else 0
            read += first + n - lowest
            seen += sum(min(first + i + 1, window) if window > 0 else first + i + 1 for i in range(n))
        q = case["batch"] * hq * t * dim * size
        return {"bytes": 2 * read * heads * dim + 2 * -(-read // page) * heads + 2 * q, "flops": 4 * seen * hq * dim}
    back = max(last - (p // page * page if case["kind"] == "append" else 0) for p, last in rows)
    out = 2 * case["batch"] * heads * back * dim * size
    if case["kind"] == "read":
        held = sum(last for _, last in rows)
        return {"bytes": out + 2 * heads * (held * dim + -(-held // page)), "flops": 0}
    new = sum(counts)
    return {"bytes": out + 2 * heads * (new * dim * (size + 1) + -(-new // page)), "flops": 0}


# ------------------------------------------------------------------ 64 bits
def _two(e):
    """2^e as f64."""
    return ((e.long() + 1023) << 52).view(F64)


def _exact_round(y, format):
    """Nearest payload, ties to the even one."""
    if format == "int8":
        return torch.round(y)
    _, ex = torch.frexp(y)
    step = _two(ex.clamp(min=-5) - 4)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    page, table, fmt = s["page"], s["table"].tolist(), s["format"]
    largest = 127.0 if fmt == "int8" else 448.0
    rows, counts = _rows(case), _counts(case)

    def held(pool, scales, b, n):
        """The first n rows of sequence b, [heads, n, dim]."""
        pages = [table[b][i] for i in range(-(-n // page))]
        scale = _two(scales[pages].int() - 127)
        value = pool.view(torch.uint8)[pages].view(pool.dtype).double() * scale[..., None, None]
        return value.transpose(0, 1).flatten(1, 2)[:, :n]

    if case["kind"] == "attend":
        q = s["q"].double()
        out = torch.zeros(q.shape, dtype=F64, device="cuda")
        group = case["q_heads"] // case["heads"]
        for b, ((first, _), n) in enumerate(zip(rows, counts)):
            k, v = (held(s[c + "_pool"], s[c + "_scales"], b, first + n) for c in "kv")
            past = torch.arange(first, first + n, device="cuda")[:, None] - torch.arange(first + n, device="cuda")
            hidden = past < 0
            if case["window"] > 0:
                hidden |= past >= case["window"]
            for h in range(case["q_heads"]):
                score = (q[b, h, :n] @ k[h // group].T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
                out[b, h, :n] = torch.softmax(score, -1) @ v[h // group]
        return out
    got = {}
    for c in "kv":
        pool, scales = s[c + "_pool"], s[c + "_scales"]
        out = torch.zeros(case["batch"], case["heads"], s["back"], case["dim"], dtype=F64, device="cuda")
        for b, ((first, last), n) in enumerate(zip(rows, counts)):
            if case["kind"] == "read":
                out[b, :, :last] = held(pool, scales, b, last)
                continue
            x = s[c][b, :, :n].double()
            begin = first // page * page
            for p0 in range(begin, last, page):
                block = table[b][p0 // page]
                lo, hi = max(first, p0), min(last, p0 + page)
                fresh = x[:, lo - first:hi - first]
                amax = fresh.abs().amax((1, 2))
                exp = torch.ceil(torch.log2(torch.clamp(amax, min=1e-300) / largest)).long().clamp(min=-126)
                # log2's own rounding: the smallest exponent that holds amax
                exp = torch.where(amax * _two(1 - exp) <= largest, (exp - 1).clamp(min=-126), exp)
                exp = torch.where(amax * _two(-exp) > largest, exp + 1, exp)
                if lo > p0:
                    was = scales[block].long() - 127
                    exp = torch.maximum(exp, was)
                    kept = pool.view(torch.uint8)[block].view(pool.dtype).double()[:, :lo - p0]
                    kept = _exact_round(kept * _two(was - exp)[:, None, None], fmt)
                    out[b, :, p0 - begin:lo - begin] = kept * _two(exp)[:, None, None]
                fresh = fresh * _two(-exp)[:, None, None]
                out[b, :, lo - begin:hi - begin] = _exact_round(fresh, fmt) * _two(exp)[:, None, None]
        got[c] = out
    return got
