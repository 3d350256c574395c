"""Matrices in 8 bits in plain numpy, 64 bits: block-scaled e4m3 payloads and their products.  A block is 128
columns of `block` rows; its values are payload * 2^(code - 127), code 255 standing for NaN."""
from __future__ import annotations

import numpy as np
import torch

from sandyrt_amd import ops
from tests.quant_reference import code_of, round_payload


def quantise(x, block):
    """(payloads, codes) of x [rows, k], float64 holding x's values exactly."""
    rows, k = x.shape
    payload, code = np.zeros((rows, k)), np.zeros((-(-rows // block), -(-k // 128)), np.int64)
    for i in range(code.shape[0]):
        for j in range(code.shape[1]):
            part = x[i * block:(i + 1) * block, 128 * j:128 * (j + 1)]
            c = code[i, j] = code_of(np.abs(part).max(), "e4m3")
            if c != 255:
                payload[i * block:(i + 1) * block, 128 * j:128 * (j + 1)] = round_payload(part * 2.0 ** (127 - c), "e4m3")
    return payload, code


def values(payload, code):
    """What payloads [rows, k] with their codes stand for."""
    rows, k = payload.shape
    block = 1 if code.shape[0] == rows else 128
    each = code.repeat(block, 0)[:rows].repeat(128, 1)[:, :k]
    return np.where(each == 255, np.nan, payload * np.exp2(np.where(each == 255, 0, each) - 127.0))


def held(q):
    """What an ops.QuantMatrix [rows, k] stands for."""
    return values(q.payload.cpu().float().double().numpy(), q.scales.cpu().numpy().astype(np.int64))


def whole(rng, shape, block, pad=16, batch_gap=0):
    """A QuantMatrix of payloads -8 .. 8 and scales 1/2, 1 or 2: products and sums of up to 5600 of them are exact in
    f32 in any order (terms are whole multiples of 1/4 up to 256).  Rows are `pad` bytes further apart than they need,
    and whatever lies between them is NaN."""
    *lead, rows, k = shape
    pitch = (k + 15) // 16 * 16 + pad
    payload = torch.full((*lead, rows + batch_gap, pitch), 0x7f, dtype=torch.uint8)
    payload[..., :rows, :k] = torch.from_numpy(rng.integers(-8, 9, shape)).float().to(torch.float8_e4m3fn).view(torch.uint8)
    code = torch.from_numpy(rng.integers(126, 129, (*lead, -(-rows // block), -(-k // 128)))).to(torch.uint8)
    return ops.QuantMatrix(payload.cuda().view(torch.float8_e4m3fn)[..., :rows, :k], code.cuda())
