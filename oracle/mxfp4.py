"""MXFP4 on the CPU in 64 bits, from the format's definition.

32 consecutive values x share the scale 2^e, e = floor(log2(max|x|)) - 2 kept between -125
and 125 (-125 for zeros), and each is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (and their
negatives) times it, a tie going to the even code. A block with a NaN or an infinity is NaN
throughout: scale byte 255, codes 0.
"""

from __future__ import annotations

import numpy as np
import torch

BLOCK = 32
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(..., K) to packed codes (..., K/2) and scale bytes (..., K/32), uint8."""

    blocks = x.detach().cpu().double().numpy().reshape(-1, BLOCK)
    codes = np.zeros(blocks.shape, dtype=np.uint8)
    scales = np.full(blocks.shape[0], 255, dtype=np.uint8)
    fine = np.isfinite(blocks).all(axis=1)
    largest = np.abs(blocks[fine]).max(axis=1, initial=0.0)
    # frexp: largest = m 2^e with m in [0.5, 1), so floor(log2) is e - 1, exactly.
    exponent = np.where(largest > 0, np.frexp(largest)[1] - 1 - 2, -125).clip(-125, 125)
    scaled = blocks[fine] / np.ldexp(1.0, exponent)[:, None]
    distance = np.abs(np.abs(scaled)[..., None] - MAGNITUDES)
    nearest = distance.min(axis=-1, keepdims=True)
    # Of two codes at the same distance the even one (a key of half a code for odd ones).
    order = np.arange(8) + np.where(np.arange(8) % 2, 100, 0)
    code = np.where(distance == nearest, order, 1000).argmin(axis=-1)
    codes[fine] = code | (np.signbit(scaled) << 3)
    scales[fine] = exponent + 127
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    lead = x.shape[:-1]
    return (torch.from_numpy(packed).reshape(*lead, x.shape[-1] // 2),
            torch.from_numpy(scales).reshape(*lead, x.shape[-1] // BLOCK))


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values (..., K) of packed codes and scale bytes, float64."""

    raw = codes.detach().cpu().view(torch.uint8).numpy()
    power = scales.detach().cpu().view(torch.uint8).numpy().astype(np.int64)
    width = 2 * raw.shape[-1]
    pair = np.stack((raw & 15, raw >> 4), axis=-1).reshape(*raw.shape[:-1], width)
    value = MAGNITUDES[pair & 7] * np.where(pair & 8, -1.0, 1.0)
    value = value.reshape(*power.shape, BLOCK)
    scale = np.where(power == 255, np.nan, np.ldexp(1.0, power - 127))
    return torch.from_numpy((value * scale[..., None]).reshape(*raw.shape[:-1], width))


def attention(query: torch.Tensor, keys: torch.Tensor, vals: torch.Tensor,
              scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Causal attention of query (T, Hq, Dh), the last T positions of keys and vals
    (S, Hkv, Dh), in 64 bits: the output, and for tolerances sum p |v| (same shape) and the
    largest |scores|'s bound, scale * sum |q_d k_d|, of each (T, Hq)."""

    t, hq, dh = query.shape
    s, hkv, _ = keys.shape
    q = query.detach().cpu().double()
    k = keys.double().repeat_interleave(hq // hkv, dim=1)
    v = vals.double().repeat_interleave(hq // hkv, dim=1)
    scale = dh ** -0.5 if scale is None else scale
    scores = torch.einsum("thd,shd->ths", q, k) * scale
    seen = torch.arange(s)[None] <= torch.arange(s - t, s)[:, None]
    probs = scores.masked_fill(~seen[:, None], -torch.inf).softmax(dim=-1)
    size = torch.einsum("thd,shd->ths", q.abs(), k.abs()) * abs(scale)
    size = size.masked_fill(~seen[:, None], 0.0).amax(dim=-1)
    return (torch.einsum("ths,shd->thd", probs, v), torch.einsum("ths,shd->thd", probs, v.abs()),
            size)
