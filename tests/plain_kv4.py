"""A cache held in 4 bits, in plain torch: how numbers are stored and read, and attention over them in 64 bits."""
from __future__ import annotations

import math

import torch

LARGEST, NOT_FINITE = 246, 255


def scale_table(device="cpu") -> torch.Tensor:
    """The scale of every byte that is written, float64; NaN for the others."""
    values = [((8 + (b & 7)) * 2.0 ** ((b >> 3) - 18) if b >= 8 else b * 2.0 ** -17) / 64.0 for b in range(LARGEST + 1)]
    return torch.tensor(values + [math.nan] * (255 - LARGEST), dtype=torch.float64, device=device)


def store(x: torch.Tensor):
    """(codes, scale bytes) of float32 ``[..., dim]``."""
    groups = x.float().unflatten(-1, (-1, 16))
    most = groups.abs().amax(-1)
    finite = torch.isfinite(groups).all(-1)
    most = torch.where(finite, most, torch.zeros_like(most))
    table = scale_table(x.device)[:LARGEST + 1].float().contiguous()
    byte = torch.searchsorted(table * 7.0, most).clamp(max=LARGEST)
    inverse = torch.where(byte > 0, 1.0 / table[byte], torch.zeros_like(most))
    steps = torch.where(finite[..., None], groups, torch.zeros_like(groups)) * inverse[..., None]
    code = steps.round().clamp(-7, 7).to(torch.int16).flatten(-2) + 8
    codes = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    return codes, torch.where(finite, byte, torch.full_like(byte, NOT_FINITE)).to(torch.uint8)


def read(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What codes and scale bytes stand for, float64."""
    code = torch.stack([codes % 16, codes // 16], dim=-1).flatten(-2).double() - 8.0
    return code * scale_table(codes.device)[scale.long()].repeat_interleave(16, dim=-1)


def rotate(x: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Heads ``[tokens, heads, dim]`` rotated in float32, every product and sum rounded."""
    if cos_sin is None:
        return x
    cos, sin = cos_sin[positions.long()][:, None].unbind(-1)
    low, high = x.chunk(2, dim=-1)
    return torch.cat([low * cos - high * sin, low * sin + high * cos], dim=-1)


def attention(q, keys, values, before: int, scale: float, window: int = 0):
    """One sequence: queries ``[new, heads, dim]`` over ``[kv_heads, positions, dim]``, all float64.  Returns the result, the
    weights' sum over |values|, which rounding errors of probabilities are relative to, and the plain sum of |values| that a row sees."""
    new, heads, dim = q.shape
    kv = keys.shape[0]
    at = torch.arange(before, before + new, device=q.device)[:, None]
    key = torch.arange(keys.shape[1], device=q.device)[None, :]
    hidden = key > at
    if window > 0:
        hidden = hidden | (key <= at - window)
    out, spread, whole = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    for h in range(heads):
        k, v = keys[h // (heads // kv)], values[h // (heads // kv)]
        score = ((q[:, h] @ k.T) * scale).masked_fill(hidden, -math.inf)
        weight = torch.softmax(score, dim=-1)
        masked = weight.masked_fill(hidden, 0.0)
        for to, what, masked in ((out, v, masked), (spread, v.abs(), masked), (whole, v.abs(), (~hidden).double())):
            # (a masked key counts for nothing, whatever it holds)
            clean = torch.nan_to_num(what, nan=0.0)
            to[:, h] = masked @ clean
            spoiled = ((~hidden).double() @ torch.isnan(what).double()) > 0
            to[:, h] = torch.where(spoiled, math.nan, to[:, h])
    return out, spread, whole
