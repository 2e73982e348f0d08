"""Plain implementations in 64 bits of the operators in ternainfer_amd/long_context.py, for the tests of them."""
from __future__ import annotations

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
HALF_FP32, HALF_BF16 = 2.0 ** -24, 2.0 ** -8            # a rounding, relative


def power_of_two(e):
    """2 ** e, exactly (the power of a float64 tensor, and torch.ldexp with it, is not): its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def turned(x, pos, inv_freq, amplitude, adjacent):
    """x float64 [B, T, H, D], pos [T] or [B, T] -> (turned, bound): `bound` = amplitude * (|a| + |b|) of each element's pair, 0 where it is copied."""
    half = inv_freq.numel()
    pos = pos.double() if pos.dim() == 2 else pos.double()[None]
    angle = (pos[..., None] * inv_freq.double())[:, :, None]
    c, s = angle.cos() * amplitude, angle.sin() * amplitude
    y, bound = x.clone(), torch.zeros_like(x)
    first = (slice(0, 2 * half, 2) if adjacent else slice(0, half))
    second = (slice(1, 2 * half, 2) if adjacent else slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    bound[..., first] = bound[..., second] = abs(amplitude) * (a.abs() + b.abs())
    return y, bound


def scale_exponents(amax):
    """The smallest e in -125 .. 125 with amax <= 7 * 2^e (float64)."""
    e = torch.full_like(amax, 125.0)
    for at in range(124, -126, -1):
        e = torch.where(amax <= 7 * 2.0 ** at, float(at), e)    # (Python's power of two numbers: exact)
    return e


def round_codes(x, e):
    """x float64 [..., D], e [..., D / 32]: the values of the nearest codes, ties to the even code, at most 6 units."""
    unit = power_of_two(e).repeat_interleave(32, -1)
    u = (x.abs() / unit)[..., None]
    levels = LEVELS.to(x.device)
    distance = (u - levels).abs()
    nearest = distance.amin(-1, keepdim=True)
    tied = distance == nearest
    even = torch.arange(8, device=x.device) % 2 == 0
    pick = torch.where(tied.sum(-1, keepdim=True) > 1, tied & even, tied)
    value = (pick * levels).sum(-1)
    return torch.where(torch.signbit(x), -value, value) * unit


def values(codes, scales):
    """float64 [..., D] of codes uint8 [..., D / 2] and scale bytes [..., D / 32]; NaN under byte 255."""
    nibble = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    level = LEVELS.to(codes.device)[nibble & 7]
    unit = torch.where(scales == 255, float("nan"), power_of_two(scales.double() - 127)).repeat_interleave(32, -1)
    return torch.where(nibble >= 8, -level, level) * unit


def random_cache(batch, kv, slots, dim, seed, device="cuda"):
    """Codes and scale bytes of every kind a cache holds, magnitudes around 1."""
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda low, high, width: torch.randint(low, high, (batch, kv, slots, width), generator=gen, device=device, dtype=torch.uint8)
    return rand(0, 256, dim // 2), rand(123, 127, dim // 32), rand(0, 256, dim // 2), rand(123, 128, dim // 32)


def attention(q, pos, cache, scale):
    """q bf16 [B, H, T, D] -> (out float64 [B, T, H, D], tolerance).  The tolerance: the output's rounding, and (2 ds + 2^-15 + n 2^-24) sum p |v|, where
    ds = (D + 4) 2^-24 scale max sum |q| |k| bounds a score's error (a sum of D products in fp32) -- it enters numerator and denominator --, 2^-15 the
    exponential's and that of probabilities in two bf16, n 2^-24 the sums over n slots.  Below the normal numbers nothing is promised: a probability and its two parts
    may each lose 2^-126 absolutely where the largest is held at 2^-26 (so that no sum of the largest values overflows): of it 2^-100, n slots n 2^-98 max |v|.
    Probabilities in fp16: 2^-11 relative in numerator and denominator each, and 2^-37 absolutely below 2^-26 of the largest (2^-25, held at 2^12)."""
    b, h, t, d = q.shape
    rounding, below = 2 * 2.0 ** -11 + 2.0 ** -15, 2.0 ** -37
    k, v = values(cache[0], cache[1]), values(cache[2], cache[3])
    kv, s = k.shape[1:3]
    at = pos if pos.dim() == 2 else pos[None].expand(b, t)
    out = torch.zeros((b, t, h, d), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for i in range(b):
        for j in range(h):
            for n in range(t):
                last = int(at[i, n])
                if last < 0:
                    continue
                if last >= s:
                    out[i, n, j] = math.nan
                    continue
                key, value = k[i, j // (h // kv), :last + 1], v[i, j // (h // kv), :last + 1]
                x = q[i, j, n].double()
                p = torch.softmax((key * x).sum(-1) * scale, 0)
                out[i, n, j] = (p[:, None] * value).sum(0)
                ds = (d + 4) * HALF_FP32 * abs(scale) * float((key.abs() * x.abs()).sum(-1).max())
                tol[i, n, j] = HALF_BF16 * out[i, n, j].abs() + (2 * ds + rounding + (last + 1) * HALF_FP32) * (p[:, None] * value.abs()).sum(0) \
                    + (last + 1) * below * value.abs().nan_to_num(0.0).max()
    return out, tol


def same_or_near(got, want, tolerance):
    """NaN where NaN is wanted, else within the tolerance; the largest excess (<= 0: fine)."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    excess = ((got - want).abs() - tolerance)[fine]
    return float(excess.max()) if excess.numel() else 0.0
