"""Long requests: rotary positions at any distance, a key/value cache in 4 bits, log probabilities of tokens.

What stands beside the bf16 cache (8192 slots) and the greedy step of the other modules.  Kernels and their conventions: csrc/rotary_kernel.h,
csrc/kv4_format.h and the files around them, csrc/logprobs_kernel.h.  Every function takes tensors of one GPU, which need not be the current one, and
enqueues on that GPU's current stream; it raises ValueError (TypeError where an argument is no tensor) for what the kernels do not take, before
anything is enqueued.  None has a backward pass.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib


def rotary_frequencies(rotary_dim: int, theta: float = 500000.0, scaling: Optional[dict] = None, device="cuda"):
    """(inv_freq, amplitude): the angle in radians that each of rotary_dim / 2 pairs turns a position, float64, and the factor on cosines and sines.
    Pair j turns theta ** (-2 j / rotary_dim); `scaling` stretches that for contexts `factor` times longer than the trained one:
      {"type": "linear", "factor"}       every frequency divided by it (position interpolation)
      {"type": "ntk", "factor"}          theta raised so that the slowest pair is divided by it and the fastest stays
      {"type": "wavelength", "factor", "original_max_position", "low_freq_factor" = 1, "high_freq_factor" = 4}
                                         pairs that turn less than low_freq_factor times within the original length are divided, those that
                                         turn more than high_freq_factor times stay, between them linearly in the number of turns
      {"type": "yarn", "factor", "original_max_position", "beta_fast" = 32, "beta_slow" = 1, "amplitude" = 0.1 ln(factor) + 1}
                                         divided, kept, and between them by a ramp over the pair's index; a larger amplitude (Peng et al.,
                                         "YaRN: Efficient Context Window Extension of Large Language Models")"""
    if rotary_dim < 2 or rotary_dim % 2 or not 0 < theta < math.inf:
        raise ValueError(f"rotary_frequencies: unsupported rotary_dim={rotary_dim} theta={theta}")
    inv = [theta ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)]
    amplitude = 1.0
    if scaling is not None:
        known = {"linear": (), "ntk": (), "wavelength": ("low_freq_factor", "high_freq_factor"), "yarn": ("beta_fast", "beta_slow", "amplitude")}
        kind = scaling.get("type")
        need = ("factor",) + (("original_max_position",) if kind in ("wavelength", "yarn") else ())
        if kind not in known or not set(need) <= set(scaling) or set(scaling) - {"type", *need, *known[kind]}:
            raise ValueError(f"rotary_frequencies: unsupported scaling {scaling}")
        factor = float(scaling["factor"])
        if not 1.0 <= factor < math.inf:
            raise ValueError(f"rotary_frequencies: a factor of {factor}")
        if kind == "linear":
            inv = [f / factor for f in inv]
        elif kind == "ntk":
            if rotary_dim > 2:
                stretched = theta * factor ** (rotary_dim / (rotary_dim - 2))
                inv = [stretched ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)]
        elif kind == "wavelength":
            length, low, high = float(scaling["original_max_position"]), float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
            if not 0 < low < high or not length > 0:
                raise ValueError(f"rotary_frequencies: unsupported scaling {scaling}")
            keep = [min(1.0, max(0.0, (length * f / (2 * math.pi) - low) / (high - low))) for f in inv]
            inv = [k * f + (1 - k) * f / factor for k, f in zip(keep, inv)]
        else:
            length, fast, slow = float(scaling["original_max_position"]), float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
            if not 0 < slow < fast or not length > 0 or theta == 1:
                raise ValueError(f"rotary_frequencies: unsupported scaling {scaling}")
            pair = lambda turns: rotary_dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))     # that turns so often within the length
            first, last = max(0, math.floor(pair(fast))), min(rotary_dim - 1, math.ceil(pair(slow)))
            ramp = [min(1.0, max(0.0, (j - first) / max(last - first, 0.001))) for j in range(rotary_dim // 2)]
            inv = [f / factor * r + f * (1 - r) for r, f in zip(ramp, inv)]
            amplitude = float(scaling.get("amplitude", 0.1 * math.log(factor) + 1.0))
    return torch.tensor(inv, dtype=torch.float64, device=device), amplitude


def rotary_embed(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, *, amplitude: float = 1.0, adjacent: bool = True,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions on x [B, T, H, D] (bfloat16 or float32, any strides: a view of a fused projection's rows takes queries and keys in one
    call).  pos int64 [T] or [B, T]; inv_freq float64 [pairs] (`rotary_frequencies`).  Pair j of a head -- dimensions 2j and 2j + 1 when
    `adjacent`, else j and j + pairs -- turns by pos * inv_freq[j], an angle formed in 64 bits; the dimensions from 2 * pairs on stay.
    `out`: x itself, or rows that lie apart from it, from their first element to their last.  Fewer than 2^24 tokens (more where a workgroup takes several: few heads, or T = 1)."""
    return _lib.native().rotary_embed(x, pos, inv_freq, amplitude, adjacent, out)


class Kv4Cache(NamedTuple):
    """Keys and values in 4 bits: codes uint8 [B, KV, S, D / 2] (e2m1, two a byte) and scale bytes uint8 [B, KV, S, D / 32] -- 4.25 bits a value,
    against 16 of the bf16 cache.  A value is code * 2 ** (byte - 127); include/ternaspmm.h has the rule by which they are chosen."""
    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, batch: int, kv_heads: int, slots: int, head_dim: int, device="cuda") -> "Kv4Cache":
        """A cache without rows (zeros; the attention does not depend on what unwritten slots hold)."""
        if head_dim not in (64, 128):
            raise ValueError(f"Kv4Cache: heads of 64 or 128 dimensions, not {head_dim}")
        make = lambda width: torch.zeros((batch, kv_heads, slots, width), dtype=torch.uint8, device=device)
        return cls(make(head_dim // 2), make(head_dim // 32), make(head_dim // 2), make(head_dim // 32))


def kv4_store(xqkv: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, cache: Kv4Cache, n_heads: int, *, amplitude: float = 1.0,
              adjacent: bool = True) -> torch.Tensor:
    """The rows xqkv bf16 [B * T, (H + 2 KV) D] of T new tokens per sequence: rotary positions on queries and keys (as `rotary_embed`), keys and values
    into slots `pos` (int64 [T] or [B, T]) of the cache.  Returns the queries, bf16 [B, H, T, D].  A position outside the cache -- -1 for padding --
    stores nothing.  The positions of one sequence have to differ."""
    return _lib.native().kv4_store(xqkv, pos, inv_freq, amplitude, *cache, n_heads, adjacent)


def kv4_rows(cache: Kv4Cache, pos: torch.Tensor):
    """(keys, values) that slots `pos` (int64 [T] or [B, T]) stand for: bf16 [B, T, KV, D] each, exactly; NaN for a position outside the cache."""
    return _lib.native().kv4_rows(*cache, pos)


def kv4_attention(q: torch.Tensor, pos: torch.Tensor, cache: Kv4Cache, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of q bf16 [B, H, T, D] over the slots 0 .. pos of the cache: bf16 [B * T, H * D].  scale: D ** -0.5 by default.  A negative position
    sees nothing and gives zeros, one past the cache NaN."""
    return _lib.native().kv4_attention(q, pos, *cache, scale)


def kv4_step(xqkv: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, cache: Kv4Cache, n_heads: int, *, amplitude: float = 1.0,
             adjacent: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """One new token per sequence: `kv4_store` and `kv4_attention` in one launch (two where the slots are split; their own launches for some shapes of
    more than 32 query heads a kv head), with their bits.  xqkv bf16 [B, (H + 2 KV) D], pos int64 [1] or [B, 1]; returns bf16 [B, H * D]."""
    return _lib.native().kv4_step(xqkv, pos, inv_freq, amplitude, *cache, n_heads, adjacent, scale)


class TokenLogprobs(NamedTuple):
    """logprob float32 [M] of the given tokens (None without), entropy float32 [M] in nats; top_ids int64 and top_logprobs float32 [M, top] (None
    without)."""
    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """Of every row of logits [M, V] (bfloat16 or float32, rows any distance apart): the log probability of its token in `targets` (int64 [M]; NaN
    for one outside the vocabulary, as -1 for padding), the entropy, and the `top` (at most 64) likeliest tokens -- equal logits by lower index,
    NaN last -- with theirs.  One pass over the logits; V up to 2^19, M below 2^24.  A row with NaN or +inf, or of -inf alone, has NaN for its probabilities and entropy."""
    return TokenLogprobs(*_lib.native().token_logprobs(logits, targets, top))
