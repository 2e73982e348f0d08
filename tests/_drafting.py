"""Plain implementations in 64 bits of the operators in ternainfer_amd/drafting.py and int8_linear.py, for the tests of them."""
from __future__ import annotations

import torch

HALF_FP32, HALF_BF16 = 2.0 ** -24, 2.0 ** -8            # a rounding, relative


def lines(parents):
    """Of every node of one sequence (a list of parents), itself and its ancestors from the root on; none for padding."""
    out = []
    for i, p in enumerate(parents):
        out.append([i] if p == -1 else out[p] + [i] if 0 <= p < i and out[p] else [])
    return out


def words_of(line, words):
    bits = sum(1 << j for j in line)
    signed = lambda w: w - (1 << 64) if w >> 63 else w
    return [signed(bits >> (64 * w) & (1 << 64) - 1) for w in range(words)]


def tree(parents):
    """(mask, depth) of parents int64 [B, T], on the CPU."""
    words = (parents.shape[1] + 63) // 64
    all_lines = [lines(p) for p in parents.tolist()]
    mask = torch.tensor([[words_of(line, words) for line in ls] for ls in all_lines], dtype=torch.int64).view(*parents.shape, words)
    return mask, torch.tensor([[len(line) - 1 for line in ls] for ls in all_lines], dtype=torch.int64).view(parents.shape)


def random_parents(batch, nodes, seed, padding=0.0):
    """Trees of short and long branches; some nodes are none."""
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *shape: torch.rand(shape, generator=gen)
    at = torch.arange(nodes)
    parents = torch.where(at == 0, -1, (at - 1 - (rand(batch, nodes) ** 3 * at).long()).clamp(min=0))
    return torch.where((rand(batch, nodes) < padding) & (at > 0), torch.randint(-9, -1, (batch, nodes), generator=gen), parents)


def accept(logits, tokens, parents):
    """(path, count, next) of logits [B, T, V], as lists."""
    out = []
    for x, tok, par in zip(logits.float().cpu(), tokens.tolist(), parents.tolist()):
        best = []
        for row in x.tolist():
            top, idx = -float("inf"), 0
            for i, v in enumerate(row):                  # NaN never wins, the first of equals does
                if v > top:
                    top, idx = v, i
            best.append(idx)
        path = [0] if par[0] == -1 else []
        while path:
            child = [i for i in range(path[-1] + 1, len(par)) if par[i] == path[-1] and tok[i] == best[path[-1]]]
            if not child:
                break
            path.append(child[0])
        out.append((path + [-1] * (len(par) - len(path)), len(path), best[path[-1]] if path else -1))
    return [list(x) for x in zip(*out)]


def attention(q, k, v, start, mask, scale):
    """q bf16 [B, H, T, D], k and v bf16 [B, KV, S, D], start [B], mask [B, T, W] -> (out float64 [B, T, H, D], tolerance).  The tolerance: the output's rounding, and
    (2 ds + rounding + n 2^-23) sum p |v|, where ds = (D + 4) 2^-24 |scale| max sum |q| |k| bounds a score's error (a sum of D products in fp32), in numerator and
    denominator, n 2^-23 the sums over n slots, their parts and the rescalings, and `rounding` the exponential's 2^-20 with the probabilities' own, in numerator and
    denominator: in two bf16 2^-15 in the numerator up to 64 query rows a kv head (2^-14 covers it and the exponential), one bf16 beyond: 2 * 2^-8.  Below the normal numbers nothing is
    promised: a term under 2^-126 of the sum, which is 1 at least, may be lost, by itself, in its low half and in its part's weight: n 2^-124 max |v|."""
    b, h, t, d = q.shape
    kv, slots = k.shape[1:3]
    rounding = 2.0 ** -14 + (2 * HALF_BF16 if t * (h // kv) > 64 else 0.0)
    out = torch.zeros((b, t, h, d), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    bits = mask.cpu().tolist()
    for i in range(b):
        first = int(start[i])
        for n in range(t):
            seen = [j for j in range(t) if bits[i][n][j // 64] >> (j % 64) & 1]
            if first < 0 or not seen:
                continue
            if first > slots or first + max(seen) >= slots:
                out[i, n] = float("nan")
                continue
            at = torch.tensor(list(range(first)) + [first + j for j in seen], device=q.device)
            for kvh in range(kv):
                key, value = k[i, kvh].index_select(0, at).double(), v[i, kvh].index_select(0, at).double()
                rows = slice(kvh * (h // kv), (kvh + 1) * (h // kv))
                x = q[i, rows, n].double()
                p = torch.softmax((x @ key.T) * scale, -1)
                out[i, n, rows] = p @ value
                ds = (d + 4) * HALF_FP32 * abs(scale) * (x.abs() @ key.abs().T).amax(-1, keepdim=True)
                tol[i, n, rows] = HALF_BF16 * out[i, n, rows].abs() + (2 * ds + rounding + 2 * len(at) * HALF_FP32) * (p @ value.abs()) \
                    + len(at) * 2.0 ** -124 * value.abs().nan_to_num(0.0, 0.0).max()
    return out, tol


def quantise(x):
    """(integers int8, scale fp32) of rows x [R, K]: fp32 operations, each rounded once (formed in 64 bits, which a quotient of two fp32 survives)."""
    x = x.float()
    top = x.abs().amax(-1)
    finite, zero = torch.isfinite(top), top < 2.0 ** -120
    by = torch.where(finite & ~zero, 127.0 / top.double(), 0.0).float()
    q = torch.where(finite[:, None], torch.round(x * by[:, None]), 0.0)
    scale = torch.where(zero, 0.0, torch.where(finite, top.double() / 127.0, float("nan"))).float()
    return torch.where(finite[:, None], q, torch.zeros_like(q)).to(torch.int8), scale


def unpack(packed, rows, columns):
    """int8 [rows, columns] of packed blocks."""
    blocks = 2 * ((columns + 127) // 128)
    x = packed.view(torch.int8).view(-1, blocks, 4, 16, 16)                  # band, block, piece, row, column
    x = x.permute(0, 3, 1, 2, 4).reshape(-1, 64 * blocks)
    assert not x[:rows, columns:].any()
    return x[:rows, :columns]


def linear(xq, xs, wq, ws, dtype):
    """The product: sums exact, then the three fp32 operations that the operator is defined by."""
    total = xq.double() @ wq.double().T.contiguous()                         # (below 2^53: exact)
    return (total.float() * xs[:, None] * ws[None, :]).to(dtype)
