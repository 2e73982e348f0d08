"""Operators of long-context serving and scoring, as cases that can be timed and compared.

  rotary   `rotary_embed`: rotary positions on the query and key heads of a fused projection's rows -- adjacent or half pairs, the whole
           head or its first dimensions, any frequencies (scaled for long contexts), an amplitude
  store    `kv4_store`: the rows of new tokens rotated, their keys and values into a cache of 4 bits (and `kv4_rows`, which reads them back)
  step     `kv4_step`: the same and attention over the cache, one new token per sequence
  attend   `kv4_attention`: attention of several new tokens per sequence over the cache (a prompt, a chunk of one, drafted tokens)
  score    `token_logprobs`: log probabilities of given tokens, entropies and the best alternatives from rows of logits

A cache row is held in 4 bits: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign; two a byte, the lower half first) and for every 32 of its
dimensions a power of two, 2^(byte - 127), the smallest for which no magnitude lies above 7 codes' units.  `run` returns stored rows as the
values they stand for.

Sizes are those of the 2B-shaped model of the benchmark and the tests (20 query heads, 5 key/value heads of 128, a vocabulary of 128256),
and generic ones.
"""
import math

import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, VOCAB = 20, 5, 128, 128256
#: magnitude of a code's lower three bits
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases -------------------------------------------------------------------------------------------------------------------------


def _rotary(name, batch, tokens, heads, extra, dim, rotary, adjacent, dtype, start, amplitude=1.0):
    return dict(name=name, kind="rotary", batch=batch, tokens=tokens, heads=heads, extra=extra, dim=dim, rotary=rotary, adjacent=adjacent, dtype=dtype,
                start=start, amplitude=amplitude)


def _cache(name, kind, batch, tokens, slots, start, heads=HEADS, kv=KV_HEADS, dim=HEAD_DIM, rotary=HEAD_DIM, adjacent=True, ragged=0, padded=0):
    """`start`: cache slots filled in front of the new tokens (sequence b: `ragged * b` fewer); `padded`: the last sequences have that many
    tokens fewer (positions of -1)."""
    return dict(name=name, kind=kind, batch=batch, tokens=tokens, slots=slots, start=start, heads=heads, kv=kv, dim=dim, rotary=rotary, adjacent=adjacent,
                ragged=ragged, padded=padded)


def _score(name, rows, vocab, dtype, top, pad=0):
    return dict(name=name, kind="score", rows=rows, vocab=vocab, dtype=dtype, top=top, pad=pad)


def listed():
    return [
        # a decode step of eight sequences at their own far positions
        _rotary("rotary_8x1", 8, 1, HEADS + KV_HEADS, KV_HEADS, HEAD_DIM, HEAD_DIM, True, "bf16", 100000),
        # a long document on float32 activations: a part of the head, half pairs, frequencies and amplitude stretched
        _rotary("rotary_fp32_1x8191", 1, 8191, 24, 0, 80, 32, False, "fp32", 40000, 1.2079),
        # prompts of 1920 tokens into an empty cache
        _cache("store_2x1920", "store", 2, 1920, 2176, 0),
        # the next chunk of several conversations, half pairs on a part of a small head
        _cache("store_7x33_d64", "store", 7, 33, 1024, 900, heads=12, kv=6, dim=64, rotary=32, adjacent=False, ragged=101),
        # one user
        _cache("step_1x384", "step", 1, 1, 384, 253),
        # a small server, requests of different lengths
        _cache("step_8x1528", "step", 8, 1, 1528, 1375, ragged=61),
        # four long documents
        _cache("step_4x32768", "step", 4, 1, 32768, 32001, ragged=1999),
        # tokens drafted ahead and checked together, eight sequences
        _cache("attend_8x5", "attend", 8, 5, 4096, 3800, ragged=333),
        # prompts of one length
        _cache("attend_2x2048", "attend", 2, 2048, 2048, 0),
        # a chunk of a long prompt, one sequence shorter than the others
        _cache("attend_3x500", "attend", 3, 500, 9000, 8001, ragged=1003, padded=77),
        # the alternatives of one sampled token
        _score("score_1x128256", 1, VOCAB, "bf16", 5),
        # a prompt's tokens under the model
        _score("score_1024x128256", 1024, VOCAB, "bf16", 20),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], uniform over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("rotary", "store", "step", "attend", "score"))
    if kind == "score":
        vocab = rng.choice((VOCAB, 32000, 50021, _spread(rng, 1000, 150000)))
        rows = _spread(rng, 1, max(1, min(1024, 130_000_000 // vocab)))
        case = _score("", rows, vocab, rng.choice(("bf16", "bf16", "fp32")), rng.choice((0, 1, 5, 20, 32)), rng.choice((0, 0, 1, 64)))
    elif kind == "rotary":
        dim = rng.choice((64, 80, 96, 128, 128, 256))
        heads = rng.choice((1, 5, 8, 12, 25, 40))
        batch = _spread(rng, 1, 64)
        case = _rotary("", batch, _spread(rng, 1, max(1, 40_000_000 // (batch * heads * dim))), heads, rng.choice((0, 1, 5)), dim, rng.choice((dim, dim // 2, 2 * (dim // 8))),
                       rng.random() < 0.5, rng.choice(("bf16", "bf16", "fp32")), _spread(rng, 1, 1_000_000), rng.choice((1.0, 1.1386, 1.2079)))
    else:
        dim = rng.choice((128, 128, 64))
        kv, group = rng.choice(((5, 4), (8, 4), (1, 8), (4, 1), (6, 2), (2, 5), (8, 8)))
        rotary, adjacent = rng.choice((dim, dim, dim // 2, dim // 4 + 2)), rng.random() < 0.5
        shape = dict(heads=kv * group, kv=kv, dim=dim, rotary=rotary, adjacent=adjacent)
        if kind == "store":
            batch = _spread(rng, 1, 16)
            tokens = _spread(rng, 1, max(1, 4000 // batch))
            start = _spread(rng, 1, 4000)
            case = _cache("", kind, batch, tokens, start + tokens + rng.randrange(50), start, ragged=rng.choice((0, start // batch)), **shape)
        elif kind == "step":
            batch = _spread(rng, 1, 64)
            start = _spread(rng, 1, min(65536, max(2, 500_000 // (batch * kv))))
            case = _cache("", kind, batch, 1, start + 1 + rng.randrange(100), start, ragged=rng.choice((0, start // batch)), padded=rng.choice((0, 0, 0, 1)), **shape)
        else:
            batch = _spread(rng, 1, 8)
            tokens = _spread(rng, 2, max(2, 40960 // max(20, kv * group) // batch))
            start = _spread(rng, 1, max(2, min(20000, 8_000_000 // (batch * tokens * kv * group) * 5)))
            case = _cache("", kind, batch, tokens, start + tokens + rng.randrange(50), start, ragged=rng.choice((0, start // batch)),
                          padded=rng.choice((0, 0, tokens // 3)), **shape)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------------------------


def _frequencies(rotary, theta=500000.0):
    """Radians a position of every pair, the slower half stretched by eight as for a context longer than the trained one."""
    pairs = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    inv = theta ** (-2.0 * pairs / rotary)
    return torch.where(pairs >= rotary // 4, inv / 8, inv)


def _starts(case):
    return [max(0, case["start"] - case["ragged"] * b) for b in range(case["batch"])]


def _tokens(case):
    """New tokens of each sequence: the last third of them is padded."""
    batch, tokens = case["batch"], case["tokens"]
    return [tokens - (case["padded"] if b >= batch - (batch + 2) // 3 else 0) for b in range(batch)]


def _positions(case):
    rows = [[start + t if t < count else -1 for t in range(case["tokens"])] for start, count in zip(_starts(case), _tokens(case))]
    return torch.tensor(rows, dtype=torch.int64).cuda()


def _rows(shape, gen, dtype=torch.bfloat16):
    """Activations with a few channels louder than the rest, as keys have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-1:], generator=gen, device="cuda") < 0.03
    return torch.where(loud, 6 * x, x).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "score":
        # peaked, as a model's logits are: a background and a few tokens well above it
        wide = torch.randn((case["rows"], case["vocab"] + case["pad"]), generator=gen, device="cuda") * 2
        above = torch.randint(0, case["vocab"], (case["rows"], 12), generator=gen, device="cuda")
        wide.scatter_add_(1, above, 6 + 4 * torch.rand(above.shape, generator=gen, device="cuda"))
        wide = wide.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        targets = torch.where(torch.rand(case["rows"], generator=gen, device="cuda") < 0.5, above[:, 0], torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda"))
        return dict(case, logits=wide[:, :case["vocab"]], targets=targets)
    if kind == "rotary":
        batch, tokens, dim = case["batch"], case["tokens"], case["dim"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        rows = _rows((batch, tokens, case["heads"] + case["extra"], dim), gen, dtype)
        pos = case["start"] + torch.arange(tokens, device="cuda")[None, :] + 11 * torch.arange(batch, device="cuda")[:, None]
        return dict(case, x=rows[:, :, :case["heads"]], pos=pos, inv_freq=_frequencies(case["rotary"]))
    batch, kv, dim, slots = case["batch"], case["kv"], case["dim"], case["slots"]
    state = dict(case, pos=_positions(case), inv_freq=_frequencies(case["rotary"]))
    parts = []
    for _ in range(2):                                   # keys, values: every slot holds a row, of this request or an earlier one
        codes = torch.empty((batch, kv, slots, dim // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((batch, kv, slots, dim // 32), dtype=torch.uint8, device="cuda")
        for b in range(batch):
            codes[b], scales[b] = _quantise(_rows((kv, slots, dim), gen).float())
        parts += [codes, scales]
    state["cache"] = tuple(parts)                        # k, k_scale, v, v_scale
    if kind == "attend":
        state["q"] = _rows((batch, case["heads"], case["tokens"], dim), gen)
    else:
        state["xqkv"] = _rows((batch * case["tokens"], (case["heads"] + 2 * kv) * dim), gen)
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------------------------


def _quantise(x):
    """float32 [..., D] -> codes uint8 [..., D / 2] and scale bytes uint8 [..., D / 32]."""
    groups = x.reshape(*x.shape[:-1], -1, 32)
    magnitude = groups.abs()
    top = magnitude.amax(-1)
    mantissa, exponent = torch.frexp(top)
    e = torch.where(mantissa > 0.875, exponent - 2, exponent - 3)
    e = torch.where(top == 0, -125, e).clamp(-125, 125)
    broken = ~torch.isfinite(top)
    unit = torch.ldexp(magnitude, -e[..., None])
    code = sum((unit >= at if even else unit > at).to(torch.uint8) for at, even in
               ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)))
    code = torch.where(broken[..., None], 0, code + 8 * torch.signbit(groups).to(torch.uint8)).to(torch.uint8).reshape(x.shape)
    return code[..., 0::2] + 16 * code[..., 1::2], torch.where(broken, 255, e + 127).to(torch.uint8)


def _dequantise(codes, scales):
    """float32 values of codes [..., D / 2] and scale bytes [..., D / 32]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    pairs = torch.stack([level.repeat(16), level.repeat_interleave(16)], -1)             # [byte][lower, upper half]
    values = pairs[codes.int()].reshape(*codes.shape[:-1], -1, 32)
    scale = torch.where(scales == 255, float("nan"), torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127))
    return (values * scale[..., None]).reshape(*codes.shape[:-1], -1)


def _turn(x, cos, sin, adjacent):
    """x [..., D] float32, its first 2 * cos.shape[-1] dimensions rotated."""
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if adjacent:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _angles(pos, inv_freq, amplitude):
    """cos, sin float32 [..., 1, pairs]: the angle in 64 bits, far positions lose nothing."""
    angle = (pos.double()[..., None] * inv_freq)[..., None, :]
    return (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()


def _plain_rotary(s):
    x = s["x"]
    return _turn(x.float(), *_angles(s["pos"], s["inv_freq"], s["amplitude"]), s["adjacent"]).to(x.dtype)


def _plain_store(s):
    """Rotated queries float32 [B, H, T, D]; the new rows into the cache."""
    batch, tokens, heads, kv, dim, pos = s["batch"], s["tokens"], s["heads"], s["kv"], s["dim"], s["pos"]
    rows = s["xqkv"].float().view(batch, tokens, heads + 2 * kv, dim)
    turned = _turn(rows[:, :, :heads + kv], *_angles(pos, s["inv_freq"], 1.0), s["adjacent"])
    k, k_scale, v, v_scale = s["cache"]
    real = pos >= 0
    b = torch.arange(batch, device=pos.device)[:, None].expand_as(pos)[real]
    at = pos[real]
    for codes, scales, new in ((k, k_scale, turned[:, :, heads:]), (v, v_scale, rows[:, :, heads + kv:])):
        codes[b, :, at], scales[b, :, at] = _quantise(new[real])
    return turned[:, :, :heads].transpose(1, 2)


def _plain_rows(s):
    """bf16 [B, T, KV, D] keys and values at the positions, NaN where there is none."""
    k, k_scale, v, v_scale = s["cache"]
    pos = s["pos"]
    b = torch.arange(pos.shape[0], device=pos.device)[:, None]
    got = []
    for codes, scales in ((k, k_scale), (v, v_scale)):
        rows = _dequantise(codes[b, :, pos.clamp(min=0)], scales[b, :, pos.clamp(min=0)])
        got.append(torch.where((pos >= 0)[..., None, None], rows, float("nan")).to(torch.bfloat16))
    return got


def _plain_attend(q, s):
    """Softmax of a row's scores over the slots up to its position, times the values: bf16 [B * T, H * D]."""
    batch, heads, tokens, dim = q.shape
    k, k_scale, v, v_scale = s["cache"]
    kv, slots = k.shape[1:3]
    keys = _dequantise(k, k_scale).transpose(2, 3).contiguous()
    scores = torch.matmul(q.float().reshape(batch, kv, heads // kv * tokens, dim), keys) * dim ** -0.5
    seen = torch.arange(slots, device=q.device) <= s["pos"][:, None, :, None]                       # [B, 1, T, S]
    scores = scores.view(batch, kv, heads // kv, tokens, slots).masked_fill_(~seen[:, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(batch, kv, heads // kv * tokens, slots), _dequantise(v, v_scale)).view(*weight.shape[:-1], dim)
    out = torch.where(total > 0, out / total, 0.0)                                                  # nothing to see: zeros
    return out.reshape(batch, heads, tokens, dim).transpose(1, 2).reshape(batch * tokens, heads * dim).to(torch.bfloat16)


def _plain_score(s):
    x, top = s["logits"].float(), s["top"]
    peak = x.amax(-1, keepdim=True)
    below = x - peak
    weight = below.exp()
    total = weight.sum(-1)
    log_total = total.log()
    got = [below.gather(1, s["targets"][:, None])[:, 0] - log_total, log_total - (weight * below).sum(-1) / total]
    if top:
        order = torch.sort(x, dim=-1, descending=True, stable=True)                                 # ties: the lowest index first
        ids = order.indices[:, :top].clone()
        got += [ids, below.gather(1, ids) - log_total[:, None]]
    return got


def run(s):
    kind = s["kind"]
    if own:
        import ternainfer_amd as T
        if kind == "rotary":
            return T.rotary_embed(s["x"], s["pos"], s["inv_freq"], amplitude=s["amplitude"], adjacent=s["adjacent"])
        if kind == "score":
            got = T.token_logprobs(s["logits"], s["targets"], top=s["top"])
            return [got.logprob, got.entropy] + ([got.top_ids, got.top_logprobs] if s["top"] else [])
        cache = T.Kv4Cache(*s["cache"])
        if kind == "attend":
            return T.kv4_attention(s["q"], s["pos"], cache)
        call = T.kv4_store if kind == "store" else T.kv4_step
        out = call(s["xqkv"], s["pos"], s["inv_freq"], cache, s["heads"], adjacent=s["adjacent"])
        return [out, *T.kv4_rows(cache, s["pos"])]
    if kind == "rotary":
        return _plain_rotary(s)
    if kind == "score":
        return _plain_score(s)
    if kind == "attend":
        return _plain_attend(s["q"], s)
    q = _plain_store(s).to(torch.bfloat16)
    return [q if kind == "store" else _plain_attend(q, s), *_plain_rows(s)]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "score":
        size = 2 if case["dtype"] == "bf16" else 4
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    if kind == "rotary":
        size = 2 if case["dtype"] == "bf16" else 4
        rows = case["batch"] * case["tokens"]
        return {"bytes": rows * (2 * case["heads"] * case["dim"] * size + 8), "flops": 3 * rows * case["heads"] * case["rotary"]}
    batch, tokens, heads, kv, dim = (case[n] for n in ("batch", "tokens", "heads", "kv", "dim"))
    row = 2 * kv * (dim // 2 + dim // 32)                # a token's keys and values in the cache
    new = batch * tokens * ((heads + 2 * kv) * dim * 2 + row + 2 * kv * dim * 2 + 8)     # rows in, cache rows out, their values back
    if kind == "store":
        return {"bytes": new + batch * tokens * heads * dim * 2, "flops": 3 * batch * tokens * (heads + kv) * case["rotary"]}
    counts = list(zip(_starts(case), _tokens(case)))
    seen = sum(count * start + count * (count + 1) // 2 for start, count in counts)      # (token, slot) pairs
    read = sum(start + count for start, count in counts if count) * row
    out = batch * tokens * heads * dim * 2
    return {"bytes": read + out + (new if kind == "step" else out), "flops": 4 * seen * heads * dim}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------------------------


def _exact_values(codes, scales):
    """float64: sign, exponent and mantissa of each code taken apart."""
    nibble = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int64)
    exponent, mantissa = (nibble >> 1) & 3, (nibble & 1).double()
    size = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2.0 ** (exponent - 1).double())
    return torch.where(nibble >= 8, -size, size) * (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)


def _exact_rounded(x):
    """float64 [..., D] -> the values that the cache keeps of it."""
    g = x.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    step = 2.0 ** torch.ceil(torch.log2(top.clamp(min=2.0 ** -120) / 7) - 1e-12).clamp(-125, 125)
    u = (g.abs() / step).clamp(max=6.0)
    grid = torch.where(u < 2, 0.5, torch.where(u < 4, 1.0, 2.0))
    return (torch.sign(g) * torch.round(u / grid) * grid * step).flatten(-2)            # (round: halves to even)


def _exact_turn(x, pos, inv_freq, adjacent, amplitude=1.0):
    """As multiplication by exp(i angle)."""
    half = inv_freq.numel()
    t = x[..., :2 * half]
    z = torch.view_as_complex(t.unflatten(-1, (half, 2)).contiguous()) if adjacent else torch.complex(t[..., :half].contiguous(), t[..., half:].contiguous())
    angle = pos.double()[..., None, None] * inv_freq
    z = z * torch.polar(torch.full_like(angle, amplitude), angle)
    t = torch.view_as_real(z).flatten(-2) if adjacent else torch.cat([z.real, z.imag], -1)
    return torch.cat([t, x[..., 2 * half:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_turn(s["x"].double(), s["pos"], s["inv_freq"], s["adjacent"], s["amplitude"])
    if kind == "score":
        parts = []
        for x, target in zip(s["logits"].split(64), s["targets"].split(64)):
            logp = torch.log_softmax(x.double(), -1)
            found = [logp.gather(1, target[:, None])[:, 0], -(logp.exp() * logp).sum(-1)]
            parts.append(found + ([torch.topk(logp, case["top"]).values] if case["top"] else []))
        got = [torch.cat(p) for p in zip(*parts)]
        return got if not case["top"] else [got[0], got[1], None, got[2]]
    batch, tokens, heads, kv, dim, pos = s["batch"], s["tokens"], s["heads"], s["kv"], s["dim"], s["pos"]
    k, k_scale, v, v_scale = s["cache"]
    new = []
    if kind == "attend":
        q = s["q"].double().transpose(1, 2)
    else:
        rows = s["xqkv"].double().view(batch, tokens, heads + 2 * kv, dim)
        q = _exact_turn(rows[:, :, :heads], pos, s["inv_freq"], s["adjacent"])
        new = [_exact_rounded(_exact_turn(rows[:, :, heads:heads + kv], pos, s["inv_freq"], s["adjacent"])), _exact_rounded(rows[:, :, heads + kv:])]
    shown = [torch.where((pos >= 0)[..., None, None], n, float("nan")) for n in new]
    if kind == "store":
        return [q.transpose(1, 2), *shown]
    if kind == "step":
        q = q.to(torch.bfloat16).double()                # what attention takes are the rows as they are handed on
    out = torch.zeros((batch, tokens, heads, dim), dtype=torch.float64, device="cuda")
    for b in range(batch):                               # one sequence and kv head at a time: 64-bit scores are large
        for h in range(kv):
            n = int(pos[b].max()) + 1
            if n < 1:
                continue
            key, value = _exact_values(k[b, h, :n], k_scale[b, h, :n]), _exact_values(v[b, h, :n], v_scale[b, h, :n])
            if new:
                key[pos[b]], value[pos[b]] = new[0][b, :, h], new[1][b, :, h]
            own_heads = slice(h * (heads // kv), (h + 1) * (heads // kv))
            scores = torch.matmul(q[b, :, own_heads], key.T.contiguous()) / math.sqrt(dim)          # [T, G, n]
            scores = scores.masked_fill(torch.arange(n, device="cuda") > pos[b][:, None, None], float("-inf"))
            out[b, :, own_heads] = torch.matmul(torch.softmax(scores, -1).nan_to_num(0.0), value)
    return [out.reshape(batch * tokens, heads * dim), *shown] if kind == "step" else out.reshape(batch * tokens, heads * dim)
