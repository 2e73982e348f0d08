"""Operators of decoding with drafted tokens, as cases that can be timed and compared.

A step of such a decoder runs a tree of drafted tokens through the model at once, next to the token that is certain (node 0, the root), keeps the
branch that the model itself would have taken, and drops the rest.

  tree     `tree_attention`: attention of a tree's nodes over the cache: every slot in front of the tree, and the node's ancestors and itself
  accept   `tree_accept`: from the nodes' logits the branch that greedy decoding takes and the token behind it (and `draft_tree`: the next
           step's masks and depths from its parents)
  move     `cache_move`: the accepted nodes' keys and values to the slots behind the text, in the caches of all layers
  linear   `int8_linear`: a matrix product in 8-bit integers, one scale a token and one a channel: the projection to the vocabulary of all nodes, or
           any other; rows in bfloat16 are quantised within the call, rows in 8 bits are taken as they are

Node i's key and value lie in slot `start + i` of its sequence.  `parents[i]` is a node before i, -1 for a root, anything else for a node that is
none (padding).  A mask is a row of 64-bit words, bit j for node j; a row without a bit is padding and sees nothing.

Sizes are those of the 2B-shaped model of the benchmark and the tests (20 query heads, 5 key/value heads of 128, rows of 2560, a gate and up
projection of 13824, a vocabulary of 128256, 30 layers), and generic ones.
"""
import math

import torch

own = False

HEADS, KV_HEADS, HEAD_DIM, DIM, GATE_UP, VOCAB, LAYERS = 20, 5, 128, 2560, 13824, 128256, 30


# ---- cases -------------------------------------------------------------------------------------------------------------------------


def _tree(name, batch, nodes, start, slots, heads=HEADS, kv=KV_HEADS, dim=HEAD_DIM, ragged=0, padded=0, idle=0):
    """`start`: slots in front of the tree (sequence b: `ragged * b` fewer); `padded`: the last third of the sequences has that many nodes fewer;
    `idle`: so many sequences at the end have none."""
    return dict(name=name, kind="tree", batch=batch, nodes=nodes, start=start, slots=slots, heads=heads, kv=kv, dim=dim, ragged=ragged, padded=padded, idle=idle)


def _accept(name, batch, nodes, vocab, dtype):
    return dict(name=name, kind="accept", batch=batch, nodes=nodes, vocab=vocab, dtype=dtype)


def _move(name, batch, nodes, slots, kv=KV_HEADS, dim=HEAD_DIM, layers=LAYERS):
    return dict(name=name, kind="move", batch=batch, nodes=nodes, slots=slots, kv=kv, dim=dim, layers=layers)


def _linear(name, rows, n, k, given, out):
    """`given`: the rows' type, bf16 or int8; `out`: bf16 or fp32."""
    return dict(name=name, kind="linear", rows=rows, n=n, k=k, given=given, out=out)


def listed():
    return [
        # one user, a small tree behind a short text
        _tree("tree_1x8", 1, 8, 301, 384),
        # one long document, a full tree
        _tree("tree_1x60_32k", 1, 60, 32001, 32768),
        # a small server, conversations of different lengths
        _tree("tree_8x32", 8, 32, 4001, 4352, ragged=333, padded=9),
        # a large one: a short tree each, two sequences without any
        _tree("tree_32x13", 32, 13, 8001, 8192, ragged=31, padded=5, idle=2),
        # one user's tree
        _accept("accept_1x16", 1, 16, VOCAB, "bf16"),
        # a server's trees
        _accept("accept_16x32", 16, 32, VOCAB, "bf16"),
        # one user
        _move("move_1x16", 1, 16, 384),
        # a server, short texts
        _move("move_12x48", 12, 48, 160),
        # the vocabulary's projection of one token
        _linear("linear_1x128256", 1, VOCAB, DIM, "bf16", "bf16"),
        # ... and of a tree's
        _linear("linear_60x128256", 60, VOCAB, DIM, "bf16", "bf16"),
        # odd sizes, rows that are quantised already
        _linear("linear_333x2501_int8", 333, 2501, 6912, "int8", "fp32"),
        # prompts through the widest projection
        _linear("linear_4096x13824", 4096, GATE_UP, DIM, "bf16", "bf16"),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], uniform over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "accept", "move", "linear", "linear"))
    dim = rng.choice((128, 128, 64))
    if kind == "tree":
        kv, group = rng.choice(((5, 4), (8, 4), (1, 8), (4, 1), (6, 2), (2, 5), (8, 8)))
        batch = _spread(rng, 1, 64)
        nodes = _spread(rng, 1, min(200, max(1, 200_000 // (batch * kv * group))))
        start = _spread(rng, 1, max(1, min(65536, 1_280_000 // (batch * kv), 60_000_000 // (batch * kv * group * nodes))))
        case = _tree("", batch, nodes, start, start + nodes + rng.randrange(100), heads=kv * group, kv=kv, dim=dim, ragged=rng.choice((0, start // batch)),
                     padded=rng.choice((0, 0, nodes // 3)), idle=rng.choice((0, 0, 0, batch // 8)))
    elif kind == "accept":
        vocab = rng.choice((VOCAB, 32000, 50021, _spread(rng, 1000, 150000)))
        nodes = _spread(rng, 1, 128)
        case = _accept("", _spread(rng, 1, max(1, min(64, 65_000_000 // (vocab * nodes)))), nodes, vocab, rng.choice(("bf16", "bf16", "fp32")))
    elif kind == "move":
        batch, nodes, kv, layers = _spread(rng, 1, 16), _spread(rng, 1, 96), rng.choice((1, 2, 5, 8)), rng.choice((1, 2, 12, LAYERS))
        case = _move("", batch, nodes, nodes + _spread(rng, 1, max(2, 10_000 // (batch * kv))), kv, dim, layers)
    else:
        n, k = rng.choice((DIM, 3840, GATE_UP, VOCAB, 50021, _spread(rng, 100, 60000))), rng.choice((DIM, 6912, 640, 16 * _spread(rng, 1, 512)))
        rows = _spread(rng, 1, max(1, min(8192, 140_000_000_000 // (n * k), 60_000_000 // n)))
        case = _linear("", rows, n, k, *rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("int8", "bf16"), ("int8", "fp32"))))
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------------------------


def _parents(batch, nodes, gen, counts=None):
    """int64 [B, T]: trees as drafted: a node's parent is one of the eight nodes before it, mostly a near one; past a sequence's count -2."""
    back = 1 + (torch.rand((batch, nodes), generator=gen, device="cuda") ** 2 * 8).long()
    at = torch.arange(nodes, device="cuda")
    parents = torch.where(at == 0, -1, (at - back).clamp(min=0))
    if counts is not None:
        parents = torch.where(at < counts[:, None], parents, -2)
    return parents


def _rows(shape, gen, dtype=torch.bfloat16):
    """Activations with a few channels louder than the rest."""
    x = torch.randn(shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-1:], generator=gen, device="cuda") < 0.03
    return torch.where(loud, 6 * x, x).to(dtype)


def _starts(case):
    return [max(0, case["start"] - case["ragged"] * b) for b in range(case["batch"])]


def _counts(case):
    """Nodes of each sequence."""
    batch = case["batch"]
    return [0 if b >= batch - case["idle"] else case["nodes"] - (case["padded"] if b >= batch - (batch + 2) // 3 else 0) for b in range(batch)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "tree":
        batch, nodes, heads, kv, dim, slots = (case[n] for n in ("batch", "nodes", "heads", "kv", "dim", "slots"))
        mask, _ = _plain_masks(_parents(batch, nodes, gen, torch.tensor(_counts(case)).cuda()))
        return dict(case, q=_rows((batch, heads, nodes, dim), gen), k=_rows((batch, kv, slots, dim), gen), v=_rows((batch, kv, slots, dim), gen),
                    start=torch.tensor(_starts(case)).cuda(), mask=mask)
    if kind == "accept":
        batch, nodes, vocab = case["batch"], case["nodes"], case["vocab"]
        logits = torch.empty((batch, nodes, vocab), dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float32, device="cuda")
        for b in range(batch):                               # peaked, as a model's logits are
            wide = torch.randn((nodes, vocab), generator=gen, device="cuda") * 2
            above = torch.randint(0, vocab, (nodes, 12), generator=gen, device="cuda")
            logits[b] = wide.scatter_add_(1, above, 6 + 4 * torch.rand(above.shape, generator=gen, device="cuda"))
        parents = _parents(batch, nodes, gen)
        # most drafts are what the model says behind their parent
        says = torch.argmax(logits, -1).gather(1, parents.clamp(min=0))
        hit = torch.rand((batch, nodes), generator=gen, device="cuda") < 0.8
        tokens = torch.where(hit, says, torch.randint(0, vocab, (batch, nodes), generator=gen, device="cuda"))
        return dict(case, logits=logits, tokens=tokens, parents=parents)
    if kind == "move":
        batch, nodes, slots = case["batch"], case["nodes"], case["slots"]
        caches = [torch.randn((batch, case["kv"], slots, case["dim"]), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2 * case["layers"])]
        start = torch.randint(0, slots - nodes + 1, (batch,), generator=gen, device="cuda")
        # a branch: the root, then nodes further and further on
        steps = 1 + (torch.rand((batch, nodes), generator=gen, device="cuda") * 4).long()
        path = torch.cumsum(steps, 1) - steps[:, :1]
        count = torch.minimum((path < nodes).sum(1), 1 + (torch.rand(batch, generator=gen, device="cuda") * 12).long())
        return dict(case, caches=caches, start=start, path=torch.where(torch.arange(nodes, device="cuda") < count[:, None], path, -1), count=count)
    w = torch.randint(-127, 128, (case["n"], case["k"]), generator=gen, device="cuda", dtype=torch.int8)
    w_scale = (0.5 + torch.rand(case["n"], generator=gen, device="cuda")) / (127 * math.sqrt(case["k"]))
    state = dict(case, w=w, w_scale=w_scale)
    if case["given"] == "int8":
        state["x"] = torch.randint(-127, 128, (case["rows"], case["k"]), generator=gen, device="cuda", dtype=torch.int8)
        state["x_scale"] = 0.01 + torch.rand(case["rows"], generator=gen, device="cuda") / 50
    else:
        state["x"] = _rows((case["rows"], case["k"]), gen)
    if own:
        import ternainfer_amd as T
        state["weight"] = T.int8_rows(w, w_scale)            # the weights as a program keeps them
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------------------------


def _plain_masks(parents):
    """(mask int64 [B, T, W], depth int64 [B, T]) of the parents."""
    batch, nodes = parents.shape
    words = (nodes + 63) // 64
    bits = torch.zeros((batch, nodes, 64 * words), dtype=torch.bool, device=parents.device)
    for i in range(nodes):
        p = parents[:, i]
        above = bits[torch.arange(batch, device=p.device), p.clamp(0, nodes - 1)]
        inside = (p >= 0) & (p < i) & above.any(-1)
        bits[:, i] = above & inside[:, None]
        bits[:, i, i] = inside | (p == -1)
    place = torch.ones((), dtype=torch.int64, device=parents.device) << torch.arange(64, device=parents.device)
    return (bits.view(batch, nodes, words, 64) * place).sum(-1), bits.sum(-1) - 1


def _plain_tree(s):
    """bf16 [B * T, H * D]."""
    q, k, v, start, mask = s["q"], s["k"], s["v"], s["start"], s["mask"]
    batch, heads, nodes, dim = q.shape
    kv, slots = k.shape[1:3]
    at = torch.arange(slots, device=q.device)
    node = at[None] - start[:, None]                                                                # [B, S]: of a slot
    inside = (node >= 0) & (node < nodes)
    held = node.clamp(0, nodes - 1)
    word = mask.gather(2, (held >> 6)[:, None].expand(batch, nodes, slots))                         # [B, T, S]
    bit = (word >> (held & 63)[:, None]) & 1
    seen = torch.where(inside[:, None], bit == 1, (node < 0)[:, None] & (mask != 0).any(-1, keepdim=True))
    scores = torch.matmul(q.float().reshape(batch, kv, heads // kv * nodes, dim), k.float().transpose(2, 3).contiguous()) * dim ** -0.5
    scores = scores.view(batch, kv, heads // kv, nodes, slots).masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(batch, kv, heads // kv * nodes, slots), v.float()).view(*weight.shape[:-1], dim)
    out = torch.where(total > 0, out / total, 0.0)
    return out.reshape(batch, heads, nodes, dim).transpose(1, 2).reshape(batch * nodes, heads * dim).to(torch.bfloat16)


def _plain_accept(s):
    logits, tokens, parents = s["logits"], s["tokens"], s["parents"]
    batch, nodes, vocab = logits.shape
    top = logits.amax(-1, keepdim=True)
    best = torch.where(logits == top, torch.arange(vocab, device=logits.device), vocab).amin(-1)    # the lowest index of the largest
    at = torch.arange(nodes, device=logits.device)
    node = torch.where(parents[:, 0] == -1, 0, -1)
    path = torch.full((batch, nodes), -1, dtype=torch.int64, device=logits.device)
    count = torch.zeros(batch, dtype=torch.int64, device=logits.device)
    behind = torch.full((batch,), -1, dtype=torch.int64, device=logits.device)
    for i in range(nodes):
        on = node >= 0
        path[:, i] = node
        count += on
        says = best.gather(1, node.clamp(min=0)[:, None])
        behind = torch.where(on, says[:, 0], behind)
        child = (parents == node[:, None]) & (tokens == says) & (at > node[:, None]) & on[:, None]
        found = torch.where(child, at, nodes).amin(-1)
        node = torch.where(found < nodes, found, -1)
    return [path, count, behind, *_plain_masks(parents)]


def _plain_move(s):
    start, path, count = s["start"], s["path"], s["count"]
    batch, nodes = path.shape
    at = torch.arange(nodes, device=path.device)
    on = at < count[:, None]
    b = torch.arange(batch, device=path.device)[:, None].expand_as(path)[on]
    source, target = (start[:, None] + path)[on], (start[:, None] + at)[on]
    for cache in s["caches"]:
        cache[b, :, target] = cache[b, :, source]            # (the right side is a copy of its own)
    return s["caches"]


def _plain_linear(s):
    x = s["x"]
    if s["given"] == "int8":
        q, scale = x.float(), s["x_scale"]
    else:
        x = x.float()
        top = x.abs().amax(-1)
        scale = top / torch.full_like(top, 127.0)
        q = torch.round(x * torch.where(top > 0, 127.0 / top, 0.0)[:, None])
    out = torch.matmul(q, s["w"].float().T) * scale[:, None] * s["w_scale"]
    return out.to(torch.bfloat16 if s["out"] == "bf16" else torch.float32)


def run(s):
    kind = s["kind"]
    if not own:
        return {"tree": _plain_tree, "accept": _plain_accept, "move": _plain_move, "linear": _plain_linear}[kind](s)
    import ternainfer_amd as T
    if kind == "tree":
        return T.tree_attention(s["q"], s["k"], s["v"], s["start"], s["mask"])
    if kind == "accept":
        return [*T.tree_accept(s["logits"], s["tokens"], s["parents"]), *T.draft_tree(s["parents"])]
    if kind == "move":
        T.cache_move(s["caches"], s["start"], s["path"], s["count"])
        return s["caches"]
    x = T.int8_rows(s["x"], s["x_scale"]) if s["given"] == "int8" else s["x"]
    return T.int8_linear(x, s["weight"], torch.bfloat16 if s["out"] == "bf16" else torch.float32)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "tree":
        batch, nodes, heads, kv, dim = (case[n] for n in ("batch", "nodes", "heads", "kv", "dim"))
        live = [(start, count) for start, count in zip(_starts(case), _counts(case)) if count]
        slots = sum(start + count for start, count in live)
        pairs = sum((start + min(count, 6)) * count for start, count in live)               # (a node has about five ancestors)
        return {"bytes": 4 * slots * kv * dim + 4 * batch * nodes * heads * dim, "flops": 4 * pairs * heads * dim}
    if kind == "accept":
        n = case["batch"] * case["nodes"]
        return {"bytes": n * (case["vocab"] * (2 if case["dtype"] == "bf16" else 4) + 32 + 8 * ((case["nodes"] + 63) // 64)), "flops": n * case["vocab"]}
    if kind == "move":
        rows = case["batch"] * min(6, (case["nodes"] + 2) // 3)                             # (accepted, in the mean)
        return {"bytes": rows * 2 * case["layers"] * 2 * case["kv"] * case["dim"] * 2, "flops": rows}
    rows, n, k = case["rows"], case["n"], case["k"]
    return {"bytes": n * k + rows * k * (2 if case["given"] == "bf16" else 1) + rows * n * (2 if case["out"] == "bf16" else 4) + 4 * n, "flops": 2 * rows * n * k}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "tree":
        q, k, v = s["q"], s["k"], s["v"]
        batch, heads, nodes, dim = q.shape
        group = heads // k.shape[1]
        out = torch.zeros((batch, nodes, heads, dim), dtype=torch.float64, device=q.device)
        words, starts = s["mask"].tolist(), s["start"].tolist()
        for b in range(batch):                               # the nodes that a node sees, by name
            sees = [[j for j in range(nodes) if words[b][i][j // 64] >> (j % 64) & 1] for i in range(nodes)]
            allowed = torch.zeros((nodes, starts[b] + nodes), dtype=torch.bool)
            for i, seen in enumerate(sees):
                if seen:
                    allowed[i, :starts[b]] = True
                    allowed[i, [starts[b] + j for j in seen]] = True
            allowed = allowed.to(q.device)
            for h in range(heads):
                key, value = k[b, h // group, :starts[b] + nodes].double(), v[b, h // group, :starts[b] + nodes].double()
                scores = torch.matmul(q[b, h].double(), key.T.contiguous()) / math.sqrt(dim)
                out[b, :, h] = torch.matmul(torch.softmax(scores.masked_fill(~allowed, float("-inf")), -1).nan_to_num(0.0), value)
        return out.reshape(batch * nodes, heads * dim)
    if kind == "accept":
        parents, tokens = s["parents"].tolist(), s["tokens"].tolist()
        batch, nodes, words = case["batch"], case["nodes"], (case["nodes"] + 63) // 64
        paths, counts, behind, masks, depths = [], [], [], [], []
        for b in range(batch):
            best = s["logits"][b].float().cpu().numpy().argmax(-1).tolist()                  # (the first of equals)
            path = [0] if parents[b][0] == -1 else []
            while path:
                child = [i for i in range(path[-1] + 1, nodes) if parents[b][i] == path[-1] and tokens[b][i] == best[path[-1]]]
                if not child:
                    break
                path.append(child[0])
            lines = []                                       # of every node, itself and its ancestors (none: no node)
            for i, p in enumerate(parents[b]):
                lines.append([i] if p == -1 else lines[p] + [i] if 0 <= p < i and lines[p] else [])
            bits = [sum(1 << j for j in line) for line in lines]
            signed = lambda word: word - (1 << 64) if word >> 63 else word
            paths.append(path + [-1] * (nodes - len(path)))
            counts.append(len(path))
            behind.append(best[path[-1]] if path else -1)
            masks.append([[signed(m >> (64 * w) & (1 << 64) - 1) for w in range(words)] for m in bits])
            depths.append([len(line) - 1 for line in lines])
        return [torch.tensor(x, device="cuda") for x in (paths, counts, behind, masks, depths)]
    if kind == "move":
        moved = [c.double() for c in s["caches"]]
        paths, starts, counts = s["path"].tolist(), s["start"].tolist(), s["count"].tolist()
        for b in range(case["batch"]):
            for i in range(counts[b]):                       # in order, a row's source is never an earlier row's target
                if paths[b][i] != i:
                    for c in moved:
                        c[b, :, starts[b] + i] = c[b, :, starts[b] + paths[b][i]]
        return moved
    if case["given"] == "int8":
        q, scale = s["x"].double(), s["x_scale"].double()
    else:
        x = s["x"].double()
        scale = x.abs().amax(-1).clamp(min=1e-300) / 127
        q = torch.round(x / scale[:, None])
    return torch.einsum("mk,nk->mn", q, s["w"].double()) * scale[:, None] * s["w_scale"].double()
