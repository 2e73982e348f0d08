"""The operators of ternainfer_amd/drafting.py against plain implementations in 64 bits, and the model's steps over trees."""
import ctypes

import pytest
import torch

import ternainfer_amd as T
import ternainfer_amd.model as model_module
from ternainfer_amd import _lib
from ternainfer_amd.model import ModelArgs, Transformer, greedy_decode, ngram_drafts, speculative_decode
from tests import _drafting as P
from tests._long_context import same_or_near

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=_gen(seed), device="cuda").to(dtype)


def _say(*what):
    print("[case]", *what, flush=True)


# ---- trees ------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("batch,nodes", [(1, 1), (3, 2), (5, 63), (2, 64), (3, 65), (2, 128), (1, 200), (2, 257), (4, 512)])
def test_masks_and_depths(batch, nodes):
    _say("masks", batch, nodes)
    for parents in (P.random_parents(batch, nodes, 1), P.random_parents(batch, nodes, 2, padding=0.2), (torch.arange(nodes) - 1).expand(batch, nodes),
                    torch.randint(-3, nodes + 3, (batch, nodes), generator=torch.Generator().manual_seed(3)), torch.full((batch, nodes), -1)):
        mask, depth = T.draft_tree(parents.cuda())
        want_mask, want_depth = P.tree(parents)
        assert torch.equal(mask.cpu(), want_mask) and torch.equal(depth.cpu(), want_depth)
    odd = torch.stack([parents, parents + 1], -1).cuda()[..., 0]                         # strided
    assert torch.equal(T.draft_tree(odd).mask.cpu(), P.tree(parents)[0])


def test_no_trees():
    empty = torch.zeros((0, 5), dtype=torch.int64, device="cuda")
    assert T.draft_tree(empty).mask.shape == (0, 5, 1) and T.draft_tree(empty.view(5, 0)).depth.shape == (5, 0)
    for bad in (empty.int(), empty[0:0, 0], torch.zeros((1, 513), dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError, match="draft_tree"):
            T.draft_tree(bad)


# ---- attention ---------------------------------------------------------------------------------------------------------------------


def _attend(q, k, v, start, mask, scale=None):
    got = T.tree_attention(q, k, v, start, mask, scale)
    b, h, t, d = q.shape
    assert got.dtype == torch.bfloat16 and got.shape == (b * t, h * d) and got.is_contiguous()
    full = mask if mask.dim() == 3 else mask[None].expand(b, *mask.shape)
    want, tol = P.attention(q, k, v, start, full, d ** -0.5 if scale is None else scale)
    assert same_or_near(got.view(b, t, h, d), want, tol) <= 0
    return got


def _case(b, t, h, kv, d, slots, seed, padding=0.0):
    q, k, v = (_randn((b, n, s, d), seed + i) for i, (n, s) in enumerate(((h, t), (kv, slots), (kv, slots))))
    return q, k, v, T.draft_tree(P.random_parents(b, t, seed, padding).cuda()).mask


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,h,kv,slots,starts", [
    (1, 1, 1, 1, 1, (0,)), (2, 1, 20, 5, 40, (31, 0)), (3, 8, 20, 5, 100, (32, 33, 92)), (2, 13, 8, 4, 300, (256, 287)), (1, 16, 20, 5, 200, (161,)), (2, 17, 4, 1, 96, (64, 63)),
    (2, 33, 12, 6, 700, (600, 5)), (1, 60, 20, 5, 1200, (1100,)), (2, 64, 8, 1, 128, (64, 0)), (1, 65, 4, 4, 400, (303,)), (1, 130, 10, 2, 500, (300,)), (1, 512, 4, 2, 700, (101,)),
    (1, 3, 64, 1, 90, (77,)), (1, 100, 17, 1, 333, (222,)), (64, 20, 20, 5, 200, tuple(range(0, 192, 3))), (2, 70, 800, 200, 400, (300, 64))])
def test_attention(d, b, t, h, kv, slots, starts):
    _say("tree attention", d, b, t, h, kv, slots, starts)
    q, k, v, mask = _case(b, t, h, kv, d, slots, 10, padding=0.1)
    start = torch.tensor(starts, device="cuda")
    got = _attend(q, k, v, start, mask)
    none = (mask == 0).all(-1).view(b * t)
    assert not got[none].any()
    _attend(q, k, v, start, mask[0])                                                     # one tree for all


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,h,kv,slots,starts", [(1, 4, 20, 5, 9000, (8991,)), (2, 16, 20, 5, 6000, (5900, 100)), (1, 40, 8, 2, 20000, (19000,)), (3, 12, 4, 2, 9000, (0, 8000, -1)),
                                                   (70, 2, 2, 1, 1500, tuple(1490 - 21 * i for i in range(70))), (5, 1, 1, 1, 30000, (29999, 3, 12000, 29998, 1))])
def test_attention_in_parts(d, b, t, h, kv, slots, starts):
    """Long caches, dealt out by the sequences' lengths; as one part, without a workspace, the same within the tolerance."""
    _say("tree attention in parts", d, b, t, h, kv, slots)
    lib = _lib.load()
    assert lib.ternaspmm_tree_attention_workspace_bytes(b, t, h, kv, d, slots) > 0
    q, k, v, mask = _case(b, t, h, kv, d, slots, 20)
    start = torch.tensor(starts, device="cuda")
    got = _attend(q, k, v, start, mask)
    assert torch.equal(got, T.tree_attention(q, k, v, start, mask))
    out = torch.empty_like(got)
    p = lambda x: ctypes.c_void_p(x.data_ptr())
    strides = lambda x: (ctypes.c_longlong * 3)(*x.stride()[:3])
    assert lib.ternaspmm_tree_attention(p(q), strides(q), p(k), strides(k), p(v), strides(v), p(start), p(mask), 1, p(out), None, b, t, h, kv, d, slots, d ** -0.5,
                                        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    want, tol = P.attention(q, k, v, start, mask, d ** -0.5)
    assert same_or_near(out.view(b, t, h, d), want, tol) <= 0


@pytest.mark.parametrize("t,h,kv,slots", [(6, 20, 5, 200), (20, 8, 2, 200), (40, 20, 5, 300), (6, 20, 5, 8000), (40, 1200, 300, 300)])
def test_what_a_node_does_not_see_does_not_reach_it(t, h, kv, slots):
    """Bit for bit: other nodes' queries; keys and values, finite ones, infinities and NaN, in the slots of nodes that are no ancestors, and behind the tree."""
    _say("unseen", t, h, kv, slots)
    d, start = 128, slots - t - 50
    q, k, v, mask = _case(1, t, h, kv, d, slots, 30)
    at = torch.tensor([start], device="cuda")
    want = T.tree_attention(q, k, v, at, mask).view(t, h, d)
    bits = (mask[0, :, 0, None] >> torch.arange(t, device="cuda") & 1).bool()             # [node, sees]
    for fill in (3.0, float("inf"), float("-inf"), float("nan")):
        for node in (t - 1, t // 2):
            unseen = (~bits[node]).nonzero()[:, 0] + start
            q2, k2, v2 = q.clone(), k.clone(), v.clone()
            for c in (k2, v2):
                c[:, :, unseen] = fill
                c[:, :, start + t:] = fill
            others = torch.arange(t, device="cuda") != node
            q2[:, :, others] = -2 * q[:, :, others]
            got = T.tree_attention(q2, k2, v2, at, mask).view(t, h, d)
            assert torch.equal(got[node], want[node]), (fill, node)


@pytest.mark.parametrize("t,h,kv,start,slots", [(5, 4, 2, 70, 100), (5, 4, 2, 0, 100), (70, 8, 1, 100, 200), (9, 20, 5, 7000, 7100), (40, 1200, 300, 190, 260), (5, 4, 2, 1000, 1010), (9, 20, 5, 1000, 1010),
                                                   (40, 20, 5, 2000, 2050), (5, 20, 5, 9000, 9010)])
def test_values_that_are_not_finite_where_they_are_seen(t, h, kv, start, slots):
    """Infinities and NaN among the seen slots -- of the text and of the tree -- come out where the definition has them."""
    _say("not finite", t, h, kv, start, slots)
    d = 128
    q, k, v, mask = _case(1, t, h, kv, d, slots, 40)
    at = torch.tensor([start], device="cuda")
    for places in ([start + t // 2], [start, start + t - 1], [start // 2], [max(start - 1, 0), start + 1]):
        broken = v.clone()
        for i, s in enumerate(places):
            broken[0, :, s, 3 + i] = float("inf")
            broken[0, 0, s, 40] = float("nan") if i else float("-inf")
        got = T.tree_attention(q, k, broken, at, mask).view(1, t, h, d)
        want, tol = P.attention(q, k, broken, at, mask, d ** -0.5)
        assert same_or_near(got, want, tol.nan_to_num(0.0, 0.0, 0.0)) <= 0
    broken = k.clone()
    broken[0, 0, start, 5] = float("nan")                                                # a score of NaN: the rows that see it
    got = T.tree_attention(q, broken, v, at, mask).view(t, h, d)
    sees = (mask[0, :, 0] & 1).bool()
    group = torch.arange(h, device="cuda") < h // kv
    assert got[sees][:, group].isnan().all() and not got[~sees].isnan().any() and not got[:, ~group].isnan().any()


@pytest.mark.parametrize("t,start,slots", [(4, 30, 32), (4, 32, 32), (4, 33, 32), (70, 40, 100), (4, -1, 32), (4, -(1 << 40), 32), (4, 1 << 40, 32)])
def test_trees_at_the_end_of_the_cache(t, start, slots):
    """A slot behind the cache: NaN for the nodes that see it, and no others; a start behind it: all; a negative one: zeros."""
    _say("end of the cache", t, start, slots)
    q, k, v, mask = _case(2, t, 4, 2, 64, slots, 50)
    at = torch.tensor([start, slots - t if t <= slots else 0], device="cuda")
    got = _attend(q, k, v, at, mask)
    if start < 0:
        assert not got[:t].any()


def test_masks_that_leave_nothing_and_bits_behind_the_tree():
    q, k, v, mask = _case(2, 5, 4, 2, 128, 64, 60)
    start = torch.tensor([0, 20], device="cuda")
    assert not T.tree_attention(q, k, v, start, torch.zeros_like(mask)).any()
    want = T.tree_attention(q, k, v, start, mask)
    assert torch.equal(T.tree_attention(q, k, v, start, mask | (-1 << 5)), want)          # bits of nodes that are none do not count
    half = mask.clone()
    half[0] = 0
    got = T.tree_attention(q, k, v, start, half)
    assert not got[:5].any() and torch.equal(got[5:], want[5:])


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-3, 4.0, 30.0])
def test_scales(scale):
    q, k, v, mask = _case(1, 12, 8, 2, 64, 150, 70)
    _attend(q, k, v, torch.tensor([100], device="cuda"), mask, scale)
    for bad in (float("inf"), float("nan")):
        with pytest.raises(ValueError, match="tree_attention"):
            T.tree_attention(q, k, v, torch.tensor([100], device="cuda"), mask, bad)


def test_scores_that_grow_and_peak():
    """Maxima that rise from tile to tile, one slot that outweighs all, and scores far apart."""
    q, k, v, mask = _case(1, 20, 8, 2, 128, 1000, 80)
    start = torch.tensor([960], device="cuda")
    ramp = torch.linspace(0.01, 6, 1000, device="cuda")[None, None, :, None]
    _attend(q, (k * ramp).to(torch.bfloat16), v, start, mask)
    _attend(q, (k * ramp.flip(2)).to(torch.bfloat16), v, start, mask)
    peak = k.clone()
    peak[:, :, 500] = 8 * q[:, ::4, 0]
    _attend((q * 4).to(torch.bfloat16), peak, v, start, mask)


def test_strides_and_views():
    b, t, h, kv, d, slots = 2, 11, 8, 2, 64, 120
    start = torch.tensor([100, 33], device="cuda")
    mask = T.draft_tree(P.random_parents(b, t, 90).cuda()).mask
    both = _randn((b, slots, 2, kv, d), 91)                                               # slots outermost, keys and values beside each other
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    rows = _randn((b * t, (h + 2 * kv) * d), 92)
    q = rows.view(b, t, h + 2 * kv, d)[:, :, :h].transpose(1, 2)                          # the rows of a fused projection
    got = _attend(q, k, v, start, mask)
    assert torch.equal(got, T.tree_attention(q.contiguous(), k.contiguous(), v.contiguous(), start, mask))
    odd = _randn((b, h, t, d + 1), 93)[..., 1:]                                           # queries that have to be copied
    _attend(odd, k, v, start, mask)
    one = _randn((b, 1, slots, d), 94).expand(b, kv, slots, d)                            # broadcast heads
    _attend(q, one, one, start, mask)
    apart = torch.stack([start, start], -1)[:, 0]
    assert torch.equal(T.tree_attention(q, k, v, apart, torch.stack([mask, mask], -1)[..., 0]), got)


def test_attention_refusals():
    q, k, v, mask = _case(2, 5, 4, 2, 64, 30, 100)
    start = torch.tensor([3, 4], device="cuda")
    assert T.tree_attention(q[:, :, :0], k, v, start, mask[:, :0, :0]).shape == (0, 256)
    assert T.tree_attention(q[:0], k[:0], v[:0], start[:0], mask[:0]).shape == (0, 256)
    wide = _randn((2, 2, 30, 65), 101)[..., :64]
    for args in ((q.float(), k, v, start, mask), (q, k.float(), v, start, mask), (q, k, v[:, :, :29], start, mask), (q[:1], k, v, start, mask), (q[:, :3], k, v, start, mask), (q[..., :32], k, v, start, mask),
                 (q, k, v, start[:1], mask), (q, k, v, start.int(), mask), (q, k, v, start, mask.int()), (q, k, v, start, mask[:, :4]), (q, k, v, start, mask[:1]), (q, k, v, start, mask.expand(2, 5, 2)),
                 (q, wide, v, start, mask), (q, k, wide, start, mask), (q, k.transpose(2, 3).contiguous().transpose(2, 3), v, start, mask), (q, k[:, :, :0], v[:, :, :0], start, mask),
                 (q.cpu(), k, v, start, mask), (q, k, v, start.cpu(), mask), (q, k, v, start, mask.cpu())):
        with pytest.raises(ValueError, match="tree_attention"):
            T.tree_attention(*args)
    for scale in (float("inf"), float("nan"), 3e38):                                     # (the last times log2(e) is none)
        with pytest.raises(ValueError, match="tree_attention"):
            T.tree_attention(q, k, v, start, mask, scale)
    with pytest.raises(ValueError, match="tree_attention"):
        T.tree_attention(_randn((1, 1, 513, 64), 102), k[:1, :1], v[:1, :1], start[:1], torch.ones((513, 9), dtype=torch.int64, device="cuda"))


def test_a_cache_of_more_than_four_gigabytes():
    """Offsets behind 2^32 bytes in one head."""
    slots, d = 17 << 20, 128
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("9 GB of keys and values")
    _say("slots", slots)
    k, v = (torch.zeros((1, 1, slots, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, mask = _randn((1, 2, 3, d), 110), T.draft_tree(torch.tensor([[-1, 0, 0]], device="cuda")).mask
    start = slots - 3
    v[0, 0, start - 5] = 1.0
    k[0, 0, start - 5] = 4 * q[0, 0, 0]                                                   # found by the first node's first head
    v[0, 0, start:] = _randn((3, d), 111)
    k[0, 0, start:] = _randn((3, d), 112)
    got = T.tree_attention(q, k, v, torch.tensor([start], device="cuda"), mask).view(3, 2, d)
    # All other scores are 0: (start - 1) equal terms of value 0 beside the named ones.
    for node, seen in enumerate(([start], [start, start + 1], [start, start + 2])):
        at = torch.tensor([start - 5, *seen], device="cuda")
        key, value = k[0, 0].index_select(0, at).double(), v[0, 0].index_select(0, at).double()
        score = q[0, :, node].double() @ key.T * d ** -0.5
        top = score.amax(-1, keepdim=True).clamp(min=0)
        p = (score - top).exp()
        total = p.sum(-1, keepdim=True) + (start - 1) * (-top).exp()
        want = p @ value / total
        ds = (d + 4) * P.HALF_FP32 * d ** -0.5 * (q[0, :, node].double().abs() @ key.abs().T).amax(-1, keepdim=True)
        # terms that count: three values, and a sum of 2^24 equal terms in parts of 2^18 and fewer
        tol = P.HALF_BF16 * want.abs() + (2 * ds + 2.0 ** -14 + 2 * 2.0 ** 19 * P.HALF_FP32) * (p @ value.abs() / total)
        assert ((got[node].double() - want).abs() <= tol).all(), node


@pytest.mark.parametrize("t,h", [(5, 2), (11, 4), (40, 4)])
def test_slots_far_apart(t, h):
    """Slots 2^23 elements apart: 32 of them are a distance of 2^29 bytes."""
    slots, d, start = 40 + t, 128, 39
    _say("far apart", t, h)
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("3 GB of keys and values")
    k, v = (torch.zeros((1, 1, slots * 65536, d), dtype=torch.bfloat16, device="cuda")[:, :, ::65536] for _ in range(2))
    k.copy_(_randn(k.shape, 114))
    v.copy_(_randn(v.shape, 115))
    assert k.stride(2) == 1 << 23
    _attend(_randn((1, h, t, d), 116), k, v, torch.tensor([start], device="cuda"), T.draft_tree(P.random_parents(1, t, 117).cuda()).mask)


def test_many_sequences():
    """As many as a call takes, of the smallest trees; more are refused."""
    b = 65535
    _say("sequences", b)
    parents = torch.tensor([[-1, 0], [-1, -1], [-2, 0]], device="cuda").repeat(21845, 1)
    tree = T.draft_tree(parents)
    mask, depth = P.tree(parents[:3].cpu())
    assert torch.equal(tree.mask.cpu(), mask.repeat(21845, 1, 1)) and torch.equal(tree.depth.cpu(), depth.repeat(21845, 1))
    q, k, v = _randn((b, 1, 2, 64), 118), _randn((b, 1, 5, 64), 119), _randn((b, 1, 5, 64), 120)
    start = torch.arange(b, device="cuda") % 5 - 1                                        # none; 0 .. 3, of which the last has no slot for the second node
    got = T.tree_attention(q, k, v, start, tree.mask).view(b, 2, 1, 64)
    for at in (slice(0, 60), slice(32700, 32760), slice(b - 60, b)):
        want, tol = P.attention(q[at], k[at], v[at], start[at], tree.mask[at], 64 ** -0.5)
        assert same_or_near(got[at], want, tol) <= 0
    logits, tokens = _randn((b, 2, 3), 121), torch.ones((b, 2), dtype=torch.int64, device="cuda")
    accepted = T.tree_accept(logits, tokens, parents)
    for at in (slice(0, 60), slice(b - 60, b)):
        assert [x[at].tolist() for x in accepted] == P.accept(logits[at], tokens[at], parents[at])
    cache = v.clone()
    T.cache_move([cache], torch.ones(b, dtype=torch.int64, device="cuda"), torch.tensor([[0, 3]], device="cuda").expand(b, 2), torch.full((b,), 2, device="cuda"))
    v[:, :, 2] = v[:, :, 4]
    assert torch.equal(cache, v)
    more = torch.full((b + 1, 1), -1, device="cuda")
    for call in (lambda: T.draft_tree(more), lambda: T.tree_accept(torch.zeros((b + 1, 1, 1), device="cuda"), more, more), lambda: T.cache_move([], more[:, 0], more, more[:, 0])):
        with pytest.raises(ValueError, match="65535"):
            call()


# ---- acceptance --------------------------------------------------------------------------------------------------------------------


def _accept(logits, tokens, parents):
    got = T.tree_accept(logits, tokens, parents)
    want = P.accept(logits, tokens, parents)
    assert [x.tolist() for x in got] == want and all(x.dtype == torch.int64 for x in got)
    return got


def _drafts(logits, parents, seed, hit=0.8):
    """Tokens that mostly are what the parent's logits say."""
    says = torch.tensor([[max(range(len(r)), key=lambda i: (r[i], -i)) for r in rows] for rows in logits.float().cpu().nan_to_num(-1e9).tolist()])
    gen = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, logits.shape[-1], parents.shape, generator=gen)
    take = torch.rand(parents.shape, generator=gen) < hit
    return torch.where(take, says.gather(1, parents.cpu().clamp(0, parents.shape[1] - 1)), tokens).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,t,v", [(1, 1, 1), (2, 5, 7), (3, 16, 1000), (1, 70, 333), (5, 8, 2049), (2, 3, 70001), (1, 300, 64), (40, 20, 129)])
def test_acceptance(dtype, b, t, v):
    _say("accept", dtype, b, t, v)
    logits = (_randn((b, t, v), 120, torch.float32) * 3).to(dtype)
    for seed, padding, hit in ((1, 0.0, 0.9), (2, 0.2, 0.8), (3, 0.0, 0.0), (4, 0.0, 1.0)):
        parents = P.random_parents(b, t, seed, padding).cuda()
        _accept(logits, _drafts(logits, parents, seed, hit), parents)
    if b > 1:
        parents[1, 0] = -2                                                                # a sequence without a step
        assert _accept(logits, _drafts(logits, parents, 5), parents).count[1] == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_acceptance_of_rows_at_any_address(dtype):
    wide = _randn((3, 7, 1003), 130, torch.float32).to(dtype)
    parents = P.random_parents(3, 7, 131).cuda()
    for logits in (wide, wide[..., 1:], wide[..., 3:998], wide[:, :, ::2], wide.transpose(0, 1).contiguous().transpose(0, 1), wide[1:, :, :5], wide[:, :1].expand(3, 7, 1003), wide[..., :1]):
        mine = parents[:logits.shape[0]]
        _accept(logits, _drafts(logits, mine, 132), mine)


def test_acceptance_where_logits_tie_and_where_they_are_not_finite():
    v = 5000
    logits = torch.zeros((1, 7, v), device="cuda")
    logits[0, 1, [77, 4000, 4999]] = 2.0                                                  # equal: the lowest
    logits[0, 2] = float("-inf")                                                          # none: 0
    logits[0, 3] = float("nan")
    logits[0, 4, 10:] = float("nan")
    logits[0, 4, 3] = 1.0
    logits[0, 5, 4999] = float("inf")
    logits[0, 6] = -float("inf")
    logits[0, 6, 4321] = -1e30
    parents = torch.tensor([[-1, 0, 1, 2, 3, 4, 5]], device="cuda")
    tokens = torch.tensor([[9, 0, 77, 0, 0, 3, 4999]], device="cuda")
    for x in (logits, logits.to(torch.bfloat16)):
        path, count, behind = _accept(x, tokens, parents)
        assert count.tolist() == [7] and behind.tolist() == [4321]
    twice = torch.tensor([[9, 0, 0, 77, 77, 0, 0]], device="cuda")                        # two children with the token: the first, whatever continues the other
    path, count, behind = _accept(logits, twice, torch.tensor([[-1, 0, 0, 2, 1, 4, 3]], device="cuda"))
    assert path.tolist()[0][:3] == [0, 1, 4] and count.item() >= 3


def test_acceptance_of_a_long_chain():
    logits = torch.zeros((2, 512, 40), device="cuda")
    says = torch.randint(0, 40, (2, 512), generator=torch.Generator().manual_seed(140)).cuda()
    logits.scatter_(2, says[..., None], 5.0)
    parents = (torch.arange(512, device="cuda") - 1).expand(2, 512).contiguous()
    tokens = torch.cat([says[:, :1], says[:, :-1]], 1)
    tokens[1, 300] += 1
    got = _accept(logits, tokens, parents)
    assert got.count.tolist() == [512, 300]


def test_acceptance_refusals():
    logits, longs = _randn((2, 3, 10), 150), torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    assert T.tree_accept(logits[:0], longs[:0], longs[:0]).path.shape == (0, 3)
    for args in ((logits[0], longs, longs), (logits.half(), longs, longs), (logits, longs[:1], longs), (logits, longs, longs[:, :2]), (logits, longs.int(), longs), (logits, longs, longs.int()),
                 (logits[..., :0], longs, longs), (logits[:, :0], longs[:, :0], longs[:, :0]), (logits, longs.cpu(), longs), (logits.cpu(), longs, longs)):
        with pytest.raises(ValueError, match="tree_accept"):
            T.tree_accept(*args)
    with pytest.raises(ValueError, match="tree_accept"):
        T.tree_accept(torch.zeros((1, 1, (1 << 19) + 1), device="cuda"), longs[:1, :1], longs[:1, :1])


# ---- moving rows -------------------------------------------------------------------------------------------------------------------


def _moved(cache, start, path, count):
    want = cache.clone()
    for b, s in enumerate(start.tolist()):
        for i in range(min(int(count[b]), path.shape[1])):
            p = int(path[b, i])
            if p > i and 0 <= s and s + p < cache.shape[2]:
                want[b, :, s + i] = want[b, :, s + p]
    return want


def _bytes(shape, dtype, seed):
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * torch.tensor([], dtype=dtype).element_size()), generator=_gen(seed), device="cuda", dtype=torch.uint8)
    return raw.view(dtype)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


PATHS = [[[0, 2, 5, 6], [0, 1, 2, 3], [0, 3, -1, -1]], [[3, 9, 10, 17], [0, 7, -1, -1], [1, 2, 3, 4]]]


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.uint8, 64), (torch.uint8, 4), (torch.uint8, 2), (torch.uint8, 5), (torch.float32, 3), (torch.bfloat16, 1),
                                         (torch.bfloat16, 1000)])
@pytest.mark.parametrize("kv", [1, 5])
def test_rows_move(dtype, width, kv):
    _say("move", dtype, width, kv)
    for path in PATHS:
        path = torch.tensor(path, device="cuda")
        for start, count in (([0, 10, 29], [4, 4, 2]), ([5, 5, 5], [0, 1, 9]), ([-1, 40, 1 << 40], [4, 4, 4]), ([36, 38, 39], [4, 4, 4]), ([0, 0, 0], [-3, 2, 1 << 40])):
            start, count = torch.tensor(start, device="cuda"), torch.tensor(count, device="cuda")
            caches = [_bytes((3, kv, 40, width), dtype, 160 + i) for i in range(2)]
            want = [_moved(c, start, path, count) for c in caches]
            T.cache_move(caches, start, path, count)
            assert all(_same(c, w) for c, w in zip(caches, want))


def test_rows_of_many_caches_and_of_views_move():
    """More than one launch takes; caches of different types, strides and lengths in one call; what lies beside them stays."""
    b, start, count = 2, torch.tensor([3, 20], device="cuda"), torch.tensor([5, 3], device="cuda")
    path = torch.tensor([[0, 2, 3, 7, 9], [1, 2, 4, -1, -1]], device="cuda")
    plain = [_bytes((b, 1 + i % 3, 30 + i % 4, 16), torch.bfloat16, 170 + i) for i in range(130)]
    both = _bytes((b, 40, 2, 4, 64), torch.bfloat16, 171)                                 # keys and values beside each other
    cut = _bytes((b, 2, 40, 70), torch.uint8, 172)
    views = [both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), cut[..., 3:68], _bytes((b, 2, 40, 2), torch.uint8, 173)]
    four = T.Kv4Cache(*(_bytes((b, 2, 40, w), torch.uint8, 174 + w) for w in (64, 4, 63, 3)))
    all_caches = plain + views + list(four)
    want = [_moved(c, start, path, count) for c in all_caches]
    beside = cut.clone()
    T.cache_move(all_caches, start, path, count)
    assert all(_same(c, w) for c, w in zip(all_caches, want))
    assert torch.equal(cut[..., :3], beside[..., :3]) and torch.equal(cut[..., 68:], beside[..., 68:])


def test_a_long_path_moves():
    path = torch.cumsum(1 + (torch.rand((1, 200), generator=_gen(180), device="cuda") * 2.5).long(), 1) - 1
    cache = _bytes((1, 2, 700, 128), torch.bfloat16, 181)
    start, count = torch.tensor([7], device="cuda"), torch.tensor([200], device="cuda")
    want = _moved(cache, start, path, count)
    T.cache_move([cache], start, path, count)
    assert _same(cache, want)


def test_move_refusals():
    cache, longs = _randn((2, 1, 10, 8), 190), torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    each = longs[:, 0].contiguous()
    before = cache.clone()
    T.cache_move([], each, longs, each)
    T.cache_move([cache, cache[:, :, :0], cache[:, :0]], each, longs[:, :0], each)
    T.cache_move([cache[:0]], each[:0], longs[:0], each[:0])
    for args in (([cache, cache], each, longs, each), ([cache[0]], each, longs, each), ([cache[:1]], each, longs, each), ([cache], each[:1], longs, each), ([cache], each, longs, each.int()),
                 ([cache], each, longs.int(), each), ([cache.cpu()], each, longs, each), ([cache], each.cpu(), longs, each), ([cache.transpose(2, 3)], each, longs, each),
                 ([cache[:, :, :1].expand(2, 1, 10, 8)], each, longs, each), ([cache], each, torch.zeros((2, 513), dtype=torch.int64, device="cuda"), each)):
        with pytest.raises(ValueError, match="cache_move"):
            T.cache_move(*args)
    assert torch.equal(cache, before)


# ---- a run of them -------------------------------------------------------------------------------------------------------------------


def _step(state):
    """One step of a decoder by drafts, without a model: attention, logits, acceptance, cache."""
    q, k, v, start, tokens, parents, weight = (state[n] for n in ("q", "k", "v", "start", "tokens", "parents", "weight"))
    tree = T.draft_tree(parents)
    o = T.tree_attention(q, k, v, start, tree.mask)
    logits = T.int8_linear(o, weight).view(*tokens.shape, -1)
    took = T.tree_accept(logits, tokens, parents)
    T.cache_move([k, v], start, took.path, took.count)
    return [o, logits, *took, *tree, k, v]


def _state(seed, b=3, t=18, h=20, kv=5, d=128, slots=5000, vocab=300):
    return dict(q=_randn((b, h, t, d), seed), k=_randn((b, kv, slots, d), seed + 1), v=_randn((b, kv, slots, d), seed + 2), start=torch.tensor([4000, 33, -1], device="cuda"),
                tokens=torch.randint(0, 2, (b, t), generator=_gen(seed + 3), device="cuda"), parents=P.random_parents(b, t, seed).cuda(),
                weight=T.quantise_rows(_randn((vocab, h * d), seed + 4) * torch.where(torch.arange(vocab, device="cuda") < 2, 20.0, 1.0)[:, None].to(torch.bfloat16)))


def _copy(state):
    return {n: x.clone() if isinstance(x, torch.Tensor) else x for n, x in state.items()}


def test_steps_eager_and_captured():
    """The operators of a step together, as a graph that is replayed with eager work between, on a stream of its own."""
    eager, held = _state(200), _state(200)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        _step(_copy(held))
        with torch.cuda.graph(graph, stream=side):
            captured = _step(held)
    torch.cuda.current_stream().wait_stream(side)
    accepted = 0
    for i in range(5):
        fresh = _state(210 + 10 * i)
        for state in (eager, held):
            for n in ("q", "tokens", "parents"):
                state[n].copy_(fresh[n])
            state["start"].copy_(torch.tensor([4000 + 7 * i, 33 + i, -1 if i % 2 else 900], device="cuda"))
        want = [x.clone() for x in _step(eager)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(_same(got, w) for got, w in zip(captured, want)), i
        accepted += int((want[3] > 1).sum())
    assert accepted > 0


def test_steps_at_once_and_two_graphs():
    states = [_state(300), _state(320)]
    want = [[x.clone() for x in _step(_copy(s))] for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(6):
        got, copies = [None, None], [_copy(s) for s in states]
        for i, stream in enumerate(streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got[i] = _step(copies[i])
        torch.cuda.synchronize()
        assert all(_same(a, b) for i in range(2) for a, b in zip(got[i], want[i]))
    held = [_copy(s) for s in states]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, stream=streams[i]):
            got[i] = _step(held[i])
    for _ in range(6):
        for i in range(2):
            for n in ("k", "v"):
                held[i][n].copy_(states[i][n])
        torch.cuda.synchronize()
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay()
        eager = _step(_copy(states[0]))
        torch.cuda.synchronize()
        assert all(_same(a, b) for i in range(2) for a, b in zip(got[i], want[i])) and all(_same(a, b) for a, b in zip(eager, want[0]))


# ---- the model -----------------------------------------------------------------------------------------------------------------------

SHAPES = [dict(dim=256, n_heads=4, n_kv_heads=2), dict(dim=512, n_heads=4, n_kv_heads=1, rope_adjacent=False)]


def _model(shape, act="int8", **more):
    return Transformer(ModelArgs(n_layers=2, vocab_size=1000, ffn_dim=384, **SHAPES[shape], **more), seed=31, act=act)


def _tokens(*shape, seed=32):
    return torch.randint(0, 1000, shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("act,shape,bsz,t", [("int8", 0, 1, 6), ("int8", 1, 3, 7), ("int8", 0, 4, 30), ("bf16", 1, 2, 12)])
@torch.inference_mode()
def test_tree_step_is_the_operators_with_the_models_positions(act, shape, bsz, t, monkeypatch):
    """Every block's attention against 64 bits; a node's keys in the first block are those that a prompt pass writes for its token at its depth, bit for bit, in the
    slot of the node; padding writes nothing."""
    _say("tree step", act, SHAPES[shape], bsz, t)
    model = _model(shape, act)
    a, plen, slots = model.args, 17, 17 + t + 5
    prompt, tokens = _tokens(bsz, plen), _tokens(bsz, t, seed=33)
    parents = P.random_parents(bsz, t, 34, padding=0.15)
    tree = T.draft_tree(parents.cuda())
    cache = model.make_cache(bsz, slots)
    model.forward(prompt, cache, torch.arange(plen, device="cuda"))
    start = torch.full((bsz,), plen, device="cuda")
    if bsz > 2:
        start[1], start[2] = 9, -1                                                       # the last tokens of a text drafted again; a sequence without a step
    before = [(k.clone(), v.clone()) for k, v in cache]
    plain, calls = model_module.tree_attention, []

    def checked(q, k, v, first, mask, *rest):
        got = plain(q, k, v, first, mask, *rest)
        want, tol = P.attention(q, k, v, first, mask, a.head_dim ** -0.5)
        assert same_or_near(got.view(bsz, t, a.n_heads, a.head_dim), want, tol) <= 0
        calls.append(first)
        return got

    monkeypatch.setattr(model_module, "tree_attention", checked)
    logits = model.tree_step(tokens, cache, start, tree)
    assert logits.shape == (bsz, t, 1000) and len(calls) == 2
    at = torch.tensor(parents.tolist())
    for b in range(bsz):
        s = int(start[b])
        lines = P.lines(at[b].tolist())
        touched = {s + i for i in range(t) if lines[i]} if s >= 0 else set()
        for j in set(range(slots)) - touched:
            assert all(torch.equal(now[b, :, j], was[b, :, j]) for pair, old in zip(cache, before) for now, was in zip(pair, old)), (b, j)
        if s < 0:
            continue
        for i, line in enumerate(lines):
            if not line:
                continue
            assert torch.isfinite(logits[b, i]).all()
            # Linears of more than 64 rows follow the prefill rule of the weights' scales (groups by 128 columns): a pass of as many rows, all of this line.
            copies = 1 if bsz * t <= 64 else 64 // len(line) + 1
            chain = model.make_cache(copies, slots)
            model.forward(tokens[b:b + 1, line].expand(copies, -1).contiguous(), chain, torch.arange(s, s + len(line), device="cuda"))
            assert all(torch.equal(now[b, :, s + i], one[0, :, s + len(line) - 1]) for now, one in zip(cache[0], chain[0])), (b, i)


@torch.inference_mode()
def test_tree_step_behind_a_long_text(monkeypatch):
    """More slots than the attention of other steps takes: every block's attention against 64 bits."""
    model, t, start = _model(1), 11, 9000
    a, cache, plain, calls = model.args, model.make_cache(1, start + t), model_module.tree_attention, []
    for i, pair in enumerate(cache):
        for j, c in enumerate(pair):
            c[:, :, :start] = _randn(c[:, :, :start].shape, 300 + 2 * i + j)

    def checked(q, k, v, first, mask, *rest):
        got = plain(q, k, v, first, mask, *rest)
        want, tol = P.attention(q, k, v, first, mask, a.head_dim ** -0.5)
        assert same_or_near(got.view(1, t, a.n_heads, a.head_dim), want, tol) <= 0
        calls.append(0)
        return got

    monkeypatch.setattr(model_module, "tree_attention", checked)
    logits = model.tree_step(_tokens(1, t, seed=38), cache, torch.tensor([start], device="cuda"), T.draft_tree(P.random_parents(1, t, 39).cuda()))
    assert torch.isfinite(logits).all() and len(calls) == 2


@torch.inference_mode()
def test_logits_of_a_node_do_not_depend_on_other_branches():
    """Bit for bit, whatever tokens the nodes have that are no ancestors of its."""
    model = _model(0)
    prompt, tokens = _tokens(2, 20), _tokens(2, 13, seed=35)
    parents = P.random_parents(2, 13, 36)
    tree, start = T.draft_tree(parents.cuda()), torch.tensor([20, 11], device="cuda")

    def run(tokens):
        cache = model.make_cache(2, 40)
        model.forward(prompt, cache, torch.arange(20, device="cuda"))
        return model.tree_step(tokens, cache, start, tree)

    want = run(tokens)
    for node in (4, 12):
        other = _tokens(2, 13, seed=37)
        for b in range(2):
            other[b, P.lines(parents[b].tolist())[node]] = tokens[b, P.lines(parents[b].tolist())[node]]
        assert torch.equal(run(other)[:, node], want[:, node])


@pytest.mark.parametrize("head8", [False, True])
@pytest.mark.parametrize("lens", [None, [16, 5, 11]])
@pytest.mark.parametrize("draft", [ngram_drafts, lambda text, length: ngram_drafts(text, length, 3, 7), lambda text, length: ngram_drafts(text, length, 0, 0)])
def test_speculative_decode(draft, lens, head8):
    """Every token is the likeliest of the logits that steps of one token have behind the same text, but for logits nearer to it than the two ways' roundings: a
    bfloat16 rounding of every sum on the way, 2^-8 of it, some ten of them in two blocks, is below a tenth of the logits' spread."""
    _say("speculative decode", lens, head8)
    model, count = _model(0), 40
    if head8:
        model.quantise_head()
    prompt = _tokens(3, 8).repeat(1, 2)                                                   # (something to look up)
    lens_t = None if lens is None else torch.tensor(lens)
    got, steps = speculative_decode(model, prompt, count, draft=draft, prompt_lens=lens_t)
    assert got.shape == (3, count) and 1 <= steps < count + 1 and got.min() >= 0 and got.max() < 1000
    again, _ = speculative_decode(model, prompt, count, draft=draft, prompt_lens=lens_t)
    assert torch.equal(got, again)
    # Linears of more than 64 rows follow the prefill rule of the weights' scales (groups by 128 columns, other ones than a step's in a model as small as this): steps
    # of as many rows here too, of one sequence.
    copies = 1 if 3 * draft(prompt, torch.full((3,), 16, device="cuda"))[0].shape[1] <= 64 else 65
    with torch.inference_mode():
        for b in range(3):
            n = 16 if lens is None else lens[b]
            cache = model.make_cache(1, n + count)
            logits = model.forward(prompt[b:b + 1, :n].contiguous(), cache, torch.arange(n, device="cuda"))
            cache = [tuple(c.repeat(copies, 1, 1, 1) for c in pair) for pair in cache]
            for i in range(count):
                row = logits[0].float()
                assert row.max() - row[got[b, i]] <= 0.1 * row.std(), (b, i)
                logits = model.forward(got[b:b + 1, i:i + 1].repeat(copies, 1), cache, torch.tensor([n + i], device="cuda"))
    assert speculative_decode(model, prompt, 0)[0].shape == (3, 0)
    assert speculative_decode(model, prompt, 1, prompt_lens=lens_t)[0].shape == (3, 1)


def test_drafts_are_accepted():
    """Drafts that are the greedy tokens take a fraction of the steps."""
    model, count = _model(0), 41
    prompt = _tokens(2, 12)
    plain, one = speculative_decode(model, prompt, count, draft=lambda text, length: ngram_drafts(text, length, 0, 0))
    assert one == count - 1
    known = torch.cat([prompt, plain, plain.new_zeros((2, 8))], 1)

    def oracle(text, length):
        at = length[:, None] - 1 + torch.arange(5, device="cuda")
        parents = torch.arange(-1, 4, device="cuda").expand(2, 5)
        return known.gather(1, at.clamp(max=known.shape[1] - 1)), parents.contiguous()

    got, steps = speculative_decode(model, prompt, count, draft=oracle)
    assert (got == plain).float().mean() >= 0.5 and steps <= one // 2


@torch.inference_mode()
def test_a_head_in_8_bits():
    """Steps, prompts and scores by it are `int8_linear` of the quantised embedding; in bf16 again, as before."""
    model, tokens = _model(0), _tokens(2, 9)
    run = lambda: model.forward(tokens, model.make_cache(2, 12), torch.arange(9, device="cuda"))
    before = run()
    model.quantise_head()
    x, pending = model.stream(tokens, model.make_cache(2, 12), torch.arange(9, device="cuda"))
    last = [y if y is None else y.view(2, 9, -1)[:, -1].contiguous() for y in (x, pending)]
    weight = T.quantise_rows(model.tok_embeddings)
    assert torch.equal(run(), T.int8_linear(model.final_norm(*last), weight))
    scores = model.score(tokens, top=2)
    assert scores.top_ids.shape == (2, 8, 2) and torch.isfinite(scores.logprob).all()
    eager = greedy_decode(model, tokens, 6, use_graph=False)[0]
    assert torch.equal(greedy_decode(model, tokens, 6)[0], eager)
    model.quantise_head(False)
    assert torch.equal(run(), before)


def test_drafts_of_any_kind_and_refusals():
    """A step takes one token at least, whatever the drafts say: roots that are none, tokens outside the vocabulary, parents anywhere."""
    model, count = _model(0), 12
    prompt = _tokens(2, 9)
    lens = torch.tensor([9, 4])
    alone = lambda text, length: (text[:, :5], torch.full((2, 5), -2, device="cuda"))      # (as many rows in the linears: the same bits)
    plain, _ = speculative_decode(model, prompt, count, draft=alone, prompt_lens=lens)

    def nonsense(text, length):
        tokens = torch.tensor([[5, -1, 1 << 40, 1000, 999]], device="cuda").expand(2, 5).contiguous()
        return tokens, torch.tensor([[-2, 0, 0, 7, -1], [3, 0, 1, 2, 1 << 40]], device="cuda")

    got, steps = speculative_decode(model, prompt, count, draft=nonsense, prompt_lens=lens)
    assert torch.equal(got, plain) and steps <= count
    calls = []

    def wider(text, length):
        calls.append(0)
        return torch.zeros((2, len(calls)), dtype=torch.int64, device="cuda"), torch.zeros((2, len(calls)), dtype=torch.int64, device="cuda")

    for draft in (wider, lambda text, length: (text[:, :3], text[:, :2]), lambda text, length: (text[:, :0], text[:, :0]), lambda text, length: (text[:, :2].int(), text[:, :2].int()),
                  lambda text, length: (text[:1, :2], text[:1, :2])):
        with pytest.raises(ValueError, match="speculative_decode"):
            speculative_decode(model, prompt, count, draft=draft)
    for bad in (torch.tensor([9, 10]), torch.tensor([0, 3]), torch.tensor([9]), torch.tensor([-1, 1 << 40])):
        with pytest.raises(ValueError, match="speculative_decode"):
            speculative_decode(model, prompt, count, draft=alone, prompt_lens=bad)
    with pytest.raises(ValueError, match="speculative_decode"):
        speculative_decode(model, prompt.int(), count, draft=alone)


@pytest.mark.parametrize("batch,length", [(1, 40000), (3, 700), (1, 3)])
def test_drafts_captured(batch, length):
    """`ngram_drafts` in a graph that is replayed on other texts, with eager work between, says what it says eagerly."""
    _say("drafts captured", batch, length)
    text, count = torch.zeros((batch, length), dtype=torch.int64, device="cuda"), torch.full((batch,), length, device="cuda")
    ngram_drafts(text, count)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ngram_drafts(text, count)
    for i in range(6):
        text.copy_(_tokens(batch, length, seed=40 + i) % (5 + 40 * i))
        count.copy_(torch.randint(1, length + 1, (batch,), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        want = ngram_drafts(text, count)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("lens", [None, [30, 7, 19, 22]])
def test_speculative_decode_captured(lens):
    """The captured step gives the eager one's tokens, in as many steps."""
    model, prompt = _model(1), _tokens(4, 10).repeat(1, 3)
    lens = None if lens is None else torch.tensor(lens)
    want, steps = speculative_decode(model, prompt, 50, prompt_lens=lens, use_graph=False)
    for graph in (None, True):
        got, replays = speculative_decode(model, prompt, 50, prompt_lens=lens, use_graph=graph)
        assert torch.equal(got, want) and replays == steps
