"""Calls of ternainfer_amd/drafting.py, int8_linear.py and of the model's steps over trees at the edges of what their documentation allows."""
import pytest
import torch

import ternainfer_amd as T
import ternainfer_amd.model as model_module
from ternainfer_amd.model import ModelArgs, Transformer, greedy_decode, speculative_decode
from tests import _drafting as P
from tests._long_context import same_or_near

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=_gen(seed), device="cuda").to(dtype)


def _say(*what):
    print("[case]", *what, flush=True)


# rows a kv head: 8 and 60 (workgroups of 32 and 64 rows), 80 and more (128), in one group of waves and in two, in one part and in several
SHAPES = [(1, 8, 2, 2, 60), (1, 30, 4, 2, 60), (1, 40, 4, 2, 60), (2, 40, 1200, 300, 60), (1, 64, 8, 1, 90), (1, 40, 20, 5, 8000), (40, 40, 20, 5, 300)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,h,kv,slots", SHAPES)
def test_values_that_nearly_cancel(d, b, t, h, kv, slots):
    """Large values of both signs, two slots in front of the tree with most of the weight: probabilities count to 2^-15, however many rows there are.  The tolerance
    is the oracle's of up to 64 rows a kv head, for every one of the heads that share it taken by itself."""
    _say("nearly cancelling", d, b, t, h, kv, slots)
    start = slots - t - 3
    q, k = _randn((b, h, t, d), 1), _randn((b, kv, slots, d), 2)
    q[..., 0], k[..., 0] = d ** 0.5, 0.0
    k[:, :, 5], k[:, :, start - 2] = 0.0, 0.0
    k[:, :, 5, 0], k[:, :, start - 2, 0] = 9.0, 9.0                                       # scores of 9 and a little, where others are about 1
    k[:, :, 5, 1:9], k[:, :, start - 2, 1:9] = _randn((b, kv, 8), 3), _randn((b, kv, 8), 4)
    v = _randn((b, kv, slots, d), 5)
    v[:, :, 5], v[:, :, start - 2] = 200.0, -200.0
    mask = T.draft_tree(P.random_parents(b, t, 6).cuda()).mask
    at = torch.full((b,), start, device="cuda")
    got = T.tree_attention(q, k, v, at, mask).view(b, t, h, d)
    group = h // kv
    for first in range(min(group, 2)):                                                    # (t rows a head here: 64 at most)
        heads = torch.arange(first, h, group, device="cuda")
        some = slice(0, 2)
        want, tol = P.attention(q[some, heads], k[some], v[some], at[some], mask[some], d ** -0.5)
        assert same_or_near(got[some][:, :, heads], want, tol) <= 0


@pytest.mark.parametrize("b,t,h,kv,slots", SHAPES)
def test_scores_that_overflow(b, t, h, kv, slots):
    """Scores whose product with the scale is beyond float32: NaN, as in elementary operations, whatever the layout of the rows -- not the zeros of a row that sees
    nothing.  Rows with nothing to see stay zeros."""
    _say("overflow", b, t, h, kv, slots)
    start = slots - t - 3
    q, k, v = _randn((b, h, t, 128), 10).abs(), _randn((b, kv, slots, 128), 11).abs(), _randn((b, kv, slots, 128), 12)
    parents = P.random_parents(b, t, 13)
    parents[:, -1] = -2
    got = T.tree_attention(q, k, v, torch.full((b,), start, device="cuda"), T.draft_tree(parents.cuda()).mask, 2e38).view(b, t, h, 128)
    assert got[:, :-1].isnan().all() and not got[:, -1].any()


# ---- moving rows -------------------------------------------------------------------------------------------------------------------


def test_caches_of_one_slot_stay():
    """Nothing moves in them; a stride between slots that are not there says nothing."""
    start, path, count = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.tensor([[0, 2], [1, 3]], device="cuda"), torch.tensor([2, 2], device="cuda")
    one = torch.randn(2 * 3 * 16, device="cuda").as_strided((2, 3, 1, 16), (48, 16, 1, 1))
    more, was = _randn((2, 3, 5, 16), 60), _randn((2, 3, 5, 16), 60)
    before = one.clone()
    T.cache_move([one, more], start, path, count)
    was[0, :, 1], was[1, :, 0], was[1, :, 1] = was[0, :, 2].clone(), was[1, :, 1].clone(), was[1, :, 3].clone()
    assert torch.equal(one, before) and torch.equal(more, was)


# ---- the model -----------------------------------------------------------------------------------------------------------------------


def _model(**more):
    """Scales that end at no multiple of 128 columns: 512 columns of three."""
    return Transformer(ModelArgs(n_layers=2, vocab_size=1000, ffn_dim=384, dim=256, n_heads=4, n_kv_heads=2, **more), seed=31)


# How far logits of two ways to the same step may be apart, in deviations of a row of logits.  Where the bfloat16 roundings of the two ways differ, an int8 code in front
# of a linear may be its neighbour: a unit, a 127th of the row's largest element.  That is 3 times the rms of 256 elements of a normal row and some 10 times that of 384 gated ones
# (squares times another), so that codes that all move change an output by 3 / 127 = 2.4 % and 8 %.  A code of 30 units is moved by up to 30 * 2^-8 = 0.12 units before it is
# rounded, so about one in ten changes: 0.1 ** 0.5 of that, 0.8 % and 2.5 %.  Two blocks have six linears of the one kind and two of the other, whose errors are independent: (6 * 0.8 ** 2 +
# 2 * 2.5 ** 2) ** 0.5 = 4 % a logit, 5.7 % the difference of two.  Four deviations of that are 23 % (one of 16000 is beyond), five of a single logit's 20 % (one of 1.7 million).
NEAR = 0.25


def _tokens(*shape, seed=32):
    return torch.randint(0, 1000, shape, generator=torch.Generator().manual_seed(seed)).cuda()


@torch.inference_mode()
def test_more_than_64_rows_by_the_decode_rule():
    """Keys and values of the first block, bit for bit those of the sequences' own steps, of fewer rows."""
    bsz, t, plen = 4, 30, 17
    model, prompt, tokens = _model(), _tokens(bsz, plen), _tokens(bsz, t, seed=33)
    tree, start = T.draft_tree(P.random_parents(bsz, t, 34).cuda()), torch.full((bsz,), plen, device="cuda")
    cache = model.make_cache(bsz, plen + t)
    model.forward(prompt, cache, torch.arange(plen, device="cuda"))
    alone = [tuple(c.clone() for c in pair) for pair in cache]
    logits = model.tree_step(tokens, cache, start, tree, decode_rule=True)
    for b in range(bsz):
        mine = [tuple(c[b:b + 1].contiguous() for c in pair) for pair in alone]
        own = model.tree_step(tokens[b:b + 1], mine, start[b:b + 1], T.DraftTree(tree.mask[b:b + 1], tree.depth[b:b + 1]))
        assert all(torch.equal(c[b], m[0]) for c, m in zip(cache[0], mine[0])), b
        assert (logits[b].float() - own[0].float()).abs().max() <= NEAR * own.float().std()


@pytest.mark.parametrize("head8", [False, True])
def test_speculative_decode_of_more_than_64_rows_against_greedy_steps(head8):
    """Eight sequences of nine nodes: every token is the likeliest behind the same text of `greedy_decode`'s steps, but for logits nearer to it than the two ways' roundings
    (by the rule of the scales that more rows follow, they are up to five deviations apart)."""
    model, count, bsz = _model(), 30, 8
    if head8:
        model.quantise_head()
    prompt = _tokens(bsz, 8, seed=35).repeat(1, 2)
    got, steps = speculative_decode(model, prompt, count, decode_rule=True)
    assert got.shape == (bsz, count) and steps < count
    with torch.inference_mode():
        cache = model.make_cache(bsz, 16 + count)
        logits = model.forward(prompt, cache, torch.arange(16, device="cuda"))
        for i in range(count):
            rows = logits.float()
            assert (rows.amax(-1) - rows.gather(1, got[:, i:i + 1])[:, 0] <= NEAR * rows.std(-1)).all(), i
            logits = model.forward(got[:, i:i + 1].contiguous(), cache, torch.tensor([16 + i], device="cuda"))


@torch.inference_mode()
def test_what_a_tree_step_refuses_leaves_the_cache_as_it_was():
    model, tokens = _model(), _tokens(2, 5)
    tree, start = T.draft_tree(P.random_parents(2, 5, 40).cuda()), torch.tensor([3, 4], device="cuda")
    cache = model.make_cache(2, 20)
    wide = tree.mask.expand(2, 5, 2).contiguous()
    for bad in ((tokens.int(), start, tree), (tokens[0], start, tree), (tokens[:, :0], start, tree), (tokens[:1], start[:1], T.DraftTree(tree.mask[:1], tree.depth[:1])), (tokens, start.int(), tree),
                (tokens, start.cpu(), tree), (tokens, start[:1], tree), (tokens, start, tree._replace(mask=wide)), (tokens, start, tree._replace(mask=tree.mask.int())),
                (tokens, start, tree._replace(mask=tree.mask[:, :4])), (tokens, start, tree._replace(mask=tree.mask.cpu())), (tokens, start, tree._replace(depth=tree.depth.int())),
                (tokens, start, tree._replace(depth=tree.depth[:, :4])), (tokens, start, tree._replace(depth=tree.depth.cpu())), (tokens.repeat(1, 103), start, tree)):
        with pytest.raises(ValueError, match="tree_step"):
            model.tree_step(bad[0], cache, *bad[1:])
        assert not any(c.any() for pair in cache for c in pair)
    model.tree_step(tokens, cache, start, tree)
    assert all(c.any() for pair in cache for c in pair)


def test_scores_a_few_rows_at_a_time(monkeypatch):
    """Rows of a text are projected by the matrix product of many rows, however few `score_rows` are."""
    model, tokens = _model(), _tokens(2, 20)
    monkeypatch.setattr(model_module, "lm_head", None)
    rows, plain = [], model_module.F.linear
    monkeypatch.setattr(model_module.F, "linear", lambda x, w: rows.append(x.shape[0]) or plain(x, w))
    for model.score_rows in (3, 16, 1024):
        assert model.score(tokens).logprob.shape == (2, 19)
    assert rows == [3] * 12 + [2] + [16, 16, 6] + [38]


@pytest.mark.parametrize("decode", [speculative_decode, greedy_decode])
@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 2.0}])
def test_a_decode_of_another_length_between_replays(decode, scaling, monkeypatch):
    """A captured step keeps its rotary table while other lengths are decoded with the same model: the same tokens."""
    model, prompt = _model(rope_scaling=scaling), _tokens(2, 8, seed=50).repeat(1, 2)
    want, replay, kept, replays = decode(model, prompt, 20)[0], torch.cuda.CUDAGraph.replay, [], []

    def disturbed(graph):
        replays.append(0)
        model.rope_tables(50 + len(replays), prompt.device)
        kept.extend(torch.full((36 + 9 * (decode is speculative_decode), 2, 32), float("nan"), device="cuda") for _ in range(8))      # where a table that was let go of may lie
        replay(graph)

    monkeypatch.setattr(torch.cuda.CUDAGraph, "replay", disturbed)
    got = decode(model, prompt, 20)[0]
    assert len(replays) > 3 and torch.equal(got, want)


@torch.inference_mode()
def test_blocks_and_linears_that_know_no_rule():
    """A prompt and a step over trees through blocks and linears of a caller's own, which take what they took before there was a rule to choose."""
    model, tokens = _model(), _tokens(2, 9)
    calls = []

    class Linear:
        def __init__(self, of):
            self.__dict__.update(of.__dict__)
            self.of = of

        def quantised(self, xq, s):
            calls.append(xq.shape[0])
            return self.of.quantised(xq, s)

    class Own(model_module.Block):
        def _norm_linear(self, lin, x, weight, residual=None, glu=False, name=None):
            return super()._norm_linear(lin, x, weight, residual, glu, name)

    tree, start = T.draft_tree(P.random_parents(2, 9, 70).cuda()), torch.tensor([0, 0], device="cuda")
    want = model.tree_step(tokens, model.make_cache(2, 12), start, tree)
    for blk in model.layers:
        blk.__class__ = Own
        blk.w2 = Linear(blk.w2)
    assert torch.equal(model.tree_step(tokens, model.make_cache(2, 12), start, tree), want) and calls == [18, 18]
    plain = model.tree_step
    model.tree_step = lambda tokens, cache, start, tree: plain(tokens, cache, start, tree)
    assert speculative_decode(model, tokens, 5)[0].shape == (2, 5)
