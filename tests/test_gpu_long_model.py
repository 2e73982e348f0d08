"""The model over a cache in 4 bits, with scaled positions, and the scores of its tokens."""
import pytest
import torch

import ternainfer_amd as T
from ternainfer_amd import _lib
from ternainfer_amd.model import Block, ModelArgs, Transformer, greedy_decode
from tests import _long_context as P

pytestmark = pytest.mark.gpu

SHAPES = [dict(dim=256, n_heads=4, n_kv_heads=2), dict(dim=512, n_heads=4, n_kv_heads=1, rope_adjacent=False)]
YARN = {"type": "yarn", "factor": 8.0, "original_max_position": 64}


def _model(shape, act="int8", seed=21, **more):
    return Transformer(ModelArgs(n_layers=2, vocab_size=1000, ffn_dim=384, **SHAPES[shape], **more), seed=seed, act=act)


def _tokens(*shape, seed=22):
    return torch.randint(0, 1000, shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _prompt_and_steps(model, cache, bsz, plen, steps, per_sequence=False):
    """Logits of a prompt pass and of single-token steps behind it."""
    tokens = _tokens(bsz, plen + steps)
    slots = torch.arange(plen + steps, device="cuda")
    if per_sequence:
        slots = slots.expand(bsz, -1).contiguous()
    return [model.forward(tokens[:, a:b].contiguous(), cache, slots[..., a:b].contiguous())
            for a, b in [(0, plen)] + [(plen + i, plen + i + 1) for i in range(steps)]]


@pytest.mark.parametrize("act,shape,bsz", [("int8", 0, 1), ("int8", 1, 3), ("int8", 0, 12), ("int8", 0, 20), ("bf16", 1, 2)])
@pytest.mark.parametrize("per_sequence", [False, True])
@torch.inference_mode()
def test_attention_is_the_operators_with_the_models_positions(act, shape, bsz, per_sequence, monkeypatch):
    """Every block's attention, in the prompt pass and in steps, is `kv4_store` and `kv4_attention` with the frequencies, pair layout and scale of the
    model: the same bits, from caches that hold the same rows."""
    print(f"[case] blocks over 4 bits {act} {SHAPES[shape]} {bsz} {per_sequence}", flush=True)
    model = _model(shape, act, rope_scaling=YARN)
    a = model.args
    inv, amplitude = T.rotary_frequencies(a.head_dim, a.rope_theta, YARN)
    plain, calls = Block.attend_kv4, []

    def checked(self, qkv, pos, cache, *rope):
        twin = T.Kv4Cache(*(c.clone() for c in cache))
        got = plain(self, qkv, pos, cache, *rope)
        q = T.kv4_store(qkv, pos, inv, twin, a.n_heads, amplitude=amplitude, adjacent=a.rope_adjacent)
        assert torch.equal(got, T.kv4_attention(q, pos, twin, scale=a.head_dim ** -0.5))
        assert all(torch.equal(one, two) for one, two in zip(cache, twin))
        calls.append(qkv.shape[0])
        return got

    monkeypatch.setattr(Block, "attend_kv4", checked)
    logits = _prompt_and_steps(model, model.make_cache(bsz, 40, bits=4), bsz, 17, 2, per_sequence)
    assert calls == [bsz * 17] * 2 + [bsz] * 4 and all(torch.isfinite(y).all() for y in logits)


@pytest.mark.parametrize("act,bsz", [("int8", 1), ("int8", 3), ("int8", 12), ("int8", 20), ("bf16", 2)])
@torch.inference_mode()
def test_what_stands_around_the_attention_is_the_same(act, bsz, monkeypatch):
    """With the attention of the 4-bit cache replaced by that of a bf16 one, a model over 4 bits has the logits of a model over 16, bit for bit: the launches
    around the attention are the same (switched to those that do without what only a bf16 step has: one launch, deferred merges, statistics)."""
    print(f"[case] around the attention {act} {bsz}", flush=True)
    model = _model(0, act)
    model.one_launch_step = model.deferred_attention_merge = False
    for blk in model.layers:
        blk.attention_stats = False
    a, native = model.args, _lib.native()
    held = {}

    def sixteen(self, qkv, pos, cache, inv, amplitude):
        if cache.k.data_ptr() not in held:
            held[cache.k.data_ptr()] = [torch.zeros((bsz, a.n_kv_heads, 40, a.head_dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        rows = model.rope_tables(40, qkv.device).index_select(0, pos.reshape(-1))
        attend = (qkv, rows[:, 0].contiguous(), rows[:, 1].contiguous(), pos, *held[cache.k.data_ptr()], a.n_heads, a.head_dim, a.head_dim ** -0.5, 1)
        if qkv.shape[0] == bsz:
            return native.decode_attention(*attend, model.attention_workspace(bsz), None, None, 0)[0]
        return native.prompt_attention(*attend, True)

    want = _prompt_and_steps(model, model.make_cache(bsz, 40), bsz, 17, 3)
    monkeypatch.setattr(Block, "attend_kv4", sixteen)
    got = _prompt_and_steps(model, model.make_cache(bsz, 40, bits=4), bsz, 17, 3)
    assert len(held) == 2
    for one, two in zip(got, want):
        assert torch.equal(one, two)


@pytest.mark.parametrize("lens", [None, [16, 3, 9]])
@pytest.mark.parametrize("kv_bits", [4, 16])
def test_greedy_decode_over_4_bits_and_its_scores(kv_bits, lens):
    """A captured step and an eager one give the same tokens and scores; these are `token_logprobs` of the logits of a plain loop."""
    print(f"[case] greedy decode {kv_bits} {lens}", flush=True)
    model, prompt, count = _model(0, rope_scaling={"type": "ntk", "factor": 2.0}), _tokens(3, 16), 9
    lens = None if lens is None else torch.tensor(lens)
    a = greedy_decode(model, prompt, count, kv_bits=kv_bits, prompt_lens=lens, logprobs=5)
    b = greedy_decode(model, prompt, count, kv_bits=kv_bits, prompt_lens=lens, logprobs=5, use_graph=False)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[3], b[3]))
    assert [tuple(f.shape) for f in a[3]] == [(3, count)] * 2 + [(3, count, 5)] * 2
    alone = greedy_decode(model, prompt, count, kv_bits=kv_bits, prompt_lens=lens)
    assert len(alone) == 3 and torch.equal(alone[0], a[0])
    none = greedy_decode(model, prompt, count, kv_bits=kv_bits, prompt_lens=lens, logprobs=0)
    assert none[3].top_ids is None and torch.equal(none[3].logprob, a[3].logprob)
    with torch.inference_mode():
        cache = model.make_cache(3, 16 + count, kv_bits)
        at = torch.full((3, 1), 16, device="cuda") if lens is None else lens.cuda().view(3, 1)
        logits = model.forward(prompt, cache, torch.arange(16, device="cuda"), last_idx=at.view(-1) - 1)
        for i in range(count):
            tok = a[0][:, i:i + 1].contiguous()
            assert torch.equal(tok, T.argmax_rows(logits.contiguous()))
            want = T.token_logprobs(logits, tok.view(-1), 5)
            for kept, w in zip(a[3], want):
                assert torch.equal(kept[:, i], w), i
            assert torch.equal(want.logprob, want.top_logprobs[:, 0])
            logits = model.forward(tok, cache, at[0] + i if lens is None else at + i)


@pytest.mark.parametrize("kv_bits,bsz,t", [(16, 2, 30), (4, 2, 30), (4, 1, 2), (16, 1, 2), (4, 3, 65)])
@torch.inference_mode()
def test_score(kv_bits, bsz, t):
    """Scores against the log-softmax in 64 bits of the same stream's logits; in pieces too; padding NaN."""
    print(f"[case] score {kv_bits} {bsz} {t}", flush=True)
    model, tokens = _model(1), _tokens(bsz, t, seed=23)
    got = model.score(tokens, top=3, kv_bits=kv_bits)
    assert [tuple(f.shape) for f in got] == [(bsz, t - 1)] * 2 + [(bsz, t - 1, 3)] * 2
    x, pending = model.stream(tokens[:, :-1].contiguous(), model.make_cache(bsz, t - 1, kv_bits), torch.arange(t - 1, device="cuda"), whole=False)
    h = model.final_norm(x, pending)
    logits = h.double() @ model.tok_embeddings.double().T
    want = torch.log_softmax(logits, -1)
    # A logit is a sum of 512 products in fp32 and its rounding to bf16; a log probability is off by at most twice the largest error of a logit, and by the
    # kernel's own: the exponentials' 2^-15 of the sum at most.
    off = 512 * P.HALF_FP32 * (h.double().abs() @ model.tok_embeddings.double().abs().T).max().item()
    tol = 2 * (off + P.HALF_BF16 * (logits.abs().max().item() + off)) + 2.0 ** -15 + 2.0 ** -20
    target = want.view(bsz, t - 1, -1).gather(-1, tokens[:, 1:, None])[..., 0]
    assert (got.logprob.double() - target).abs().max().item() <= tol
    assert (got.top_logprobs[..., 0].double() - want.view(bsz, t - 1, -1).amax(-1)).abs().max().item() <= tol
    model.score_rows = 7
    pieces = model.score(tokens, top=3, kv_bits=kv_bits)
    assert (pieces.logprob - got.logprob).abs().max().item() <= 2 * tol
    lens = torch.arange(bsz) % t + 1
    padded = model.score(tokens, lens, kv_bits=kv_bits)
    outside = torch.arange(1, t)[None] >= lens[:, None]
    assert torch.equal(torch.isnan(padded.logprob).cpu(), outside) and padded.top_ids is None
    with pytest.raises(ValueError):
        model.score(tokens[:, :1])
    with pytest.raises(ValueError):
        model.score(tokens, torch.ones(bsz + 1, dtype=torch.int64))


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, YARN])
@torch.inference_mode()
def test_tables_of_scaled_positions(scaling):
    """The bf16 cache's tables hold the scaled angles' cosines and sines with the amplitude, each rounded once from 64 bits."""
    model = _model(1, rope_scaling=scaling)
    inv, amplitude = T.rotary_frequencies(128, model.args.rope_theta, scaling)
    angle = torch.arange(100, device="cuda").double()[:, None] * inv
    want = torch.stack([angle.cos(), angle.sin()], 1) * amplitude
    got = model.rope_tables(100, torch.device("cuda:0"))
    assert got.dtype == torch.float32 and ((got.double() - want).abs() <= P.HALF_FP32 * want.abs() + 2.0 ** -50).all()
    assert all(torch.isfinite(y).all() for y in _prompt_and_steps(model, model.make_cache(2, 40), 2, 17, 2))


@torch.inference_mode()
def test_a_cache_longer_than_the_bf16_kernels_take(monkeypatch):
    """9000 slots: a step behind a long text attends over all of it, its first token too, whose values are then made larger.  (Whether the logits change is up
    to the weights that a random model gives that token; the attention is held against 64 bits.)"""
    print("[case] 9000 slots", flush=True)
    model = _model(0)
    a = model.args
    cache = model.make_cache(1, 9000, bits=4)
    tokens = _tokens(1, 8990, seed=24)
    for first in range(0, 8990, 2997):
        last = min(first + 2997, 8990)
        model.forward(tokens[:, first:last].contiguous(), cache, torch.arange(first, last, device="cuda"))
    plain, calls = Block.attend_kv4, []

    def checked(self, qkv, pos, held, inv, amplitude):
        got = plain(self, qkv, pos, held, inv, amplitude)
        q = T.kv4_store(qkv, pos, inv, held, a.n_heads, amplitude=amplitude)           # (the same row once more)
        want, tol = P.attention(q, pos, held, a.head_dim ** -0.5)
        assert P.same_or_near(got.view(1, 1, a.n_heads, a.head_dim), want, tol) <= 0
        calls.append(qkv.shape[0])
        return got

    monkeypatch.setattr(Block, "attend_kv4", checked)
    step = lambda: model.forward(tokens[:, :1].contiguous(), cache, torch.tensor([8990], device="cuda"))
    one, two = step(), step()
    assert torch.equal(one, two) and torch.isfinite(one).all()
    for held in cache:
        held.v_scale[:, :, 0] = 140
    step()
    assert calls == [1] * 6


@torch.inference_mode()
def test_what_a_cache_in_4_bits_does_not_take():
    model = _model(0)
    cache = model.make_cache(1, 8, bits=4)
    for blk in model.layers:
        blk.fused = False
    with pytest.raises(ValueError):
        model.forward(_tokens(1, 4), cache, torch.arange(4, device="cuda"))
    with pytest.raises(ValueError):
        model.make_cache(1, 8, bits=8)


@torch.inference_mode()
def test_tokens_outside_the_vocabulary_do_not_fault():
    """As over the bf16 cache: a prompt's row of such a token is NaN, and nothing but it and those that see it."""
    model = _model(0)
    tokens = _tokens(2, 12, seed=25)
    clean = model.forward(tokens, model.make_cache(2, 16, bits=4), torch.arange(12, device="cuda"))
    tokens[1, 5] = 1 << 40
    got = model.forward(tokens, model.make_cache(2, 16, bits=4), torch.arange(12, device="cuda"))
    assert torch.equal(got[0], clean[0]) and torch.isnan(got[1]).all()


@torch.inference_mode()
def test_blocks_of_a_users_own_run_as_before(monkeypatch):
    """A block whose methods know nothing of a cache in 4 bits is called without it."""
    model = _model(0)
    want = _prompt_and_steps(model, model.make_cache(2, 40), 2, 17, 2)
    forward, chain = Block.forward, Block.forward_chain
    monkeypatch.setattr(Block, "forward", lambda self, x, pending, cache_k, cache_v, pos_idx, cos, sin, mask, attn_ws=None:
                        forward(self, x, pending, cache_k, cache_v, pos_idx, cos, sin, mask, attn_ws))
    monkeypatch.setattr(Block, "forward_chain", lambda self, x, stats, cache_k, cache_v, pos_idx, cos, sin, attn_ws, next_norm, split=False:
                        chain(self, x, stats, cache_k, cache_v, pos_idx, cos, sin, attn_ws, next_norm, split))
    model.one_launch_step = False
    got = _prompt_and_steps(model, model.make_cache(2, 40), 2, 17, 2)
    assert all(torch.equal(one, two) for one, two in zip(got, want))
