"""The operators of ternainfer_amd/long_context.py against plain implementations in 64 bits."""
import ctypes
import math

import pytest
import torch

import ternainfer_amd as T
from ternainfer_amd import _lib
from tests import _long_context as P

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=_gen(seed), device="cuda").to(dtype)


def _say(*what):
    print("[case]", *what, flush=True)


# ---- rotary ------------------------------------------------------------------------------------------------------------------------


def _check_rotary(x, got, pos, inv_freq, amplitude, adjacent):
    want, bound = P.turned(x.double(), pos, inv_freq, amplitude, adjacent)
    # cos or sin rounded (and times the amplitude: the rounding covers both), a product, the sum: three roundings of at most amplitude (|a| + |b|) each;
    # then the output's own.  Copied elements are the same.
    out = P.HALF_BF16 if x.dtype == torch.bfloat16 else P.HALF_FP32
    tol = 3.01 * P.HALF_FP32 * bound + out * (want.abs() + 3.01 * P.HALF_FP32 * bound) * (bound > 0)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert P.same_or_near(got, want, tol) <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("adjacent", [True, False])
@pytest.mark.parametrize("b,t,h,d,r", [(1, 1, 1, 2, 2), (3, 1, 25, 128, 128), (2, 37, 5, 64, 32), (1, 700, 3, 80, 20), (2, 5, 7, 66, 66), (5, 3, 4, 256, 2), (1, 3, 2, 1024, 1024), (4, 300, 1, 8, 6)])
def test_rotary(dtype, adjacent, b, t, h, d, r):
    _say("rotary", dtype, adjacent, b, t, h, d, r)
    x = _randn((b, t, h, d), 1, dtype)
    inv, _ = T.rotary_frequencies(r, 10000.0)
    pos = torch.randint(0, 200000, (b, t), generator=_gen(2), device="cuda")
    got = T.rotary_embed(x, pos, inv, adjacent=adjacent, amplitude=1.25)
    assert got.is_contiguous()
    _check_rotary(x, got, pos, inv, 1.25, adjacent)
    shared = T.rotary_embed(x, pos[0], inv, adjacent=adjacent)
    _check_rotary(x, shared, pos[0], inv, 1.0, adjacent)


@pytest.mark.parametrize("adjacent", [True, False])
@pytest.mark.parametrize("cut", [0, 3, 8])
def test_rotary_on_views_and_in_place(adjacent, cut):
    """A view of a projection's rows: the other heads stay; rows that start at any element; a broadcast head; a last dimension that is not contiguous."""
    rows = _randn((2, 9, 12, 128), 3)
    inv, _ = T.rotary_frequencies(64)
    pos = torch.arange(100, 109, device="cuda")
    x = rows[:, :, 2:9, cut:cut + 72]
    before = rows.clone()
    _check_rotary(x, T.rotary_embed(x, pos, inv, adjacent=adjacent), pos, inv, 1.0, adjacent)
    assert torch.equal(rows, before)
    out = torch.zeros((2, 9, 7, 80), dtype=torch.bfloat16, device="cuda")
    assert T.rotary_embed(x, pos, inv, adjacent=adjacent, out=out[..., 1:73]).data_ptr() == out[..., 1:].data_ptr()
    _check_rotary(x, out[..., 1:73], pos, inv, 1.0, adjacent)
    assert not out[..., 0].any() and not out[..., 73:].any()
    assert T.rotary_embed(x, pos, inv, adjacent=adjacent, out=x) is not None
    _check_rotary(before[:, :, 2:9, cut:cut + 72], x, pos, inv, 1.0, adjacent)
    rows[:, :, 2:9, cut:cut + 72] = before[:, :, 2:9, cut:cut + 72]
    assert torch.equal(rows, before)
    wide = before[:, :, :1].expand(2, 9, 4, 128)
    _check_rotary(wide, T.rotary_embed(wide, pos, inv, adjacent=adjacent), pos, inv, 1.0, adjacent)
    across = before.transpose(2, 3)[..., :64, :].transpose(2, 3)
    _check_rotary(across, T.rotary_embed(across, pos, inv, adjacent=adjacent), pos, inv, 1.0, adjacent)
    turned = before.transpose(2, 3).contiguous().transpose(2, 3)             # last dimension strided
    _check_rotary(turned, T.rotary_embed(turned, pos, inv, adjacent=adjacent), pos, inv, 1.0, adjacent)


def test_rotary_far_and_negative_positions():
    x = _randn((1, 6, 2, 64), 4, torch.float32)
    inv, _ = T.rotary_frequencies(64)
    pos = torch.tensor([0, -1, -70000, 1 << 20, (1 << 31) + 7, -(1 << 33)], device="cuda")
    _check_rotary(x, T.rotary_embed(x, pos, inv), pos, inv, 1.0, True)
    # a quarter, a half, three quarters and whole turns, where the angle's reduction changes its branch
    quarter = torch.tensor([math.pi / 2], dtype=torch.float64, device="cuda")
    y = T.rotary_embed(x[..., :2], torch.arange(6, device="cuda"), quarter)
    _check_rotary(x[..., :2], y, torch.arange(6, device="cuda"), quarter, 1.0, True)


def test_rotary_of_nothing_and_refusals():
    inv = torch.ones(4, dtype=torch.float64, device="cuda")
    x = _randn((2, 3, 2, 8), 5)
    pos = torch.arange(3, device="cuda")
    assert T.rotary_embed(x[:, :0], pos[:0], inv).shape == (2, 0, 2, 8) and T.rotary_embed(x[:0], pos, inv).shape == (0, 3, 2, 8)
    for call in (lambda: T.rotary_embed(x[0], pos, inv), lambda: T.rotary_embed(x.half(), pos, inv), lambda: T.rotary_embed(x, pos[:2], inv), lambda: T.rotary_embed(x, pos.int(), inv),
                 lambda: T.rotary_embed(x, pos[None], inv), lambda: T.rotary_embed(x, pos.cpu(), inv), lambda: T.rotary_embed(x, pos, inv.float()), lambda: T.rotary_embed(x, pos, inv.cpu()),
                 lambda: T.rotary_embed(x, pos, torch.cat([inv, inv])), lambda: T.rotary_embed(x, pos, inv[:0]), lambda: T.rotary_embed(x, pos, inv, out=x[:1]),
                 lambda: T.rotary_embed(x, pos, inv, out=x.float()), lambda: T.rotary_embed(x[:, :2], pos[:2], inv, out=x[:, 1:]),
                 lambda: T.rotary_embed(x[:1].expand(2, 3, 2, 8), pos, inv, out=x[:1].expand(2, 3, 2, 8)), lambda: T.rotary_embed(x, pos, inv, out=torch.empty_like(x.transpose(2, 3).contiguous()).transpose(2, 3))):
        with pytest.raises(ValueError, match="rotary_embed"):
            call()


# ---- store and rows ------------------------------------------------------------------------------------------------------------------


def _stored(cache, at):
    """Values and scale exponents of keys and values at slots at [B, T]: [B, T, KV, ...]."""
    b = torch.arange(at.shape[0], device="cuda")[:, None]
    got = []
    for codes, scales in (cache[:2], cache[2:]):
        got.append((P.values(codes[b, :, at], scales[b, :, at]), scales[b, :, at].double() - 127))
    return got


@pytest.mark.parametrize("adjacent", [True, False])
@pytest.mark.parametrize("b,t,h,kv,d,r,slots", [(1, 1, 1, 1, 64, 64, 1), (2, 1, 20, 5, 128, 128, 40), (3, 33, 4, 2, 128, 32, 200), (1, 700, 5, 1, 64, 22, 700), (2, 17, 16, 2, 128, 90, 64)])
def test_store(adjacent, b, t, h, kv, d, r, slots):
    _say("store", adjacent, b, t, h, kv, d, r, slots)
    cache = T.Kv4Cache(*P.random_cache(b, kv, slots, d, 7))
    before = [c.clone() for c in cache]
    wide = _randn((b * t, (h + 2 * kv) * d + 8), 8)
    x = wide[:, :-8]                                                             # rows further apart than their length
    inv, _ = T.rotary_frequencies(r)
    pos = torch.stack([torch.randperm(slots, generator=_gen(9 + i), device="cuda")[:t] for i in range(b)])
    pos[-1, t // 2] = -1 if t > 1 else 0                                         # padding
    if t > 2:
        pos[0, 1] = slots                                                        # outside
    q = T.kv4_store(x, pos, inv, cache, h, adjacent=adjacent, amplitude=1.125)
    rows = x.double().view(b, t, h + 2 * kv, d)
    want, bound = P.turned(rows, pos, inv, 1.125, adjacent)
    arithmetic = 3.01 * P.HALF_FP32 * bound
    tol = arithmetic + P.HALF_BF16 * (want.abs() + arithmetic)
    assert q.shape == (b, h, t, d) and P.same_or_near(q, want[:, :, :h].transpose(1, 2), tol[:, :, :h].transpose(1, 2)) <= 0

    inside = (pos >= 0) & (pos < slots)
    (keys, key_e), (vals, val_e) = _stored(cache, pos.clamp(0, slots - 1))
    # values are not turned: exactly the nearest codes
    v = rows[:, :, h + kv:]
    e = P.scale_exponents(v.abs().unflatten(-1, (-1, 32)).amax(-1))
    assert torch.equal(val_e[inside], e[inside]) and torch.equal(vals[inside], P.round_codes(v, e)[inside])
    # keys: turned in fp32 with the error `arithmetic`; rounding and choice of scale are monotonous, so the results of the two ends bracket them
    k, slack = want[:, :, h:h + kv], arithmetic[:, :, h:h + kv]
    groups = k.abs().unflatten(-1, (-1, 32))
    slack_groups = slack.unflatten(-1, (-1, 32))
    low, high = P.scale_exponents((groups - slack_groups).amax(-1).clamp(min=0)), P.scale_exponents((groups + slack_groups).amax(-1))
    assert ((low <= key_e) & (key_e <= high))[inside].all()
    assert ((P.round_codes(k - slack, key_e) <= keys) & (keys <= P.round_codes(k + slack, key_e)))[inside].all()

    # other slots are as they were
    b_at = torch.arange(b, device="cuda")[:, None].expand(b, t)
    for now, then in zip(cache, before):
        then[b_at[inside], :, pos[inside]] = now[b_at[inside], :, pos[inside]]
        assert torch.equal(now, then)
    # rows read back: the values, exactly
    k_rows, v_rows = T.kv4_rows(cache, pos)
    assert k_rows.dtype == torch.bfloat16 and k_rows.shape == (b, t, kv, d)
    assert torch.equal(k_rows.double()[inside], keys[inside]) and torch.equal(v_rows.double()[inside], vals[inside])
    assert torch.isnan(k_rows[~inside]).all() and torch.isnan(v_rows[~inside]).all()


def test_store_at_every_border_and_at_the_ends_of_the_range():
    """Values on the borders between codes and next to them, powers of two over the whole range of bf16, zeros, signs, NaN, infinities."""
    halves = torch.arange(0, 33, device="cuda").float() / 4
    near = torch.cat([halves, halves * (1 + 2.0 ** -7), halves * (1 - 2.0 ** -8)])
    rows = []
    for e in (-133, -130, -127, -126, -125, -124, -60, -3, 0, 1, 70, 119, 120, 121, 122, 123):
        for peak in (4.0, 6.0, 6.9375, 7.0, 7.0625, 7.96875):
            for part in near.split(31):
                row = torch.zeros(32, device="cuda")
                row[:part.numel()] = part.clamp(max=peak)
                row[31] = peak
                rows.append(torch.ldexp(row.double(), torch.tensor(e, device="cuda")).to(torch.bfloat16))
    rows.append(torch.zeros(32, device="cuda").to(torch.bfloat16))
    rows.append(torch.full((32,), torch.finfo(torch.bfloat16).max, device="cuda").to(torch.bfloat16))
    signs = torch.where(torch.rand((len(rows), 32), generator=_gen(10), device="cuda") < 0.5, -1.0, 1.0).to(torch.bfloat16)
    x = torch.stack(rows) * signs
    n = x.shape[0] // 4 * 4
    x = torch.cat([x[:n], x[-4:]]).view(-1, 128)
    t = x.shape[0]
    cache = T.Kv4Cache.empty(1, 1, t, 128)
    T.kv4_store(torch.cat([x, x, x], 1), torch.arange(t, device="cuda"), torch.zeros(64, dtype=torch.float64, device="cuda"), cache, 1)   # angle 0: nothing turns
    e = P.scale_exponents(x.double().abs().unflatten(-1, (-1, 32)).amax(-1))
    want = P.round_codes(x.double(), e)
    for codes, scales in (cache[:2], cache[2:]):
        assert torch.equal(scales[0, 0].double() - 127, e)
        assert torch.equal(P.values(codes[0, 0], scales[0, 0]), want)
    assert torch.equal(T.kv4_rows(cache, torch.arange(t, device="cuda"))[1][0, :, 0].double(), want)
    # a group with NaN or an infinity stands for NaN, its neighbours do not
    for broken in (math.nan, math.inf, -math.inf):
        row = torch.ones((1, 384), dtype=torch.bfloat16, device="cuda")
        row[0, 256 + 33] = broken
        T.kv4_store(row, torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(64, dtype=torch.float64, device="cuda"), cache, 1)
        assert cache.v_scale[0, 0, 0].tolist() == [125, 255, 125, 125] and cache.v[0, 0, 0, 16:32].eq(0).all()
        back = T.kv4_rows(cache, torch.zeros(1, dtype=torch.int64, device="cuda"))[1][0, 0, 0]
        assert torch.isnan(back[32:64]).all() and back[:32].eq(1).all() and back[64:].eq(1).all()


def test_store_refusals_and_nothing_to_store():
    inv = torch.ones(64, dtype=torch.float64, device="cuda")
    cache = T.Kv4Cache.empty(2, 2, 16, 128)
    x, pos = _randn((6, 8 * 128), 11), torch.arange(3, device="cuda")
    assert T.kv4_store(x[:0], pos[:0], inv, cache, 4).shape == (2, 4, 0, 128)
    assert T.kv4_store(x[:0], pos[:0], inv, T.Kv4Cache.empty(0, 2, 16, 128), 4).shape == (0, 4, 0, 128)
    assert T.kv4_rows(cache, pos[:0])[0].shape == (2, 0, 2, 128)
    bad = lambda **kw: T.Kv4Cache(*(kw.get(n, getattr(cache, n)) for n in cache._fields))
    for call in (lambda: T.kv4_store(x, pos, inv, cache, 3), lambda: T.kv4_store(x[:5], pos, inv, cache, 4), lambda: T.kv4_store(x.float(), pos, inv, cache, 4), lambda: T.kv4_store(x[:, :-8], pos, inv, cache, 4),
                 lambda: T.kv4_store(x, pos[:2], inv, cache, 4), lambda: T.kv4_store(x, pos, inv.float(), cache, 4), lambda: T.kv4_store(x, pos, torch.cat([inv, inv]), cache, 4),
                 lambda: T.kv4_store(x, pos.cpu(), inv, cache, 4), lambda: T.kv4_store(x.cpu(), pos, inv, cache, 4), lambda: T.kv4_store(x, pos, inv, bad(k=cache.k[:1]), 4),
                 lambda: T.kv4_store(x, pos, inv, bad(v_scale=cache.v_scale[:, :, :, :2]), 4), lambda: T.kv4_store(x, pos, inv, bad(v=cache.v.char()), 4),
                 lambda: T.kv4_store(x, pos, inv, bad(v=cache.v.cpu()), 4), lambda: T.kv4_store(x, pos, inv, bad(k=cache.k.transpose(1, 2).contiguous().transpose(1, 2)), 4),
                 lambda: T.kv4_store(x, pos, inv, bad(k=torch.empty(cache.k.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(cache.k.shape)), 4),
                 lambda: T.kv4_step(x, pos, inv, cache, 4), lambda: T.kv4_step(x[:2], pos[:2], inv, cache, 4), lambda: T.kv4_rows(cache, pos.int()), lambda: T.kv4_rows(cache, torch.zeros((3, 1), dtype=torch.int64, device="cuda")),
                 lambda: T.kv4_attention(_randn((2, 3, 1, 128), 1), pos[:1], cache), lambda: T.kv4_attention(_randn((1, 4, 1, 128), 1), pos[:1], cache),
                 lambda: T.kv4_attention(_randn((2, 4, 1, 64), 1), pos[:1], cache), lambda: T.kv4_attention(_randn((2, 4, 1, 128), 1).float(), pos[:1], cache),
                 lambda: T.kv4_attention(_randn((2, 4, 2, 128), 1), pos[:1], cache)):
        with pytest.raises(ValueError, match="kv4_"):
            call()


# ---- attention -----------------------------------------------------------------------------------------------------------------------


def _attend(q, pos, cache, scale=None):
    got = T.kv4_attention(q, pos, cache, scale)
    b, h, t, d = q.shape
    want, tol = P.attention(q, pos, cache, d ** -0.5 if scale is None else scale)
    assert got.dtype == torch.bfloat16 and got.shape == (b * t, h * d)
    assert P.same_or_near(got.view(b, t, h, d), want, tol) <= 0
    return got


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 511]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,kv", [(1, 1), (4, 1), (20, 5), (10, 2), (16, 1), (17, 1), (6, 3)])
def test_attention_of_single_tokens(d, h, kv):
    """Every length around the steps of 32 slots and the four waves' rounds, an empty row, a position behind the cache; the rest of the cache holds other rows."""
    slots = 512
    pos = torch.tensor([[n - 1] for n in LENGTHS] + [[slots - 1], [slots], [1 << 40], [-(1 << 40)]], device="cuda")
    b = pos.shape[0]
    _say("attention", d, h, kv)
    cache = T.Kv4Cache(*P.random_cache(b, kv, slots, d, 20))
    _attend(_randn((b, h, 1, d), 21), pos, cache)


@pytest.mark.parametrize("b,t,h,kv,d,slots", [(2, 2, 4, 1, 128, 40), (1, 5, 20, 5, 128, 333), (2, 33, 6, 2, 64, 100), (1, 70, 8, 8, 128, 97), (1, 130, 8, 2, 128, 260), (1, 129, 5, 1, 64, 300), (3, 1, 20, 5, 128, 1),
                                              (1, 300, 4, 1, 128, 300), (1, 200, 16, 1, 64, 1000), (2, 90, 3, 1, 128, 200)])
def test_attention_of_several_tokens(b, t, h, kv, d, slots):
    _say("attention", b, t, h, kv, d, slots)
    cache = T.Kv4Cache(*P.random_cache(b, kv, slots, d, 30))
    start = torch.tensor([(slots - t) // (i + 1) for i in range(b)], device="cuda")
    pos = start[:, None] + torch.arange(t, device="cuda")
    _attend(_randn((b, h, t, d), 31), pos, cache)
    _attend(_randn((b, h, t, d), 32), torch.arange(t, device="cuda") + (slots - t), cache, scale=0.02)
    # in any order, some padded, some behind the cache
    mixed = torch.randint(-1, slots, (b, t), generator=_gen(33), device="cuda")
    mixed[0, 0] = slots if t > 1 else 0
    _attend(_randn((b, h, t, d), 34), mixed, cache)


def test_attention_with_nothing_to_see_and_nothing_to_do():
    cache = T.Kv4Cache(*P.random_cache(2, 1, 64, 128, 40))
    q = _randn((2, 4, 9, 128), 41)
    assert not T.kv4_attention(q, torch.full((9,), -1, device="cuda"), cache).any()
    assert T.kv4_attention(q[:, :, :0], torch.zeros(0, dtype=torch.int64, device="cuda"), cache).shape == (0, 512)


@pytest.mark.parametrize("t", [1, 3, 40, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_slots_that_a_row_does_not_see_do_not_reach_it(t, d):
    """Whatever they hold: any byte as a scale, the one that stands for NaN among them."""
    slots, h, kv = 400, 8, 2
    cache = T.Kv4Cache(*P.random_cache(1, kv, slots, d, 50))
    pos = torch.arange(t, device="cuda") * 150 // t + 37
    q = _randn((1, h, t, d), 51)
    clean = _attend(q, pos, cache)
    last = int(pos[-1])
    for fill in (255, 254, 253, 0):
        dirty = T.Kv4Cache(*(c.clone() for c in cache))
        for c in dirty:
            c[:, :, last + 1:] = torch.randint(0, 256, c[:, :, last + 1:].shape, generator=_gen(52), device="cuda", dtype=torch.uint8)
        dirty.v_scale[:, :, last + 1:] = fill
        dirty.k_scale[:, :, last + 1:] = fill
        assert torch.equal(T.kv4_attention(q, pos, dirty), clean)
    if t > 1:                                                                    # within the tokens: rows in front of the slot are clean, those behind it see it
        middle = int(pos[t // 2])
        for name in ("k_scale", "v_scale"):
            dirty = T.Kv4Cache(*(c.clone() for c in cache))
            getattr(dirty, name)[0, 1, middle, -1] = 255
            got = _attend(q, pos, dirty).view(t, h, d)
            assert torch.equal(got[:t // 2], clean.view(t, h, d)[:t // 2])
            assert torch.isnan(got[t // 2:, 4:, -32:]).all() and torch.equal(got[:, :4], clean.view(t, h, d)[:, :4])


def test_attention_of_queries_that_are_not_finite():
    cache = T.Kv4Cache(*P.random_cache(1, 1, 100, 128, 60))
    for broken in (math.nan, math.inf, -math.inf):
        q = _randn((1, 4, 3, 128), 61)
        q[0, 1, 1, 5] = broken
        clean = q.clone()
        clean[0, 1, 1] = 0
        pos = torch.tensor([50, 60, 99], device="cuda")
        got, want = T.kv4_attention(q, pos, cache).view(3, 4, 128), T.kv4_attention(clean, pos, cache).view(3, 4, 128)
        assert torch.isnan(got[1, 1]).all()
        got[1, 1], want[1, 1] = 0, 0
        assert torch.equal(got, want)


def test_attention_of_large_and_of_one_dominating_score():
    """Scores of thousands, all negative ones, and one key far above the others, first or last."""
    cache = T.Kv4Cache(*P.random_cache(1, 1, 300, 128, 70))
    q = _randn((1, 4, 1, 128), 71)
    pos = torch.tensor([299], device="cuda")
    for factor in (300.0, -300.0, 1e-20):
        _attend((q * factor).to(torch.bfloat16), pos, cache)
    for slot in (0, 150, 299):
        peaked = T.Kv4Cache(*(c.clone() for c in cache))
        peaked.k[0, 0, slot] = 0x66                                              # 4s under a large scale
        peaked.k_scale[0, 0, slot] = 132
        _attend(q.abs(), pos, peaked)


@pytest.mark.parametrize("t", [1, 9, 120])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_with_any_scale(t, d):
    cache = T.Kv4Cache(*P.random_cache(2, 2, 150, d, 72))
    q = _randn((2, 4, t, d), 73)
    pos = torch.arange(t, device="cuda") + 150 - t
    for scale in (0.0, -0.3, 1e-30, 4.0):
        _attend(q, pos, cache, scale)


@pytest.mark.parametrize("t", [1, 9, 120])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_over_scales_from_end_to_end(t, d):
    """Values whose scales reach over the whole range of the format, and one such slot among ordinary ones."""
    cache = T.Kv4Cache(*P.random_cache(1, 2, 300, d, 74))
    q = _randn((1, 4, t, d), 75)
    pos = torch.arange(t, device="cuda") + 300 - t
    for low, high in ((2, 253), (104, 141), (100, 108), (138, 144)):
        wide = T.Kv4Cache(*(c.clone() for c in cache))
        wide.v_scale.copy_(torch.randint(low, high, cache.v_scale.shape, generator=_gen(76), device="cuda", dtype=torch.uint8))
        _attend(q, pos, wide)
    for byte in (2, 103, 104, 140, 141, 250):
        one = T.Kv4Cache(*(c.clone() for c in cache))
        one.v_scale[0, 1, 77, 0] = byte
        _attend(q, pos, one)
    # groups of zeros, as the store leaves them: the smallest scale, codes 0 and -0; alone and with one of another value among them
    zeros = T.Kv4Cache(*(c.clone() for c in cache))
    for slot in (0, 5, 31, 150, 299):
        zeros.v[0, :, slot] = 0x80 if slot % 2 else 0x08
        zeros.v_scale[0, :, slot] = 2
    _attend(q, pos, zeros)
    zeros.v[0, 0, 150, 3] = 0x70
    _attend(q, pos, zeros)
    low = T.Kv4Cache(*(c.clone() for c in cache))
    low.k_scale.copy_(torch.randint(2, 128, cache.k_scale.shape, generator=_gen(77), device="cuda", dtype=torch.uint8))
    _attend(q, pos, low)


def test_caches_of_more_than_two_gigabytes():
    """Offsets beyond 2^31: the last sequence's rows."""
    b, kv, slots, d = 3, 8, 1 << 21, 128
    cache = T.Kv4Cache(*(torch.zeros((b, kv, slots, w), dtype=torch.uint8, device="cuda") for w in (64, 4, 64, 4)))
    x = _randn((b, 24 * d), 80)
    inv, _ = T.rotary_frequencies(d)
    pos = torch.tensor([[5], [slots - 40], [slots - 1]], device="cuda")
    assert cache.k.numel() > 1 << 31
    first = slots - 64
    small = P.random_cache(b, kv, 64, d, 81)
    for c, s in zip(cache, small):
        c[:, :, first:] = s
    q = T.kv4_store(x, pos, inv, cache, 8)
    k, v = T.kv4_rows(cache, pos)
    assert torch.equal(v.view(b, kv, d).double(), P.round_codes(x[:, 16 * d:].double().view(b, kv, d), P.scale_exponents(x[:, 16 * d:].double().view(b, kv, d).abs().unflatten(-1, (-1, 32)).amax(-1))))
    # keys of zero codes score 0: over n slots, of which the first n - 64 hold zero values
    got = T.kv4_attention(q, pos, cache).view(b, 8, d)
    end = int(pos[2])
    key, value = P.values(cache.k[2, :, first:], cache.k_scale[2, :, first:]), P.values(cache.v[2, :, first:], cache.v_scale[2, :, first:])
    score = (key * q[2].double()).sum(-1) * d ** -0.5                            # [8, 64]
    weight = score.exp()
    want = (weight[..., None] * value).sum(1) / (weight.sum(-1, keepdim=True) + first)
    ds = (d + 4) * P.HALF_FP32 * d ** -0.5 * float((key.abs() * q[2].double().abs()).sum(-1).max())
    tol = P.HALF_BF16 * want.abs() + (2 * ds + 2.0 ** -10 + 2.0 ** -15 + (end + 1) / 8192 * P.HALF_FP32) * (weight[..., None] * value.abs()).sum(1) / (weight.sum(-1, keepdim=True) + first) * 1.0
    # (2^-10: fp16 probabilities in the numerator, and in the sum that divides it: there relative to the result.  Equal terms: a wave adds the same number again
    # and again, whose sum over 2^21 slots in 32 bits is off by less than 2^-12.)
    assert P.same_or_near(got[2], want, tol + (2.0 ** -10 + 2.0 ** -12) * want.abs()) <= 0


@pytest.mark.parametrize("adjacent", [True, False])
@pytest.mark.parametrize("b,h,kv,d,r,slots,filled", [(1, 20, 5, 128, 128, 384, 253), (3, 20, 5, 128, 64, 40, 31), (1, 8, 8, 64, 64, 3000, 2999), (2, 34, 2, 128, 20, 700, 500), (4, 5, 1, 64, 50, 64, 0), (1, 4, 1, 128, 128, 20000, 19999)])
def test_step_is_store_and_attention(adjacent, b, h, kv, d, r, slots, filled):
    """Outputs and cache, bit for bit; also with a padded sequence and one behind the cache."""
    _say("step", adjacent, b, h, kv, d, r, slots, filled)
    inv, amplitude = T.rotary_frequencies(r, 500000.0, {"type": "yarn", "factor": 4, "original_max_position": 8192})
    one, two = (T.Kv4Cache(*P.random_cache(b, kv, slots, d, 90)) for _ in range(2))
    pos = (torch.full((b, 1), filled, device="cuda") - 3 * torch.arange(b, device="cuda")[:, None]).clamp(min=0)
    for change in range(3):
        if change == 1:
            pos[-1] = -1
        if change == 2:
            pos[-1] = slots
        x = _randn((b, (h + 2 * kv) * d), 91 + change)
        got = T.kv4_step(x, pos, inv, one, h, adjacent=adjacent, amplitude=amplitude)
        q = T.kv4_store(x, pos, inv, two, h, adjacent=adjacent, amplitude=amplitude)
        want = T.kv4_attention(q, pos, two)
        for x1, x2 in zip(one, two):
            assert torch.equal(x1, x2)
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        assert same.all()
        assert torch.isnan(got[-1]).all() == (change == 2) and (change != 1 or not got[-1].any())
    if b > 1:
        shared = torch.tensor([filled], device="cuda")
        x = _randn((b, (h + 2 * kv) * d), 99)
        assert torch.equal(T.kv4_step(x, shared, inv, one, h, adjacent=adjacent), T.kv4_step(x, shared.expand(b)[:, None].contiguous(), inv, two, h, adjacent=adjacent))


def test_step_of_rows_that_are_not_finite():
    """A key or value with NaN: its group for NaN from then on, other sequences as without."""
    inv, _ = T.rotary_frequencies(128)
    for at in (20 * 128 + 5, 25 * 128 + 40):
        cache, other = (T.Kv4Cache(*P.random_cache(2, 5, 100, 128, 100)) for _ in range(2))
        x = _randn((2, 30 * 128), 101)
        pos = torch.tensor([[40], [99]], device="cuda")
        want = T.kv4_step(x, pos, inv, other, 20)
        x[0, at] = math.nan
        got = T.kv4_step(x, pos, inv, cache, 20)
        assert torch.equal(got[1], want[1])
        # 4 query heads of the first kv head: everything under a broken key, the second 32 dimensions under a broken value
        head = torch.isnan(got[0].view(20, 128)[:4])
        assert head.all() if at < 25 * 128 else (head[:, 32:64].all() and not head[:, :32].any() and not head[:, 64:].any())
        assert torch.equal(got[0].view(20, 128)[4:], want[0].view(20, 128)[4:])


class _Kv4(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "k_scale", "v", "v_scale")]


def test_c_entry_point_without_a_workspace():
    """One part a row: within the tolerance of the split form."""
    lib = _lib.load()
    b, h, kv, d, slots = 1, 20, 5, 128, 2000
    cache = P.random_cache(b, kv, slots, d, 110)
    q, pos = _randn((b, h, 1, d), 111), torch.tensor([1990], device="cuda")
    out = torch.empty((b, h * d), dtype=torch.bfloat16, device="cuda")
    assert lib.ternaspmm_kv4_splits(b, 1, h, kv, d, slots) > 1
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.ternaspmm_kv4_attention(q.data_ptr(), ctypes.byref(_Kv4(*(c.data_ptr() for c in cache))), pos.data_ptr(), 0, out.data_ptr(), None, b, 1, h, kv, d, slots, d ** -0.5, stream) == 0
    want, tol = P.attention(q, pos, cache, d ** -0.5)
    assert P.same_or_near(out.view(b, 1, h, d), want, tol) <= 0


@pytest.mark.parametrize("t", [1, 48])
def test_the_longest_cache(t):
    """2^25 slots of two sequences: byte offsets beyond 2^32, requests beyond 2^31.  All slots are zeros but a few written ones, whose keys weigh against the
    zeros' 2^25 times exp(0)."""
    slots, h, d = 1 << 25, 4, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("9 GB of caches, with room to spare")
    _say("the longest cache", t)
    cache = T.Kv4Cache.empty(2, 1, slots, d)
    inv, _ = T.rotary_frequencies(d)
    written = torch.tensor([0, 5, 1 << 24, (1 << 24) + 77, slots - 100 - t, slots - 70 - t], device="cuda")
    last = torch.arange(slots - t, slots, device="cuda")
    unit = _randn((2, 1, d), 80) * 0.5
    rows = torch.cat([_randn((2, 6 + t, h * d), 81), (unit + 0.1 * _randn((2, 6 + t, d), 82)).to(torch.bfloat16), _randn((2, 6 + t, d), 83)], -1).to(torch.bfloat16)
    T.kv4_store(rows.view(-1, (h + 2) * d), torch.cat([written, last]), inv * 0, cache, h)
    if t == 1:                                                                   # the same bits, by the step's own launch
        again = T.kv4_step(rows[:, -1].contiguous(), last, inv * 0, cache, h)
    keys, values = (x[:, :, 0].double() for x in T.kv4_rows(cache, torch.cat([written, last])))
    assert (keys != 0).any(-1).all() and torch.isfinite(keys).all()
    one_row = T.kv4_rows(cache, torch.tensor([6, slots - 60 - t], device="cuda"))
    assert not one_row[0].any() and not one_row[1].any()                         # nothing went elsewhere nearby
    q = (unit[:, None, :, :].expand(2, h, t, d) * 6 + _randn((2, h, t, d), 84)).to(torch.bfloat16)
    scale = d ** -0.5
    got = T.kv4_attention(q, last, cache, scale).view(2, t, h, d).double()
    score = scale * q.double() @ keys.transpose(1, 2)[:, None]                   # [2, H, T, 6 + t]
    seen = torch.arange(6 + t, device="cuda")[None] < 7 + torch.arange(t, device="cuda")[:, None]
    weight = torch.where(seen, score.exp(), torch.zeros_like(score))
    mass = (last + 1 - 7 - torch.arange(t, device="cuda")).double()[None, None, :, None] + weight.sum(-1, keepdim=True)
    want = (weight @ values[:, None] / mass).transpose(1, 2)
    # A wave or half row adds at most 2^25 / 128 slots one after the other (2^18 half steps of an fp32, in truth far fewer), several at a time: 2^-6 of the sum and
    # of the numerators at most; fp16 probabilities 2^-11, scores of magnitude below 40 off by (128 + 4) 2^-24 40 < 2^-11.
    tol = (2 * 2.0 ** -6) * (weight @ values.abs()[:, None] / mass).transpose(1, 2) + P.HALF_BF16 * want.abs() + 2.0 ** -40
    assert P.same_or_near(got, want, tol) <= 0
    assert want.abs().max() > 1e-3                                               # (the written slots weigh something)
    if t == 1:
        own = T.kv4_attention(rows[:, -1, :h * d].reshape(2, h, 1, d).contiguous(), last, cache)
        assert torch.equal(again, own)


# ---- log probabilities ---------------------------------------------------------------------------------------------------------------


def _check_logprobs(logits, targets, top):
    got = T.token_logprobs(logits, targets, top)
    x = logits.double()
    m, v = x.shape
    peak = x.amax(-1, keepdim=True)
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    terms = torch.where(p == 0, torch.zeros_like(p), p * logp)
    entropy = -terms.sum(-1)
    # e = exp2((x - m) log2 e): relative error (|x - m| + 4) 2^-23 (difference, product, the exponential's); a sum of V / 256 and more terms in fp32 by one
    # thread and then a tree; log, and the last differences.
    far = torch.where(p > 0, (peak - x), torch.zeros_like(x)).amax(-1).clamp(max=110.0)
    relative = (far + 8) * 2.0 ** -23 + (v / 256 + 64) * P.HALF_FP32
    spread = (p * torch.where(p > 0, (logp - logp.amax(-1, keepdim=True)).abs(), torch.zeros_like(p))).sum(-1)
    tol_entropy = relative * (1 + 2 * spread) + 2.0 ** -22 * (spread + math.log(v) + 1)
    assert got.entropy.dtype == torch.float32 and P.same_or_near(got.entropy, entropy, tol_entropy) <= 0
    size = lambda lp: relative.view(-1, *[1] * (lp.dim() - 1)) + 2.0 ** -22 * (lp.abs().clamp(max=1e30) + math.log(v) + 1)
    if targets is not None:
        inside = (targets >= 0) & (targets < v)
        want = torch.where(inside, logp.gather(1, targets.clamp(0, v - 1)[:, None])[:, 0], torch.tensor(math.nan, dtype=torch.float64, device="cuda"))
        assert P.same_or_near(got.logprob, want, size(want)) <= 0
    else:
        assert got.logprob is None
    if top == 0:
        assert got.top_ids is None and got.top_logprobs is None
        return got
    order = torch.where(torch.isnan(logits.float()), -math.inf, logits.float())
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices
    if torch.isnan(logits).any():                                                # numbers first, -inf among them
        nan = torch.isnan(logits)
        ids = torch.stack([torch.cat([row[~gone[row]], torch.nonzero(gone)[:, 0]]) for row, gone in zip(ids, nan)])
    assert torch.equal(got.top_ids, ids[:, :top])
    want = logp.gather(1, ids[:, :top])
    assert P.same_or_near(got.top_logprobs, want, size(want)) <= 0
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,v,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (5, 7, 5), (2, 64, 64), (4, 100, 64), (1, 2047, 1), (7, 2048, 3), (2, 2049, 33), (1, 32000, 5), (600, 4096, 20), (3, 50021, 64),
                                     (1, 128256, 5), (40, 128256, 20), (2, 128256, 0), (3, 300001, 64),
                                     (700, 140007, 3), (1, 1 << 19, 64)])
def test_logprobs(dtype, m, v, top):
    _say("logprobs", dtype, m, v, top)
    logits = (_randn((m, v), 200 + v, torch.float32) * 3).to(dtype)
    targets = torch.randint(0, v, (m,), generator=_gen(201), device="cuda")
    targets[0] = v - 1
    _check_logprobs(logits, targets, top)
    _check_logprobs(logits, None, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v,ld,cut", [(4999, 4999, 0), (4999, 5003, 1), (5000, 5001, 7), (129, 131, 3), (3, 5, 2), (128256, 128259, 5)])
def test_logprobs_of_rows_at_any_element(dtype, v, ld, cut):
    wide = (_randn((9, ld + cut), 210, torch.float32) * 2).to(dtype)
    wide[:, :cut] = math.inf                                                     # what lies around a row does not count
    wide[:, cut + v:] = math.nan
    logits = wide[:, cut:cut + v]
    targets = torch.tensor([0, v - 1, -1, v, 1, 1 << 40, -(1 << 40), 0, 2], device="cuda")
    _check_logprobs(logits, targets, min(v, 20))
    _check_logprobs(logits.t().contiguous().t(), targets, min(v, 20))
    same = logits[:1].expand(9, v)
    _check_logprobs(same, targets, min(v, 20))


def test_logprobs_where_values_tie_and_where_they_are_not_finite():
    v = 128256
    gen = _gen(220)
    base = (_randn((13, v), 221, torch.float32) * 2).to(torch.bfloat16)
    base[0] = 1.5                                                                # all the same
    base[1] = -math.inf
    base[1, [77, 128000, 5, 6000]] = torch.tensor([1.0, 2.0, 1.0, -3.0], device="cuda").to(torch.bfloat16)      # four tokens allowed
    base[2] = -math.inf                                                          # none
    base[3, 1000] = math.nan
    base[4, [3, 99]] = math.inf
    base[5] = math.nan
    base[6] = torch.arange(v, device="cuda").to(torch.bfloat16)                  # rising, in runs of equal values
    base[7] = -torch.arange(v, device="cuda").to(torch.bfloat16)
    base[8] = torch.where(torch.arange(v, device="cuda") % 2048 < 512, 20.0, -20.0).to(torch.bfloat16)          # all that is large with a quarter of the threads
    base[8] += torch.randn(v, generator=gen, device="cuda").to(torch.bfloat16)
    base[9] = 0.0
    base[9, ::2] = -0.0
    base[10, :] = math.nan
    base[10, [4, 9000, 128255]] = torch.tensor([1.0, -math.inf, 7.0], device="cuda").to(torch.bfloat16)
    base[11, :127000] = -math.inf
    base[12, 3] = 3e38
    base[12, 4] = -3e38
    targets = torch.randint(0, v, (13,), generator=gen, device="cuda")
    targets[1] = 128000
    base9 = base.clone()
    base9[9] = 0.0                                                               # (the oracle's sort: zeros of both signs are equal, the lower index first)
    for rows in (slice(0, 9), slice(10, 13)):
        for top in (1, 20, 64):
            _check_logprobs(base[rows], targets[rows], top)
            _check_logprobs(base[rows].float(), targets[rows], top)
    got = T.token_logprobs(base[9:10], None, 20)
    assert got.top_ids.tolist() == T.token_logprobs(base9[9:10], None, 20).top_ids.tolist() == [list(range(20))]


def test_logprobs_many_rows_do_not_depend_on_the_split():
    """A row alone (split over workgroups) and among many (one workgroup each): same ids, probabilities within two roundings of each sum."""
    logits = (_randn((700, 20000), 230, torch.float32) * 3).to(torch.bfloat16)
    many = T.token_logprobs(logits, logits.argmax(-1), 10)
    for i in (0, 699):
        one = T.token_logprobs(logits[i:i + 1], logits.argmax(-1)[i:i + 1], 10)
        assert torch.equal(one.top_ids[0], many.top_ids[i])
        assert (one.top_logprobs[0] - many.top_logprobs[i]).abs().max() <= 2 * (20000 / 256 + 64) * P.HALF_FP32 + 2.0 ** -20
    again = T.token_logprobs(logits, logits.argmax(-1), 10)
    assert all(torch.equal(a, b) for a, b in zip(many, again))


def test_logprobs_refusals_and_no_rows():
    x = _randn((4, 10), 240)
    targets = torch.zeros(4, dtype=torch.int64, device="cuda")
    assert T.token_logprobs(x[:0], targets[:0], 3).top_ids.shape == (0, 3)
    for call in (lambda: T.token_logprobs(x[0], None), lambda: T.token_logprobs(x.half()), lambda: T.token_logprobs(x[:, :0]), lambda: T.token_logprobs(x, targets[:3]),
                 lambda: T.token_logprobs(x, targets.int()), lambda: T.token_logprobs(x, targets.cpu()), lambda: T.token_logprobs(x, None, 11), lambda: T.token_logprobs(x, None, -1),
                 lambda: T.token_logprobs(_randn((1, 100), 1), None, 65)):
        with pytest.raises(ValueError, match="token_logprobs"):
            call()


# ---- a run of them -------------------------------------------------------------------------------------------------------------------


def test_a_request_from_positions_to_scores_eager_and_captured():
    """A prompt stored and attended, then steps and their scores: eager, and as a graph replayed with eager work between, on a stream of its own."""
    b, h, kv, d, slots, vocab = 2, 20, 5, 128, 1200, 32000
    inv, amplitude = T.rotary_frequencies(d, 500000.0, {"type": "linear", "factor": 4.0})
    prompt = torch.tensor([700, 650], device="cuda")
    head = _randn((h * d, vocab), 300) * 0.05
    eager, graphed = T.Kv4Cache.empty(b, kv, slots, d), T.Kv4Cache.empty(b, kv, slots, d)
    x0 = _randn((b * 700, (h + 2 * kv) * d), 301)
    at = torch.arange(700, device="cuda").expand(b, 700)
    at = torch.where(at < prompt[:, None], at, -1)
    outs = []
    for cache in (eager, graphed):
        q = T.kv4_store(x0, at, inv, cache, h, amplitude=amplitude)
        outs.append(T.kv4_attention(q, at, cache))
    assert torch.equal(outs[0], outs[1]) and not outs[0].view(b, 700, -1)[1, 650:].any()
    assert not eager.v_scale[1, :, 650:].any()

    def step(x, pos, cache):
        o = T.kv4_step(x, pos, inv, cache, h, amplitude=amplitude)
        turned = T.rotary_embed(o.view(b, 1, h, d), pos, inv)
        logits = torch.matmul(turned.view(b, h * d), head)
        return (o, *T.token_logprobs(logits, pos[:, 0], 5))

    steps = [_randn((b, (h + 2 * kv) * d), 310 + i) for i in range(6)]
    x, pos = steps[0].clone(), prompt[:, None].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        spare = T.Kv4Cache(*(c.clone() for c in graphed))
        step(x, pos, spare)                                                      # loads what a first call loads
        with torch.cuda.graph(graph, stream=side):
            captured = step(x, pos, graphed)
    torch.cuda.current_stream().wait_stream(side)
    for i, rows in enumerate(steps):
        want = step(rows, prompt[:, None] + i, eager)
        torch.cuda.synchronize()
        x.copy_(rows)
        pos.copy_(prompt[:, None] + i)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(captured, want):
            assert torch.equal(got, w), i
        for one, two in zip(eager, graphed):
            assert torch.equal(one, two)


def test_calls_at_once_and_two_graphs():
    """The same operators on two streams at the same time, eager and as two captured graphs replayed together: split launches keep to scratch of their own."""
    h, kv, d, slots = 20, 5, 128, 4000
    caches = [T.Kv4Cache(*P.random_cache(2, kv, slots, d, 320 + i)) for i in range(2)]
    logits = [_randn((3, 60000), 330 + i, torch.float32) for i in range(2)]
    q = [_randn((2, h, 1, d), 340 + i) for i in range(2)]
    many = [_randn((2, h, 60, d), 350 + i) for i in range(2)]
    last, inv = torch.tensor([slots - 1], device="cuda"), T.rotary_frequencies(d)[0]
    span = torch.arange(slots - 60, slots, device="cuda")

    def work(i):
        return [T.kv4_attention(q[i], last, caches[i]), *T.token_logprobs(logits[i], last.expand(3), 20), T.kv4_attention(many[i], span, caches[i]),
                T.rotary_embed(many[i], span[:h].repeat(2, 1), inv)]

    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = [None, None]
        for i, stream in enumerate(streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got[i] = work(i)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, stream=streams[i]):
            got[i] = work(i)
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay()
        eager = work(0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))


@pytest.mark.parametrize("b,h,kv,d", [(300, 8, 8, 64), (257, 5, 1, 128), (1, 64, 2, 128), (2, 33, 1, 64)])
def test_steps_of_many_sequences_and_of_many_heads(b, h, kv, d):
    """More workgroups than CUs; more query heads than a tile has rows."""
    _say("step", b, h, kv, d)
    slots = 50
    cache = T.Kv4Cache(*P.random_cache(b, kv, slots, d, 360))
    twin = T.Kv4Cache(*(c.clone() for c in cache))
    pos = torch.randint(-1, slots + 1, (b, 1), generator=_gen(361), device="cuda")
    inv, _ = T.rotary_frequencies(d)
    x = _randn((b, (h + 2 * kv) * d), 362)
    got = T.kv4_step(x, pos, inv, cache, h)
    q = T.kv4_store(x, pos, inv, twin, h)
    assert all(torch.equal(one, two) for one, two in zip(cache, twin))
    assert torch.equal(got.isnan(), T.kv4_attention(q, pos, twin).isnan())
    _attend(q, pos, twin)
    want, tol = P.attention(q, pos, twin, d ** -0.5)
    assert P.same_or_near(got.view(b, 1, h, d), want, tol) <= 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t,h,kv", [(1, 8, 1), (3, 5, 1), (4, 20, 5), (40, 8, 2), (120, 4, 1), (200, 8, 2)])
def test_a_row_does_not_depend_on_the_rows_beside_it(t, h, kv, d):
    """Bit for bit: other queries, and other keys and values in slots that it does not see (with scales that fp16 has room for), in both layouts."""
    _say("rows beside", t, h, kv, d)
    slots = 900
    cache = T.Kv4Cache(*P.random_cache(1, kv, slots, d, 390))
    pos = 600 + torch.arange(t, device="cuda")
    q = _randn((1, h, t, d), 391)
    want = T.kv4_attention(q, pos, cache).view(t, h, d)
    for seed, factor in ((392, 1.0), (393, 30.0), (394, 300.0)):
        other = (_randn(q.shape, seed) * factor).to(torch.bfloat16)
        even = torch.arange(h, device="cuda") % 2 == 0
        mixed = torch.where(even[None, :, None, None], q, other)
        assert torch.equal(T.kv4_attention(mixed, pos, cache).view(t, h, d)[:, even], want[:, even])
        if t > 1:
            first = t // 2
            mixed = torch.cat([q[:, :, :first], other[:, :, first:]], 2)
            later = T.Kv4Cache(*(c.clone() for c in cache))
            for c, fresh in zip(later, P.random_cache(1, kv, slots, d, seed)):
                c[:, :, 600 + first:] = fresh[:, :, 600 + first:]
            later.k_scale[:, :, 600 + first::7] = 135
            assert torch.equal(T.kv4_attention(mixed, pos, later).view(t, h, d)[:first], want[:first])


@pytest.mark.parametrize("b,h,kv,d,slots", [(2, 300, 1, 128, 20000), (3, 23, 1, 128, 700), (2, 40, 2, 64, 2000)])
def test_step_is_store_and_attention_where_a_tile_has_few_rows(b, h, kv, d, slots):
    """The last tile of a kv head's query heads: what fills up its sixteen rows does not count."""
    _say("step", b, h, kv, d, slots)
    cache = T.Kv4Cache(*P.random_cache(b, kv, slots, d, 395))
    pos = torch.randint(slots // 2, slots, (b, 1), generator=_gen(396), device="cuda")
    inv, _ = T.rotary_frequencies(d)
    x = _randn((b, (h + 2 * kv) * d), 397) * 3
    got = T.kv4_step(x, pos, inv, cache, h)
    assert torch.equal(got, T.kv4_attention(T.kv4_store(x, pos, inv, cache, h), pos, cache))


# Query heads of one kv head enough for the layout of many rows, in one part and in several, with parts whose rows are an odd number.
MANY_HEADS = [(128, 128, 1, 128, 40), (256, 64, 1, 128, 128), (96, 48, 1, 128, 6000), (48, 96, 2, 128, 5600), (8, 71, 1, 64, 32768), (1, 568, 8, 64, 32768), (4, 128, 1, 64, 32768),
              (2, 300, 1, 128, 20000)]


@pytest.mark.parametrize("b,h,kv,d,slots", MANY_HEADS)
def test_steps_of_many_query_heads_a_kv_head(b, h, kv, d, slots):
    """Every head against 64 bits; outputs and cache are those of kv4_store and kv4_attention, bit for bit."""
    _say("step of many heads", b, h, kv, d, slots)
    cache = T.Kv4Cache(*P.random_cache(b, kv, slots, d, 370))
    twin = T.Kv4Cache(*(c.clone() for c in cache))
    pos = torch.randint(slots // 2, slots, (b, 1), generator=_gen(371), device="cuda")
    if b > 2:
        pos[0], pos[1] = -1, slots
    inv, _ = T.rotary_frequencies(d)
    x = _randn((b, (h + 2 * kv) * d), 372)
    got = T.kv4_step(x, pos, inv, cache, h, adjacent=False)
    q = T.kv4_store(x, pos, inv, twin, h, adjacent=False)
    want = _attend(q, pos, twin)
    assert all(torch.equal(one, two) for one, two in zip(cache, twin))
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("b,h,kv,d,slots", [(96, 48, 1, 128, 6000), (8, 71, 1, 64, 32768)])
def test_a_captured_step_of_many_query_heads(b, h, kv, d, slots):
    """Replayed with eager work between, and without a workspace."""
    _say("captured step of many heads", b, h, kv, d, slots)
    cache = T.Kv4Cache(*P.random_cache(b, kv, slots, d, 380))
    twin = T.Kv4Cache(*(c.clone() for c in cache))
    pos = torch.randint(slots // 2, slots - 8, (b, 1), generator=_gen(381), device="cuda")
    now, inv = pos.clone(), T.rotary_frequencies(d)[0]
    steps = [_randn((b, (h + 2 * kv) * d), 382 + i) for i in range(4)]
    x = steps[0].clone()
    T.kv4_step(x, now, inv, T.Kv4Cache(*(c.clone() for c in cache)), h)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = T.kv4_step(x, now, inv, cache, h)
    for i, rows in enumerate(steps):
        x.copy_(rows)
        now.copy_(pos + i)
        want = T.kv4_step(rows, pos + i, inv, twin, h)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want) and all(torch.equal(one, two) for one, two in zip(cache, twin)), i
    lib = _lib.load()
    out = torch.empty((b, h * d), dtype=torch.bfloat16, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    c = ctypes.byref(_Kv4(*(t.data_ptr() for t in cache)))
    assert lib.ternaspmm_kv4_step(x.data_ptr(), x.shape[1], now.data_ptr(), 1, inv.data_ptr(), inv.numel(), 1.0, c, out.data_ptr(), None, b, h, kv, d, slots, d ** -0.5, 1, stream) == 0
    q = T.kv4_store(x, now, inv, twin, h)
    want, tol = P.attention(q, now, twin, d ** -0.5)
    assert P.same_or_near(out.view(b, 1, h, d), want, tol) <= 0


# ---- the most that a launch has room for ---------------------------------------------------------------------------------------------


def test_the_most_rows_of_log_probabilities():
    m = (1 << 24) - 1
    _say("log probabilities of", m)
    logits = _randn((m, 2), 400)
    got = T.token_logprobs(logits, torch.ones(m, dtype=torch.int64, device="cuda"), 1)
    a, b = logits.double().unbind(-1)
    peak, gap = torch.maximum(a, b), (a - b).abs()
    lse = torch.log1p((-gap).exp())
    # differences below 16 in fp32, an exponential and a logarithm: the same bound as for few logits above
    for value, want in ((got.logprob, b - peak - lse), (got.top_logprobs[:, 0], -lse), (got.entropy, lse + gap * (-gap).exp() / (1 + (-gap).exp()))):
        assert ((value.double() - want).abs() <= 40 * 2.0 ** -23 * (1 + want.abs())).all()
    assert torch.equal(got.top_ids[:, 0], (b > a).long())
    with pytest.raises(ValueError, match="token_logprobs"):
        T.token_logprobs(logits[:1].expand(m + 1, 2))


def test_the_most_tokens_of_rotary_positions():
    b = 1 << 23
    _say("rotary of", 3 * b)
    x, pos = _randn((b, 3, 1, 2), 401), torch.tensor([5, 70000, -3], device="cuda")
    inv = torch.tensor([0.37], dtype=torch.float64, device="cuda")
    _check_rotary(x, T.rotary_embed(x, pos, inv), pos, inv, 1.0, True)
    with pytest.raises(ValueError, match="rotary_embed"):
        T.rotary_embed(x[:1].expand(1 << 25, 3, 1, 2), pos, inv)


def test_the_most_sequences_of_the_cache():
    """One slot each: attention's result is its value, exactly."""
    b, d = (1 << 24) - 8, 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("20 GB of queries and rows")
    _say("attention of", b)
    cache = T.Kv4Cache(*P.random_cache(b, 1, 1, d, 402))
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    rows = T.kv4_rows(cache, pos)[1].view(b, d)
    assert torch.equal(rows[-1000:].double(), P.values(cache.v, cache.v_scale)[-1000:].view(1000, d))
    q = _randn((1, 1, 1, d), 403).expand(b, 1, 1, d)
    assert torch.equal(T.kv4_attention(q, pos, cache), rows)
    more = T.Kv4Cache.empty(1 << 24, 1, 1, d)
    with pytest.raises(ValueError, match="kv4_attention"):
        T.kv4_attention(q[:1].expand(1 << 24, 1, 1, d), pos, more)
