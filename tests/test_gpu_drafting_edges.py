"""Calls of ternainfer_amd/drafting.py, int8_linear.py and of the model's steps over trees at the edges of what their documentation allows."""
import pytest
import torch

import ternainfer_amd as T
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
