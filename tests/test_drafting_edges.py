"""What ternainfer_amd/drafting.py, int8_linear.py and the model's drafts do at the edges of their documentation, where no GPU is needed."""
import types

import pytest
import torch

import ternainfer_amd as T
from ternainfer_amd import _lib
from ternainfer_amd.model import ngram_drafts, speculative_decode
from tests import _drafting as P


def test_scales_are_looked_at_before_rows_are_packed(monkeypatch):
    """TypeError where an argument is no tensor, ValueError for scales that do not belong to the rows; nothing is enqueued by then."""
    def enqueued(*_):
        raise AssertionError("enqueued")

    monkeypatch.setattr(_lib, "native", lambda: type("Native", (), {"int8_pack": staticmethod(enqueued)}))
    rows, scale = torch.zeros((2, 3), dtype=torch.int8), torch.zeros(2)
    for q, s in ((rows, [0.0, 0.0]), (rows, None), ([[1]], scale), (rows, 1.0)):
        with pytest.raises(TypeError, match="int8_rows"):
            T.int8_rows(q, s)
    for s in (scale.double(), torch.zeros(3), torch.zeros((2, 1)), torch.zeros(2, device="meta")):
        with pytest.raises(ValueError, match="int8_rows"):
            T.int8_rows(rows, s)


def test_decoding_goes_by_the_prompts_device(monkeypatch):
    """A prompt on another device than the current one: that device is the current one meanwhile (a step captured elsewhere would be empty, and its replays would never end)."""
    current, entered = [0], []

    class On:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            entered.append(self.index)
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[-1])
    monkeypatch.setattr(torch.cuda, "device", On)
    prompt = types.SimpleNamespace(shape=(1, 4), device=torch.device("cuda", 1), is_cuda=True, dtype=torch.int32)
    with pytest.raises(ValueError, match="speculative_decode"):                          # (refused there: int32)
        speculative_decode(None, prompt, 5)
    assert entered == [1] and current == [0]


def _branches(text, branches, depth):
    """What followed the last two tokens of a text (a list) at the latest places where they stood before."""
    places = [i for i in range(len(text) - 2, 0, -1) if text[i - 1:i + 1] == text[-2:]][:branches]
    return [text[i + 1:i + 1 + depth] for i in places]


@pytest.mark.parametrize("branches,depth", [(1, 1), (2, 4), (3, 7), (5, 2), (0, 3), (3, 0)])
@pytest.mark.parametrize("kinds", [1, 2, 5, 40])
def test_drafts_that_begin_alike_share_their_nodes(branches, depth, kinds):
    """The lines of the tree are the beginnings of the branches, each of them once, so that none hides what continues another."""
    gen = torch.Generator().manual_seed(10 * branches + kinds)
    text = torch.randint(0, kinds, (60, 30), generator=gen)
    text[40:] = torch.randint(0, kinds, (20, 4), generator=gen).repeat(1, 8)[:, :30]     # periodic ones
    length = torch.randint(1, 31, (60,), generator=gen)
    tokens, parents = ngram_drafts(text, length, branches, depth)
    assert tokens.shape == parents.shape == (60, 1 + branches * depth) and tokens.dtype == parents.dtype == torch.int64 and tokens.min() >= 0
    for row, n, says, of in zip(text.tolist(), length.tolist(), tokens.tolist(), parents.tolist()):
        assert says[0] == row[n - 1] and of[0] == -1
        got = sorted([says[i] for i in line[1:]] for line in P.lines(of) if line)
        want = {tuple(b[:j]) for b in _branches(row[:n], branches, depth) for j in range(len(b) + 1)} | {()}
        assert got == sorted(map(list, want))


def test_drafts_of_periodic_texts_are_accepted():
    """A model that goes on with the period accepts two drafts of 20 equal tokens (the places end with the text) and four of a period of two."""
    for text, steps in (([7] * 20, 2), ([1, 2] * 10, 4)):
        tokens, parents = ngram_drafts(torch.tensor([text]), torch.tensor([20]))
        follows = torch.nn.functional.one_hot(torch.tensor([[{7: 7, 1: 2, 2: 1, 0: 0}[t] for t in tokens[0].tolist()]]), 8)
        _, count, behind = P.accept(follows, tokens, parents)
        assert count == [1 + steps] and behind == [(text + text)[20 + steps]]
