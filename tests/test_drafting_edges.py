"""What ternainfer_amd/drafting.py, int8_linear.py and the model's drafts do at the edges of their documentation, where no GPU is needed."""
import types

import pytest
import torch

import ternainfer_amd as T
from ternainfer_amd import _lib
from ternainfer_amd.model import speculative_decode


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
