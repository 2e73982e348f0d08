"""ternainfer_amd/long_context.py where no GPU is needed: frequencies, sizes, and what is refused before anything is enqueued."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import ternainfer_amd as T
from ternainfer_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _inv(dim, theta):
    return [theta ** (-2 * j / dim) for j in range(dim // 2)]


def test_plain_and_linear_frequencies():
    inv, amplitude = T.rotary_frequencies(128, 500000.0, device="cpu")
    assert inv.dtype == torch.float64 and inv.tolist() == _inv(128, 500000.0) and amplitude == 1.0
    half, amplitude = T.rotary_frequencies(128, 500000.0, {"type": "linear", "factor": 4}, device="cpu")
    assert torch.equal(half, inv / 4) and amplitude == 1.0


def test_ntk_keeps_the_fastest_pair_and_divides_the_slowest():
    inv, _ = T.rotary_frequencies(64, 10000.0, device="cpu")
    got, _ = T.rotary_frequencies(64, 10000.0, {"type": "ntk", "factor": 8.0}, device="cpu")
    assert got[0] == inv[0] and math.isclose(got[-1], inv[-1] / 8, rel_tol=1e-12)
    assert T.rotary_frequencies(2, 10000.0, {"type": "ntk", "factor": 8.0}, device="cpu")[0].tolist() == [1.0]


def test_wavelength_scaling_by_turns_within_the_original_length():
    inv = _inv(128, 500000.0)
    got, amplitude = T.rotary_frequencies(128, 500000.0, {"type": "wavelength", "factor": 8.0, "original_max_position": 8192}, device="cpu")
    assert amplitude == 1.0
    kinds = set()
    for f, y in zip(inv, got.tolist()):
        turns = 8192 * f / (2 * math.pi)
        if turns < 1:
            want, kind = f / 8, "divided"
        elif turns > 4:
            want, kind = f, "kept"
        else:
            smooth = (turns - 1) / 3
            want, kind = (1 - smooth) * f / 8 + smooth * f, "between"
        kinds.add(kind)
        assert math.isclose(y, want, rel_tol=1e-12)
    assert kinds == {"divided", "kept", "between"}


def test_yarn_ramp_and_amplitude():
    dim, theta, factor, length = 128, 10000.0, 16.0, 4096
    got, amplitude = T.rotary_frequencies(dim, theta, {"type": "yarn", "factor": factor, "original_max_position": length}, device="cpu")
    assert math.isclose(amplitude, 0.1 * math.log(16) + 1)
    turns_at = lambda turns: dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))
    low, high = math.floor(turns_at(32)), math.ceil(turns_at(1))
    assert 0 < low < high < dim // 2
    for j, (f, y) in enumerate(zip(_inv(dim, theta), got.tolist())):
        ramp = min(1, max(0, (j - low) / (high - low)))
        assert math.isclose(y, f * (1 - ramp) + f / factor * ramp, rel_tol=1e-12)
    assert T.rotary_frequencies(dim, theta, {"type": "yarn", "factor": 4, "original_max_position": 64, "amplitude": 1.5}, device="cpu")[1] == 1.5


@pytest.mark.parametrize("scaling", [{"type": "other", "factor": 2}, {"factor": 2}, {"type": "linear"}, {"type": "linear", "factor": 0.5}, {"type": "linear", "factor": float("nan")},
                                     {"type": "linear", "factor": 2, "beta_fast": 3}, {"type": "yarn", "factor": 2},
                                     {"type": "yarn", "factor": 2, "original_max_position": 64, "beta_fast": 1, "beta_slow": 1},
                                     {"type": "wavelength", "factor": 2, "original_max_position": 0},
                                     {"type": "wavelength", "factor": 2, "original_max_position": 64, "low_freq_factor": 4}])
def test_unknown_scalings_are_refused(scaling):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        T.rotary_frequencies(64, 10000.0, scaling, device="cpu")


@pytest.mark.parametrize("dim,theta", [(0, 1e4), (3, 1e4), (64, 0.0)])
def test_frequencies_refuse_odd_dimensions(dim, theta):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        T.rotary_frequencies(dim, theta, device="cpu")


def test_cache_has_heads_of_64_or_128():
    cache = T.Kv4Cache.empty(2, 3, 10, 128, device="cpu")
    assert [tuple(t.shape) for t in cache] == [(2, 3, 10, 64), (2, 3, 10, 4)] * 2
    with pytest.raises(ValueError, match="Kv4Cache"):
        T.Kv4Cache.empty(2, 3, 10, 96, device="cpu")


def test_splits_and_workspaces():
    lib = _lib.load()
    assert lib.ternaspmm_kv4_splits(1, 1, 20, 5, 96, 100) == -1 and lib.ternaspmm_kv4_splits(1, 1, 20, 3, 128, 100) == -1
    assert lib.ternaspmm_kv4_splits(0, 1, 20, 5, 128, 100) == -1 and lib.ternaspmm_kv4_splits(1, 1, 20, 5, 128, (1 << 25) + 1) == -1
    for shape in ((1, 1, 20, 5, 128, 1), (1, 1, 20, 5, 128, 384), (64, 1, 20, 5, 128, 1000), (1, 1, 20, 5, 128, 1 << 20), (3, 500, 20, 5, 128, 9000)):
        splits = lib.ternaspmm_kv4_splits(*shape)
        b, t, h, _, d, s = shape
        assert 1 <= splits <= 128 and (splits - 1) * 32 < s
        assert lib.ternaspmm_kv4_workspace_bytes(*shape) == (0 if splits == 1 else 4 * b * t * h * splits * (d + 2))
    logprobs = lib.ternaspmm_token_logprobs_workspace_bytes
    assert logprobs(0, 10, 0, 0) == -1 and logprobs(1, 10, 0, 11) == -1 and logprobs(1, 100, 0, 65) == -1 and logprobs(1, (1 << 19) + 1, 0, 0) == -1
    assert logprobs(2048, 128256, 0, 20) == 0 and logprobs(1, 128256, 0, 5) > 0 and logprobs(2048, 1 << 19, 0, 20) == 0 and logprobs(20, 200000, 1, 0) > 0


class _Kv4(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "k_scale", "v", "v_scale")]


def test_c_entry_points_refuse_before_they_enqueue():
    """Missing and misaligned pointers and unsupported sizes: -1 without a launch, so this runs without a GPU."""
    lib = _lib.load()
    p = lambda address: ctypes.c_void_p(address)
    strides = (ctypes.c_longlong * 3)(128, 128, 128)
    other = (ctypes.c_longlong * 3)(256, 128, 128)
    cache = _Kv4(64, 64, 64, 64)

    def refused(call, names, good, wrongs):
        for wrong in wrongs:
            arguments = {**good, **wrong}
            assert getattr(lib, call)(*(arguments[n] for n in names)) == -1, (call, wrong)

    names = "x xs out os fp32 pos each f pairs amp B T H D adj stream".split()
    good = dict(x=p(64), xs=strides, out=p(128), os=strides, fp32=0, pos=p(64), each=0, f=p(64), pairs=64, amp=1.0, B=1, T=1, H=1, D=128, adj=1, stream=None)
    refused("ternaspmm_rotary", names, good, [*({n: None} for n in ("x", "xs", "out", "os", "pos", "f")), dict(pairs=0), dict(pairs=65), dict(D=1026), dict(B=0), dict(T=0),
                                              dict(H=0), dict(H=65536), dict(B=1 << 16, T=1 << 15), dict(x=p(64), out=p(64), os=other)])
    names = "qkv row pos each f pairs amp q cache B T H KV D S adj stream".split()
    good = dict(qkv=p(64), row=384, pos=p(64), each=0, f=p(64), pairs=64, amp=1.0, q=p(64), cache=ctypes.byref(cache), B=1, T=1, H=1, KV=1, D=128, S=10, adj=1, stream=None)
    bad_cache = [dict(cache=ctypes.byref(_Kv4(*(None if i == j else 64 for i in range(4))))) for j in range(4)] + [dict(cache=ctypes.byref(_Kv4(72, 64, 64, 64)))]
    shapes = [dict(B=0), dict(H=0), dict(KV=0), dict(H=3, KV=2, row=900), dict(D=96), dict(S=0), dict(S=(1 << 25) + 1), dict(cache=None)]
    refused("ternaspmm_kv4_store", names, good, [*({n: None} for n in ("qkv", "pos", "f", "q")), *bad_cache, *shapes, dict(T=0), dict(row=376), dict(row=388), dict(pairs=0), dict(pairs=65),
                                                 dict(qkv=p(72)), dict(q=p(72))])
    names = "qkv row pos each f pairs amp cache out work B H KV D S scale adj stream".split()
    good = dict(qkv=p(64), row=384, pos=p(64), each=0, f=p(64), pairs=64, amp=1.0, cache=ctypes.byref(cache), out=p(64), work=None, B=1, H=1, KV=1, D=128, S=10, scale=1.0, adj=1, stream=None)
    refused("ternaspmm_kv4_step", names, good, [*({n: None} for n in ("qkv", "pos", "f", "out")), *bad_cache, *shapes, dict(row=376), dict(row=388), dict(pairs=65), dict(out=p(72)),
                                                dict(work=p(72))])
    names = "q cache pos each out work B T H KV D S scale stream".split()
    good = dict(q=p(64), cache=ctypes.byref(cache), pos=p(64), each=0, out=p(64), work=None, B=1, T=1, H=1, KV=1, D=128, S=10, scale=1.0, stream=None)
    refused("ternaspmm_kv4_attention", names, good, [*({n: None} for n in ("q", "pos", "out")), *bad_cache, *shapes, dict(T=0), dict(q=p(72)), dict(out=p(72)), dict(work=p(72))])
    names = "cache pos each k v B T KV D S stream".split()
    good = dict(cache=ctypes.byref(cache), pos=p(64), each=0, k=p(64), v=p(64), B=1, T=1, KV=1, D=128, S=10, stream=None)
    refused("ternaspmm_kv4_rows", names, good, [*({n: None} for n in ("pos", "k", "v")), *bad_cache, dict(B=0), dict(T=0), dict(KV=0), dict(D=32), dict(S=0), dict(k=p(72)), dict(v=p(72))])
    names = "logits row fp32 targets logprob entropy ids lps top work M V stream".split()
    good = dict(logits=p(64), row=10, fp32=0, targets=p(64), logprob=p(64), entropy=p(64), ids=p(64), lps=p(64), top=3, work=None, M=1, V=10, stream=None)
    refused("ternaspmm_token_logprobs", names, good, [*({n: None} for n in ("logits", "logprob", "entropy", "ids", "lps")), dict(top=-1), dict(top=11), dict(top=65, V=100), dict(M=0), dict(V=0),
                                                      dict(logits=p(65)), dict(logits=p(66), fp32=1), dict(work=p(66)), dict(row=-1), dict(V=(1 << 19) + 1)])


LAUNCHES = r"""
import ctypes
from ternainfer_amd import _lib
lib = _lib.load()
class Kv4(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "k_scale", "v", "v_scale")]
p, cache, strides = ctypes.c_void_p(64), ctypes.byref(Kv4(64, 64, 64, 64)), (ctypes.c_longlong * 3)(128, 128, 128)
rotary = lambda b, t, h, d: lib.ternaspmm_rotary(p, strides, ctypes.c_void_p(128), strides, 0, p, 0, p, 1, 1.0, b, t, h, d, 1, None)
assert rotary(1 << 24, 2, 1, 64) == -1 and rotary(1 << 23, 4, 600, 16) == -1 and rotary(1, 1 << 24, 600, 16) == -1 and rotary(1 << 25, 3, 1, 2) == -1
store = lambda b, t, h, kv: lib.ternaspmm_kv4_store(p, (h + 2 * kv) * 128, p, 0, p, 64, 1.0, p, cache, b, t, h, kv, 128, 1, 1, None)
assert store(1 << 24, 1, 16, 16) == -1
assert lib.ternaspmm_kv4_rows(cache, p, 0, p, p, 1 << 24, 1, 16, 128, 1, None) == -1
attention = lambda b, t, h, kv: lib.ternaspmm_kv4_attention(p, cache, p, 0, p, None, b, t, h, kv, 64, 1, 1.0, None)
assert attention(1 << 24, 1, 1, 1) == -1 and attention(1 << 20, 1, 256, 16) == -1 and attention(1 << 16, 16, 256, 256) == -1 and attention(1 << 21, 1, 128, 1) == -1
step = lambda b, h, kv: lib.ternaspmm_kv4_step(p, (h + 2 * kv) * 64, p, 0, p, 32, 1.0, cache, p, None, b, h, kv, 64, 1, 1.0, 1, None)
assert step(1 << 24, 1, 1) == -1 and step(1 << 20, 256, 16) == -1 and step(1 << 21, 128, 1) == -1
assert lib.ternaspmm_kv4_splits(1 << 24, 1, 1, 1, 64, 1) == -1 and lib.ternaspmm_kv4_workspace_bytes(1 << 24, 1, 1, 1, 64, 1) == -1
assert lib.ternaspmm_kv4_splits((1 << 24) - 8, 1, 1, 1, 64, 1) == 1
assert lib.ternaspmm_token_logprobs(p, 1, 0, None, None, p, None, None, 0, None, 1 << 24, 1, None) == -1
assert lib.ternaspmm_token_logprobs_workspace_bytes(1 << 24, 1, 0, 0) == -1 and lib.ternaspmm_token_logprobs_workspace_bytes((1 << 24) - 1, 1, 0, 0) == 0
print("refused")
"""


def test_sizes_that_a_launch_has_no_room_for_are_refused():
    """2^32 threads and more.  In a process of its own: one that is not refused ends it at the launch."""
    r = subprocess.run([sys.executable, "-c", LAUNCHES], capture_output=True, text=True, timeout=120, cwd=ROOT)
    assert r.returncode == 0 and "refused" in r.stdout, r.stdout + r.stderr


def test_python_functions_refuse_tensors_that_are_not_on_the_gpu():
    f = torch.ones(64, dtype=torch.float64)
    pos = torch.zeros(1, dtype=torch.int64)
    cache = T.Kv4Cache.empty(1, 1, 10, 128, device="cpu")
    rows = torch.zeros(1, 384, dtype=torch.bfloat16)
    for call in (lambda: T.rotary_embed(torch.zeros(1, 1, 1, 128), pos, f), lambda: T.kv4_store(rows, pos, f, cache, 1), lambda: T.kv4_step(rows, pos, f, cache, 1),
                 lambda: T.kv4_rows(cache, pos), lambda: T.kv4_attention(torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16), pos, cache), lambda: T.token_logprobs(torch.zeros(2, 5))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        T.token_logprobs([1.0])


def test_the_model_refuses_what_its_cache_does_not_take():
    from ternainfer_amd.model import ModelArgs, Transformer
    model = Transformer.__new__(Transformer)
    model.args = ModelArgs(dim=256, n_layers=2, n_heads=4, n_kv_heads=2)
    model.tok_embeddings = torch.zeros((10, 256), dtype=torch.bfloat16)
    assert [tuple(t.shape) for t in model.make_cache(2, 9, bits=4)[1]] == [(2, 2, 9, 32), (2, 2, 9, 2)] * 2
    assert [tuple(t.shape) for t in model.make_cache(2, 9)[1]] == [(2, 2, 9, 64)] * 2
    for bits in (0, 8, "4"):
        with pytest.raises(ValueError):
            model.make_cache(2, 9, bits=bits)
    model.args.n_heads = 8                       # heads of 32 dimensions
    with pytest.raises(ValueError):
        model.make_cache(2, 9, bits=4)
    model.args.n_heads = 4
    layer = type("Layer", (), {"fused": True})()
    model.layers = [layer]
    with pytest.raises(ValueError):              # no GPU
        model.forward(torch.zeros((2, 1), dtype=torch.int64), model.make_cache(2, 9, bits=4), torch.arange(1))
    for tokens, lens in ((torch.zeros((2, 1), dtype=torch.int64), None), (torch.zeros((2, 4), dtype=torch.int64), torch.ones(3))):
        with pytest.raises(ValueError):
            model.score(tokens, lens)


def test_what_has_no_truth_value_is_refused_with_its_own_error():
    f, pos, cache = torch.ones(64, dtype=torch.float64), torch.zeros(1, dtype=torch.int64), T.Kv4Cache.empty(1, 1, 10, 128, device="cpu")
    rows, both = torch.zeros(1, 384, dtype=torch.bfloat16), torch.tensor([True, False])
    for call in (lambda: T.rotary_embed(torch.zeros(1, 1, 1, 128), pos, f, adjacent=both), lambda: T.kv4_store(rows, pos, f, cache, 1, adjacent=both),
                 lambda: T.kv4_step(rows, pos, f, cache, 1, adjacent=both)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            call()


def test_the_default_scale_does_not_stand_in_front_of_the_checks():
    """What is no tensor: TypeError; no query of four dimensions, or one of none: ValueError -- also where the scale is left to the default."""
    f, pos, cache = torch.ones(64, dtype=torch.float64), torch.zeros(1, dtype=torch.int64), T.Kv4Cache.empty(1, 1, 10, 128, device="cpu")
    rows = torch.zeros(1, 384, dtype=torch.bfloat16)
    empty = T.Kv4Cache(*(torch.zeros((1, 1, 10, 0), dtype=torch.uint8) for _ in range(4)))
    for call in (lambda: T.kv4_attention([1.0], pos, cache), lambda: T.kv4_step([1.0], pos, f, cache, 1), lambda: T.kv4_step(rows, pos, f, (1, 2, 3, 4), 1)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: T.kv4_attention(torch.tensor(1.0), pos, cache), lambda: T.kv4_attention(torch.zeros(1, 1, 1, 0), pos, cache), lambda: T.kv4_step(rows, pos, f, empty, 1),
                 lambda: T.kv4_step(rows, pos, f, tuple(cache), 1)):
        with pytest.raises(ValueError, match="kv4_"):
            call()


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_frequencies_are_finite(value):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        T.rotary_frequencies(64, value, device="cpu")
    for more in ({"type": "linear"}, {"type": "ntk"}, {"type": "wavelength", "original_max_position": 64}, {"type": "yarn", "original_max_position": 64}):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            T.rotary_frequencies(64, 10000.0, {**more, "factor": value}, device="cpu")


def test_the_models_positions_follow_its_arguments():
    """Frequencies and tables that are kept from one call to the next: of the base and the scaling that the model has then."""
    from ternainfer_amd.model import ModelArgs, Transformer
    model, dev = Transformer.__new__(Transformer), torch.device("cpu")
    model.args = ModelArgs(dim=256, n_layers=1, n_heads=4, n_kv_heads=2)
    scaling = {"type": "linear", "factor": 2.0}
    seen = []
    for change in (lambda: None, lambda: setattr(model.args, "rope_scaling", scaling), lambda: scaling.update(factor=8.0), lambda: setattr(model.args, "rope_theta", 10000.0)):
        change()
        inv, _ = model.rope_frequencies(dev)
        assert torch.equal(inv, T.rotary_frequencies(64, model.args.rope_theta, model.args.rope_scaling, device="cpu")[0])
        assert model.rope_frequencies(dev)[0] is inv                             # kept
        table = model.rope_tables(7, dev)
        assert (table[6, 0].double() - (6 * inv).cos()).abs().max() < 1e-5 and model.rope_tables(7, dev) is table
        seen.append(inv)
    assert len({tuple(inv.tolist()) for inv in seen}) == 4
