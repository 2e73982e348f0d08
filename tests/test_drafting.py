"""ternainfer_amd/drafting.py and int8_linear.py where no GPU is needed: layouts, and what is refused before anything is enqueued."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import ternainfer_amd as T
from ternainfer_amd import _lib
from ternainfer_amd.model import ModelArgs, Transformer, ngram_drafts
from tests import _drafting as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plans_cover_every_row(tmp_path):
    exe = tmp_path / "draft_plan_check"
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", os.path.join(ROOT, "tests", "draft_plan_check.cpp"), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "draft plans ok" in r.stdout, r.stdout + r.stderr


def test_sizes():
    lib = _lib.load()
    tree = lib.ternaspmm_tree_attention_workspace_bytes
    assert tree(1, 8, 20, 5, 96, 384) == tree(1, 8, 20, 3, 128, 384) == tree(0, 8, 20, 5, 128, 384) == tree(1, 513, 20, 5, 128, 384) == tree(1, 8, 20, 5, 128, (1 << 25) + 1) == -1
    assert tree(1 << 20, 512, 4, 1, 64, 10) == -1 and tree(1, 1, 1, 1, 64, 1) == 0 and tree(1, 60, 20, 5, 128, 32768) > 0
    accept = lib.ternaspmm_tree_accept_workspace_bytes
    assert accept(1, 0, 10, 0) == accept(1, 513, 10, 0) == accept(0, 1, 10, 0) == accept(1, 1, 0, 0) == accept(1, 1, (1 << 19) + 1, 0) == -1 and accept(3, 5, 10, 1) == 8 * 15
    int8 = lib.ternaspmm_int8_bytes
    assert int8(0, 5) == int8(5, 0) == int8(1, 131057) == int8((1 << 28) + 1, 64) == -1
    assert int8(1, 1) == 2048 and int8(16, 128) == 2048 and int8(17, 129) == 2 * 4 * 1024 and int8(1, 131056) == 2 * 1024 * 1024
    work = lib.ternaspmm_int8_linear_workspace_bytes
    assert work(0, 5, 5) == work(5, 0, 5) == work(5, 5, 0) == work(1 << 28, 1 << 28, 64) == -1
    assert work(60, 2560, 6912) > 0 and work(4096, 13824, 2560) == 0


def _refused(call, names, good, wrongs):
    lib = _lib.load()
    for wrong in wrongs:
        arguments = {**good, **wrong}
        assert getattr(lib, call)(*(arguments[n] for n in names)) == -1, (call, wrong)


class _Rows(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_void_p), ("sequence", ctypes.c_longlong), ("head", ctypes.c_longlong), ("slot", ctypes.c_longlong), ("heads", ctypes.c_int),
                ("slots", ctypes.c_int), ("bytes", ctypes.c_int)]


def test_c_entry_points_refuse_before_they_enqueue():
    """Missing and misaligned pointers and unsupported sizes: -1 without a launch, so this runs without a GPU."""
    p = lambda address: ctypes.c_void_p(address)
    names = "parents mask depth B T stream".split()
    good = dict(parents=p(64), mask=p(64), depth=p(64), B=1, T=1, stream=None)
    _refused("ternaspmm_draft_tree", names, good, [*({n: None} for n in names[:3]), dict(B=0), dict(T=0), dict(T=513), dict(B=1 << 24)])
    strides = lambda *s: (ctypes.c_longlong * 3)(*s)
    fine = strides(1280, 128, 128)
    names = "q qs k ks v vs start mask each out work B T H KV D S scale stream".split()
    good = dict(q=p(64), qs=fine, k=p(64), ks=fine, v=p(64), vs=fine, start=p(64), mask=p(64), each=0, out=p(64), work=None, B=1, T=1, H=1, KV=1, D=128, S=10, scale=1.0, stream=None)
    _refused("ternaspmm_tree_attention", names, good,
             [*({n: None} for n in ("q", "qs", "k", "ks", "v", "vs", "start", "mask", "out")), *({n: p(72)} for n in ("q", "k", "v", "out", "work")),
              *({n: strides(1280, 128, 4)} for n in ("qs", "ks", "vs")), dict(ks=strides(1280, 128, -128)), dict(vs=strides(1280, 128, 1 << 24)), dict(B=0), dict(T=0), dict(T=513),
              dict(H=0), dict(KV=0), dict(H=3, KV=2), dict(H=4097), dict(D=96), dict(S=0), dict(S=(1 << 25) + 1), dict(scale=float("nan")), dict(scale=float("inf")),
              dict(B=1 << 21, H=256, T=1)])
    names = "logits row fp32 tokens parents path count next work B T V stream".split()
    good = dict(logits=p(64), row=10, fp32=0, tokens=p(64), parents=p(64), path=p(64), count=p(64), next=p(64), work=p(64), B=1, T=1, V=10, stream=None)
    _refused("ternaspmm_tree_accept", names, good, [*({n: None} for n in ("logits", "tokens", "parents", "path", "count", "next", "work")), dict(work=p(68)), dict(logits=p(65)),
                                                    dict(logits=p(66), fp32=1), dict(row=-1), dict(B=0), dict(T=0), dict(T=513), dict(V=0), dict(V=(1 << 19) + 1), dict(B=1 << 24)])
    rows = lambda **more: ctypes.byref(_Rows(**{**dict(rows=64, sequence=1000, head=100, slot=10, heads=1, slots=5, bytes=10), **more}))
    names = "caches n start path count B T stream".split()
    good = dict(caches=rows(), n=1, start=p(64), path=p(64), count=p(64), B=1, T=1, stream=None)
    _refused("ternaspmm_cache_move", names, good, [*({n: None} for n in ("caches", "start", "path", "count")), dict(n=-1), dict(B=0), dict(B=65536), dict(T=0), dict(T=513),
                                                   *(dict(caches=rows(**{n: 0})) for n in ("rows", "heads", "slots", "bytes")), dict(caches=rows(slot=9)), dict(caches=rows(head=-1)),
                                                   dict(caches=rows(sequence=-1))])
    names = "x row fp32 packed scale R K stream".split()
    good = dict(x=p(64), row=10, fp32=0, packed=p(64), scale=p(64), R=1, K=10, stream=None)
    _refused("ternaspmm_int8_quantise", names, good, [*({n: None} for n in ("x", "packed", "scale")), dict(x=p(65)), dict(x=p(66), fp32=1), dict(packed=p(72)), dict(row=-1), dict(R=0),
                                                      dict(K=0), dict(K=131057), dict(R=1 << 28)])
    names = "x row packed R K stream".split()
    good = dict(x=p(64), row=10, packed=p(64), R=1, K=10, stream=None)
    _refused("ternaspmm_int8_pack", names, good, [dict(x=None), dict(packed=None), dict(packed=p(72)), dict(row=-1), dict(R=0), dict(K=0), dict(K=131057)])
    names = "x xs w ws out fp32 work M N K stream".split()
    good = dict(x=p(64), xs=p(64), w=p(64), ws=p(64), out=p(64), fp32=0, work=None, M=1, N=1, K=10, stream=None)
    _refused("ternaspmm_int8_linear", names, good, [*({n: None} for n in ("x", "xs", "w", "ws", "out")), *({n: p(72)} for n in ("x", "w", "out", "work")), dict(M=0), dict(N=0), dict(K=0),
                                                    dict(K=131057), dict(M=1 << 28, N=1 << 28)])


def test_python_functions_refuse_what_they_do_not_take():
    longs, rows = torch.zeros((1, 3), dtype=torch.int64), torch.zeros((1, 1, 4, 64), dtype=torch.bfloat16)
    for call in (lambda: T.draft_tree(longs), lambda: T.tree_attention(rows, rows, rows, longs[0, :1], longs), lambda: T.tree_accept(torch.zeros(1, 3, 5), longs, longs),
                 lambda: T.cache_move([rows], longs[0, :1], longs, longs[0, :1]), lambda: T.quantise_rows(torch.zeros(2, 3)), lambda: T.int8_rows(torch.zeros((2, 3), dtype=torch.int8), torch.zeros(2))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: T.draft_tree([0]), lambda: T.tree_attention(rows, [1], rows, longs, longs), lambda: T.tree_accept(rows, [1], longs), lambda: T.cache_move([1], longs[0, :1], longs, longs[0, :1]),
                 lambda: T.quantise_rows([1.0]), lambda: T.int8_linear(torch.zeros(2, 3), torch.zeros(2, 3))):
        with pytest.raises((TypeError, ValueError)):
            call()
    weight = T.Int8Rows(torch.zeros(2048, dtype=torch.uint8), torch.zeros(3), 3, 3)
    for call in (lambda: T.int8_linear(torch.zeros(2, 3), weight), lambda: T.int8_linear(torch.zeros(2, 3), weight, torch.float16),
                 lambda: T.int8_linear(weight._replace(columns=4), weight)):
        with pytest.raises(ValueError, match="int8_linear"):
            call()


def test_the_oracles_trees():
    parents = torch.tensor([[-1, 0, 1, 1, -2, 4, 7, -1, 7]])
    mask, depth = P.tree(parents)
    assert depth.tolist() == [[0, 1, 2, 2, -1, -1, -1, 0, 1]]
    assert mask[0, :, 0].tolist() == [1, 3, 7, 11, 0, 0, 0, 128, 384]


def test_drafts_from_the_text():
    text = torch.tensor([[5, 6, 7, 8, 5, 6, 9, 9, 5, 6, 0, 0], [1, 2, 3, 4, 0, 0, 0, 0, 0, 0, 0, 0], [7, 7, 7, 0, 0, 0, 0, 0, 0, 0, 0, 0], [4, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0]])
    tokens, parents = ngram_drafts(text, torch.tensor([10, 4, 3, 1]), 2, 3)
    assert tokens.tolist()[0] == [6, 9, 9, 5, 7, 8, 5] and parents.tolist()[0] == [-1, 0, 1, 2, 0, 4, 5]       # the latest place first
    assert tokens.tolist()[1][0] == 4 and parents.tolist()[1] == [-1] + [-2] * 6
    assert tokens.tolist()[2][:2] == [7, 7] and parents.tolist()[2] == [-1, 0] + [-2] * 5                       # what follows ends with the text
    assert parents.tolist()[3] == [-1] + [-2] * 6                                                               # no two tokens yet
    assert ngram_drafts(text, torch.tensor([0, 0, 0, 0]))[1][:, 0].tolist() == [-2] * 4
    tokens, parents = ngram_drafts(text[:, :3], torch.tensor([3, 3, 3, 1]), 5, 2)                               # more branches than the text is long
    assert tokens.shape == parents.shape == (4, 11)


def test_the_model_refuses_what_a_tree_step_does_not_take():
    model = Transformer.__new__(Transformer)
    model.args = ModelArgs(dim=256, n_layers=1, n_heads=4, n_kv_heads=2)
    model.tok_embeddings = torch.zeros((10, 256), dtype=torch.bfloat16)
    model.layers = [type("Layer", (), {"fused": True})()]
    tree = T.DraftTree(torch.ones((1, 2, 1), dtype=torch.int64), torch.zeros((1, 2), dtype=torch.int64))
    for bits in (4, 16):
        with pytest.raises(ValueError, match="tree_step"):
            model.tree_step(torch.zeros((1, 2), dtype=torch.int64), model.make_cache(1, 9, bits), torch.zeros(1, dtype=torch.int64), tree)
