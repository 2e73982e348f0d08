"""The layout of the attention over the 4-bit cache (csrc/kv4_plan.h), on the CPU."""
import os
import subprocess

from ternainfer_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_plan_covers_every_row(tmp_path):
    exe = tmp_path / "kv4_plan_check"
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", os.path.join(ROOT, "tests", "kv4_plan_check.cpp"), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "kv4 plan ok" in r.stdout, r.stdout + r.stderr


def test_a_step_of_many_query_heads_has_room_for_its_queries():
    lib = _lib.load()
    for b, h, kv, d, s in ((128, 128, 1, 128, 40), (256, 64, 1, 128, 128), (96, 48, 1, 128, 6000), (8, 71, 1, 64, 32768), (4, 128, 1, 64, 32768)):
        splits = lib.ternaspmm_kv4_splits(b, 1, h, kv, d, s)
        parts = 0 if splits == 1 else 4 * b * h * splits * (d + 2)
        assert lib.ternaspmm_kv4_workspace_bytes(b, 1, h, kv, d, s) == 2 * b * h * d + parts
