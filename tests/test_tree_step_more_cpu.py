"""More of what the operations on drafted trees refuse, and how an attention call's work is cut, without a GPU."""
import subprocess

import pytest

from test_tree_step_cpu import ROOT, P, accept, attn, choose, maps, refused


def test_ranges_take_every_tile_once(tmp_path):
    exe = tmp_path / "tree_ranges_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "kubeai_b200" / "csrc"),
                    str(ROOT / "tests" / "native" / "tree_ranges_check.cc"), "-o", str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
