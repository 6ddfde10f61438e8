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


@pytest.mark.parametrize("kw", [dict(T=(1 << 30) + 1), dict(num_free=(1 << 31) - 1)])
def test_maps_refuse_what_indexes_would_pass(kw):
    refused("b200_op_step_maps", maps(**kw), "2^30")


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, float("inf"), float("-inf"), 1e30, float("nan")])
def test_attention_refuses_scales_that_turn_scores_around(scale):
    refused("b200_op_paged_attn_tree", attn(scale=scale), "above 0")


@pytest.mark.parametrize("kw", [dict(T=(1 << 30) + 1, allow_count=(1 << 30) + 1), dict(history_len=(1 << 29) + 1), dict(bias_len=(1 << 31) - 1)])
def test_constrain_refuses_what_indexes_would_pass(kw):
    refused("b200_op_constrain", choose(**kw), "2^30")
