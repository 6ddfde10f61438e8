"""The bookkeeping of a ring of chunks, without a GPU: what a warp does where a copy never comes."""
import subprocess

from test_tree_step_cpu import ROOT


def test_a_ring_ends_at_the_chunk_that_does_not_come(tmp_path):
    exe = tmp_path / "chunk_ring_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "kubeai_b200" / "csrc"),
                    str(ROOT / "tests" / "native" / "chunk_ring_check.cc"), "-o", str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
