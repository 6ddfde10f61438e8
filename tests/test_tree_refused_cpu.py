"""A request that step_maps turns away, as the operations behind it see it, without a GPU."""
import subprocess

from test_tree_step_cpu import ROOT


def test_requests_that_are_turned_away_have_no_rows(tmp_path):
    exe = tmp_path / "tree_refused_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "kubeai_b200" / "csrc"),
                    str(ROOT / "tests" / "native" / "tree_refused_check.cc"), "-o", str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
