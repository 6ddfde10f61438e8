"""What the operations on drafted trees refuse, and their index arithmetic, without a GPU."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
P = 0x10000          # a pointer that nothing follows: refusals come before any use


def refused(name, args, why):
    from kubeai_b200 import lib
    l = lib()
    assert getattr(l, name)(C.byref(args), None) == -1, why
    assert why in l.b200_last_error().decode(), l.b200_last_error()


def test_index_arithmetic_stays_in_its_buffers(tmp_path):
    exe = tmp_path / "tree_step_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "kubeai_b200" / "csrc"),
                    str(ROOT / "tests" / "native" / "tree_step_check.cc"), "-o", str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_arguments_are_laid_out_as_in_the_header(tmp_path):
    from kubeai_b200 import _lib
    kinds = dict(step_maps=_lib.StepMapsArgs, tree_attn=_lib.TreeAttnArgs, constrain=_lib.ConstrainArgs, tree_accept=_lib.TreeAcceptArgs)
    lines = [f'printf("%zu ", sizeof(b200_{k}_args));' + "".join(f'printf("%zu ", offsetof(b200_{k}_args, {f}));' for f, _ in t._fields_) for k, t in kinds.items()]
    (tmp_path / "t.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200engine.h"\nint main(void){' + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [v for t in kinds.values() for v in (C.sizeof(t), *(getattr(t, f).offset for f, _ in t._fields_))]


def maps(**kw):
    from kubeai_b200._lib import StepMapsArgs
    a = dict(S=2, T=4, max_blocks=3, ld_tables=3, num_free=5, words=1) | {k: P for k, _ in StepMapsArgs._fields_[6:]}
    return StepMapsArgs(**(a | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(S=-1), "bad sizes"), (dict(T=-1), "bad sizes"), (dict(max_blocks=-1), "bad sizes"), (dict(ld_tables=2), "bad sizes"), (dict(num_free=-1), "bad sizes"),
    (dict(S=8193), "8192"), (dict(words=9), "8 words"), (dict(words=-1), "8 words"), (dict(max_blocks=1 << 27, ld_tables=1 << 27), "32 bits"),
    *((dict([(k, None)]), "missing") for k in ("ctx", "rows", "held", "cursor", "held_out", "cursor_out", "starts", "positions", "slots", "masks", "status", "free_pages", "block_tables"))])
def test_maps_refuse(kw, why):
    refused("b200_op_step_maps", maps(**kw), why)


def attn(**kw):
    from kubeai_b200._lib import TreeAttnArgs
    a = dict(S=2, T=4, q_heads=8, kv_heads=2, ldq=1536, ldo=1024, max_blocks=3, ld_tables=3, words=1, max_tree=4, max_ctx=0, scale=0.1, num_pages=6)
    return TreeAttnArgs(**(a | {k: P for k in ("q", "out", "kv_layer", "block_tables", "starts", "ctx", "masks", "workspace")} | dict(workspace_bytes=1 << 30) | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(S=-1), "bad sizes"), (dict(T=-2), "bad sizes"), (dict(ld_tables=2), "bad sizes"), (dict(max_tree=-1), "bad sizes"), (dict(max_ctx=-1), "bad sizes"), (dict(num_pages=-1), "bad sizes"),
    (dict(q_heads=6), "1, 2, 4 or 8"), (dict(q_heads=7), "1, 2, 4 or 8"), (dict(q_heads=32, ldq=8192, ldo=4096), "1, 2, 4 or 8"), (dict(kv_heads=0), "1, 2, 4 or 8"), (dict(q_heads=0), "1, 2, 4 or 8"),
    (dict(words=0), "1 to 8 words"), (dict(words=9), "1 to 8 words"), (dict(max_tree=33), "than its masks have bits"), (dict(S=65535), "too many"),
    (dict(max_blocks=1 << 27, ld_tables=1 << 27), "32 bits"), (dict(num_pages=1 << 25), "32 bits"), (dict(ldq=1000), "whole heads"), (dict(ldo=1020), "whole heads"), (dict(ldq=1540), "whole heads"),
    (dict(scale=float("nan")), "no number"), (dict(q=P + 8), "aligned"), (dict(out=P + 2), "aligned"), (dict(kv_layer=P + 128), "aligned"), (dict(num_pages=0), "missing"),
    (dict(S=60000, max_blocks=1 << 18, ld_tables=1 << 18), "the tiles of all requests"), (dict(workspace_bytes=1 << 20), "workspace"), (dict(workspace=P + 8), "workspace"),
    *((dict([(k, None)]), "missing") for k in ("q", "out", "kv_layer", "block_tables", "starts", "ctx", "workspace"))])
def test_attention_refuses(kw, why):
    refused("b200_op_paged_attn_tree", attn(**kw), why)


def choose(**kw):
    from kubeai_b200._lib import ConstrainArgs
    a = dict(S=2, T=4, V=100, ld=100, logits_f32=1, ld_out=100, out_f32=1, words=1, history_len=9, bias_len=3, allow_count=4, ld_allow=4)
    return ConstrainArgs(**(a | {k: P for k, _ in ConstrainArgs._fields_[12:]} | dict(out=2 * P) | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(S=-1), "bad sizes"), (dict(T=-1), "bad sizes"), (dict(V=0), "bad sizes"), (dict(ld=99), "bad sizes"), (dict(ld_out=99), "bad sizes"), (dict(bias_len=-1), "bad sizes"),
    (dict(V=393217, ld=393217, ld_out=393217), "393216"), (dict(S=65535), "65534"), (dict(starts=None), "every row is a request"), (dict(ids=None, out=None), "neither"),
    (dict(words=0), "1 to 8 words"), (dict(words=9), "1 to 8 words"), (dict(drafts=None), "masks without drafts"), (dict(starts=None, S=4, masks=None), "drafts without starts"),
    (dict(hist_starts=None), "without its starts"), (dict(history_len=-1), "without its starts"), (dict(bias_ids=None), "without their tokens"), (dict(bias_values=None), "without their tokens"),
    (dict(ld_allow=3), "narrower"), (dict(allow_count=-1), "narrower"), (dict(allow_rows=None, allow_count=3), "fewer masks"), (dict(allow=None), "that are not there"), (dict(logits=None), "missing"),
    (dict(logits=P + 2), "alignment"), (dict(out=P + 1), "alignment"), (dict(out=P, out_f32=0), "in place"), (dict(out=P, ld_out=104), "in place")])
def test_constrain_refuses(kw, why):
    refused("b200_op_constrain", choose(**kw), why)


def accept(**kw):
    from kubeai_b200._lib import TreeAcceptArgs
    a = dict(S=2, T=4, max_blocks=3, ld_tables=3, max_path=4, layers=2, kv_heads=2, num_pages=6, layer_stride=6 * 2 * 4096)
    return TreeAcceptArgs(**(a | {k: P for k, _ in TreeAcceptArgs._fields_[9:]} | dict(new_ctx=2 * P) | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(S=-1), "bad sizes"), (dict(T=-1), "bad sizes"), (dict(ld_tables=1), "bad sizes"), (dict(layers=-1), "bad sizes"), (dict(num_pages=-1), "bad sizes"), (dict(max_path=0), "1 to 256"),
    (dict(max_path=257), "1 to 256"), (dict(max_blocks=1 << 27, ld_tables=1 << 27), "32 bits"), (dict(kv=None), "layers"), (dict(kv_heads=0), "layers"), (dict(layer_stride=6 * 2 * 4096 - 8), "layers"),
    (dict(layer_stride=6 * 2 * 4096 + 4), "layers"), (dict(kv=P + 8), "aligned"), (dict(new_ctx=P), "of its own"),
    *((dict([(k, None)]), "missing") for k in ("starts", "ctx", "accepted", "path", "tokens", "new_ctx", "ids", "drafts", "block_tables"))])
def test_accept_refuses(kw, why):
    refused("b200_op_tree_accept", accept(**kw), why)


def test_null_arguments_are_refused():
    from kubeai_b200 import lib
    for name in ("b200_op_step_maps", "b200_op_paged_attn_tree", "b200_op_constrain", "b200_op_tree_accept"):
        assert getattr(lib(), name)(None, None) == -1


def test_the_driver_takes_tensors_of_a_gpu_only():
    from kubeai_b200 import B200Error, ops
    i, t = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(B200Error):
        ops.step_maps(i, i, i, t, i, i, 1)
    with pytest.raises(B200Error):
        ops.paged_attn_tree(torch.zeros(1, 512).bfloat16(), torch.zeros(1, 2, 1, 16, 128).bfloat16(), t, torch.zeros(2, dtype=torch.int32), i, None, 4, 1, 1)
    with pytest.raises(B200Error):
        ops.constrain(torch.zeros(1, 10))
    with pytest.raises(B200Error):
        ops.tree_accept(i, i, None, torch.zeros(2, dtype=torch.int32), i, t, None, 1)


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a box WITHOUT a GPU")
def test_what_would_run_needs_a_gpu():
    from kubeai_b200 import lib
    l = lib()
    for name, a in (("b200_op_step_maps", maps()), ("b200_op_paged_attn_tree", attn()), ("b200_op_constrain", choose()), ("b200_op_tree_accept", accept())):
        assert getattr(l, name)(C.byref(a), None) == -5
