"""What the operations of a step whose requests share their beginnings refuse, and their index arithmetic, without a GPU."""
import ctypes as C
import math
import subprocess

import numpy as np
import pytest
import torch

from test_tree_step_cpu import ROOT, P, refused


def test_index_arithmetic_stays_in_its_buffers(tmp_path):
    exe = tmp_path / "beam_step_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "kubeai_b200" / "csrc"),
                    str(ROOT / "tests" / "native" / "beam_step_check.cc"), "-o", str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_arguments_are_laid_out_as_in_the_header(tmp_path):
    from kubeai_b200 import _lib
    kinds = dict(norm_rope=_lib.NormRopeArgs, shared_attn=_lib.SharedAttnArgs, beam_select=_lib.BeamSelectArgs, beam_reorder=_lib.BeamReorderArgs)
    lines = [f'printf("%zu ", sizeof(b200_{k}_args));' + "".join(f'printf("%zu ", offsetof(b200_{k}_args, {f}));' for f, _ in t._fields_) for k, t in kinds.items()]
    (tmp_path / "t.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200engine.h"\nint main(void){' + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [v for t in kinds.values() for v in (C.sizeof(t), *(getattr(t, f).offset for f, _ in t._fields_))]


def turn(**kw):
    from kubeai_b200._lib import NormRopeArgs
    a = dict(T=2, q_heads=4, kv_heads=2, ldx=1024, ldo=512, dims=128, interleaved=0, q_norm_ld=0, k_norm_ld=128, norm_f32=0, eps=1e-6, gain=1.0, num_pages=3)
    return NormRopeArgs(**(a | {k: P for k, _ in NormRopeArgs._fields_[13:]} | dict(out=2 * P) | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(T=-1), "bad sizes"), (dict(q_heads=-1), "bad sizes"), (dict(kv_heads=-1), "bad sizes"), (dict(num_pages=-1), "bad sizes"), (dict(q_heads=4097), "4096"), (dict(dims=130), "even number"),
    (dict(dims=-2), "even number"), (dict(dims=7), "even number"), (dict(ldx=1016), "whole heads"), (dict(ldo=504), "whole heads"), (dict(ldx=1028), "whole heads"), (dict(ldo=516), "whole heads"),
    (dict(q_norm_ld=64), "128 weights"), (dict(k_norm_ld=-128), "128 weights"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(gain=float("inf")), "eps"), (dict(qkv=P + 8), "aligned"),
    (dict(out=P + 2), "aligned"), (dict(kv_layer=P + 8), "aligned"), (dict(q_norm=P + 4), "aligned"), (dict(k_norm=P + 8, norm_f32=1), "aligned"), (dict(out=P), "in place"),
    *((dict([(k, None)]), "missing") for k in ("qkv", "out", "kv_layer", "positions", "slots", "freqs"))])
def test_rotation_refuses(kw, why):
    refused("b200_op_norm_rope_kvwrite", turn(**kw), why)


def attn(**kw):
    from kubeai_b200._lib import SharedAttnArgs
    a = dict(S=2, T=4, G=1, q_heads=8, kv_heads=2, ldq=1536, ldo=1024, max_blocks=3, ld_tables=3, max_rows=4, max_ctx=0, scale=0.1, num_pages=6)
    return SharedAttnArgs(**(a | {k: P for k, _ in SharedAttnArgs._fields_[14:-1]} | dict(workspace_bytes=1 << 30) | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(S=-1), "bad sizes"), (dict(T=-2), "bad sizes"), (dict(G=-1), "bad sizes"), (dict(ld_tables=2), "bad sizes"), (dict(max_rows=-1), "bad sizes"), (dict(max_ctx=-1), "bad sizes"),
    (dict(num_pages=-1), "bad sizes"), (dict(q_heads=6), "1, 2, 4 or 8"), (dict(q_heads=7), "1, 2, 4 or 8"), (dict(q_heads=32, ldq=8192, ldo=4096), "1, 2, 4 or 8"), (dict(kv_heads=0), "1, 2, 4 or 8"),
    (dict(q_heads=0), "1, 2, 4 or 8"), (dict(S=65535), "too many"), (dict(G=65535), "too many"), (dict(max_blocks=1 << 27, ld_tables=1 << 27), "32 bits"), (dict(num_pages=1 << 25), "32 bits"),
    (dict(ldq=1000), "whole heads"), (dict(ldo=1020), "whole heads"), (dict(ldq=1540), "whole heads"), (dict(scale=float("nan")), "no number"), (dict(scale=0.0), "no number"),
    (dict(scale=-1.0), "no number"), (dict(q=P + 8), "aligned"), (dict(out=P + 2), "aligned"), (dict(kv_layer=P + 128), "aligned"), (dict(num_pages=0), "missing"), (dict(T=1 << 29), "too many rows"),
    (dict(S=60000, max_blocks=1 << 20, ld_tables=1 << 20), "the pages of all requests"), (dict(workspace_bytes=1 << 20), "workspace"), (dict(workspace=P + 8), "workspace"),
    *((dict([(k, None)]), "missing") for k in ("q", "out", "kv_layer", "block_tables", "starts", "ctx", "group_starts", "shared", "workspace"))])
def test_attention_refuses(kw, why):
    refused("b200_op_paged_attn_shared", attn(**kw), why)


def choose(**kw):
    from kubeai_b200._lib import BeamSelectArgs
    a = dict(S=2, beams=3, V=100, ld=100, logits_f32=1, k=6, num_ends=1)
    return BeamSelectArgs(**(a | {k: P for k, _ in BeamSelectArgs._fields_[7:-1]} | dict(scores=2 * P, workspace_bytes=1 << 20) | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(S=-1), "bad sizes"), (dict(V=0), "bad sizes"), (dict(ld=99), "bad sizes"), (dict(num_ends=-1), "bad sizes"), (dict(beams=0), "32 beams"), (dict(beams=33), "32 beams"), (dict(k=0), "64 candidates"),
    (dict(k=65), "64 candidates"), (dict(V=393217, ld=393217), "393216"), (dict(num_ends=1025), "1024"), (dict(S=1 << 28), "too many"), (dict(logits=P + 2), "alignment"), (dict(logits=P + 1, logits_f32=0), "alignment"),
    (dict(scores=P), "of their own"), (dict(workspace_bytes=10), "workspace"), (dict(workspace=P + 8), "workspace"),
    *((dict([(k, None)]), "missing") for k in ("logits", "scores", "ends", "parents", "tokens", "new_scores", "found_parents", "found_tokens", "found_scores"))])
def test_selection_refuses(kw, why):
    refused("b200_op_beam_select", choose(**kw), why)


def move(**kw):
    from kubeai_b200._lib import BeamReorderArgs
    a = dict(S=2, beams=3, max_blocks=3, ld_tables=3, ld_tables_out=3, layers=2, kv_heads=2, room=5, ld_texts=5, ld_texts_out=5, num_pages=6, layer_stride=6 * 2 * 4096)
    return BeamReorderArgs(**(a | {k: P for k, _ in BeamReorderArgs._fields_[12:]} | dict(tables_out=2 * P, texts_out=3 * P, text_lens_out=4 * P) | kw))


@pytest.mark.parametrize("kw,why", [
    (dict(S=-1), "bad sizes"), (dict(ld_tables=2), "bad sizes"), (dict(ld_tables_out=2), "bad sizes"), (dict(layers=-1), "bad sizes"), (dict(room=-1), "bad sizes"), (dict(num_pages=-1), "bad sizes"),
    (dict(beams=0), "32 beams"), (dict(beams=33), "32 beams"), (dict(max_blocks=1 << 27, ld_tables=1 << 27, ld_tables_out=1 << 27), "32 bits"), (dict(S=1 << 27), "too many"), (dict(kv=None), "layers"),
    (dict(kv_heads=0), "layers"), (dict(layer_stride=6 * 2 * 4096 - 8), "layers"), (dict(layer_stride=6 * 2 * 4096 + 4), "layers"), (dict(kv=P + 8), "aligned"), (dict(ld_texts=4), "less room"),
    (dict(ld_texts_out=4), "less room"), (dict(tables_out=P), "of its own"), (dict(texts_out=P), "of its own"), (dict(text_lens_out=P), "of its own"),
    *((dict([(k, None)]), "missing") for k in ("parents", "ctx", "shared", "block_tables", "tables_out", "released", "tokens", "texts_out", "text_lens", "text_lens_out"))])
def test_reordering_refuses(kw, why):
    refused("b200_op_beam_reorder", move(**kw), why)


def test_null_arguments_are_refused():
    from kubeai_b200 import lib
    for name in ("b200_op_norm_rope_kvwrite", "b200_op_paged_attn_shared", "b200_op_beam_select", "b200_op_beam_reorder"):
        assert getattr(lib(), name)(None, None) == -1


def test_calls_without_work_need_no_device():
    from kubeai_b200 import lib
    for name, a in (("norm_rope_kvwrite", turn(T=0)), ("paged_attn_shared", attn(T=0)), ("beam_select", choose(S=0)), ("beam_reorder", move(S=0))):
        assert getattr(lib(), "b200_op_" + name)(C.byref(a), None) == 0, name


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_the_driver_takes_tensors_of_a_gpu_only():
    from kubeai_b200 import B200Error, ops
    i = ints(1)
    kv, q, f = torch.zeros(1, 2, 1, 16, 128).bfloat16(), torch.zeros(1, 512).bfloat16(), torch.zeros(64, dtype=torch.float64)
    for call in (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 2, 1, f), lambda: ops.paged_attn_shared(q, kv, ints(1, 1), ints(2), i, ints(1), ints(0), 4, 1, 1),
                 lambda: ops.beam_select(torch.zeros(1, 10), torch.zeros(1, 1)), lambda: ops.beam_reorder(ints(1, 1), ints(1, 1), i, ints(1, 1), None)):
        with pytest.raises(B200Error, match="current GPU"):
            call()


@pytest.fixture
def ops(monkeypatch):
    from kubeai_b200 import ops
    monkeypatch.setattr(ops, "_gpu", lambda t: t.get_device())
    return ops


def test_the_driver_refuses_what_does_not_fit(ops):
    from kubeai_b200 import B200Error
    i, kv, f = ints(2), torch.zeros(1, 2, 1, 16, 128).bfloat16(), torch.zeros(64, dtype=torch.float64)
    q, w = torch.zeros(2, 512).bfloat16(), torch.zeros(128).bfloat16()
    x, sc, one = torch.zeros(4, 10), torch.zeros(2, 2), ints(2, 2)
    calls = [
        (lambda: ops.norm_rope_kvwrite(q, ints(3), i, kv, 2, 1, f), "positions"), (lambda: ops.norm_rope_kvwrite(q, i, ints(3), kv, 2, 1, f), "slots"), (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 3, 1, f), "qkv"),
        (lambda: ops.norm_rope_kvwrite(q.float(), i, i, kv, 2, 1, f), "qkv"), (lambda: ops.norm_rope_kvwrite(q, i, i, kv[0], 2, 1, f), "kv_layer"), (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 2, 1, f.float()), "freqs"),
        (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 2, 1, torch.zeros(65, dtype=torch.float64)), "freqs"), (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 2, 1, f, q_norm=w[:64]), "q_norm"),
        (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 2, 1, f, k_norm=torch.zeros(2, 128).bfloat16()), "k_norm"), (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 2, 1, f, q_norm=w, k_norm=w.float()), "one type"),
        (lambda: ops.norm_rope_kvwrite(q, i, i, kv, 2, 1, f, out=q[:1]), "out"), (lambda: ops.norm_rope_kvwrite(q, i.long(), i, kv, 2, 1, f), "int32"),
        (lambda: ops.paged_attn_shared(q, kv, ints(2, 4), ints(3), i, ints(1), ints(1), 4, 1, 1), "group_starts"), (lambda: ops.paged_attn_shared(q, kv, ints(2, 4), ints(2), i, ints(2), ints(1), 4, 1, 1), "starts"),
        (lambda: ops.paged_attn_shared(q, kv, ints(3, 4), ints(3), i, ints(2), ints(1), 4, 1, 1), "block tables"), (lambda: ops.paged_attn_shared(q, kv, ints(2, 4), ints(3), i, ints(2), ints(1), 4, 2, 1), "kv_layer"),
        (lambda: ops.paged_attn_shared(q, kv, ints(2, 4), ints(3), i, ints(2), ints(1), 4, 1, 1, status=ints(3)), "status"),
        (lambda: ops.beam_select(x[:3], sc), "rows"), (lambda: ops.beam_select(x.half(), sc), "logits"), (lambda: ops.beam_select(x, sc.double()), "scores"), (lambda: ops.beam_select(x, sc[0]), "scores"),
        (lambda: ops.beam_select(x, sc, ends=ints(2).long()), "int32"), (lambda: ops.beam_select(x, sc, k=1 << 33), "32 bits"),
        (lambda: ops.beam_reorder(ints(4), one, ints(4), ints(4, 2), None), "parents"), (lambda: ops.beam_reorder(one, ints(3), ints(4), ints(4, 2), None), "tokens"),
        (lambda: ops.beam_reorder(one, one, ints(2), ints(4, 2), None), "ctx_lens"), (lambda: ops.beam_reorder(one, one, ints(4), ints(3, 2), None), "block tables"),
        (lambda: ops.beam_reorder(one, one, ints(4), ints(4, 2), kv), "kv: "), (lambda: ops.beam_reorder(one, one, ints(4), ints(4, 2), None, texts=ints(4, 3)), "without their lengths"),
        (lambda: ops.beam_reorder(one, one, ints(4), ints(4, 2), None, texts=ints(3, 3), text_lens=ints(4)), "texts"), (lambda: ops.beam_reorder(one, one, ints(4), ints(4, 2), None, out=ints(4, 1)), "out"),
    ]
    for n, (call, why) in enumerate(calls):
        with pytest.raises(B200Error, match=why):
            call()
            pytest.fail(f"call {n} was taken")


@pytest.mark.parametrize("scaling", [None, dict(rope_type="linear", factor=4.0), dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192),
                                     dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)])
def test_frequencies_are_those_of_the_configuration(scaling):
    """Against the scalings as transformers computes them from a configuration, in 32 bits: 2^-22 for a handful of roundings (a power, a quotient, two products and a sum)."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    from kubeai_b200 import ops
    dims, base = 128, 500000.0
    r = ops.rotary(dims, base, scaling, device="cpu")
    assert r.freqs.dtype is torch.float64 and r.freqs.shape == (64,)
    if scaling is None:
        want, gain = base ** (-np.arange(0, dims, 2) / dims), 1.0
    else:
        kind = scaling.get("rope_type", scaling.get("type"))
        cfg = LlamaConfig(hidden_size=128, num_attention_heads=1, head_dim=128, max_position_embeddings=131072, rope_theta=base, rope_scaling={k: v for k, v in scaling.items() if k != "type"} | dict(rope_type=kind, rope_theta=base))
        want, gain = ROPE_INIT_FUNCTIONS[kind](cfg, "cpu")
        want = want.double().numpy()
    assert abs(r.gain - gain) < 1e-6
    assert np.allclose(r.freqs.numpy(), want, rtol=2.0 ** -20 if scaling else 1e-14, atol=0)


@pytest.mark.parametrize("dims,base,scaling,why", [
    (130, 1e4, None, "even number"), (7, 1e4, None, "even number"), (-2, 1e4, None, "even number"), (64, 0.0, None, "even number"), (64, 1e4, dict(type="dynamic", factor=2), "not supported"),
    (64, 1e4, dict(type="linear"), "lacks"), (64, 1e4, dict(type="linear", factor=0), "above 0"), (64, 1e4, dict(rope_type="llama3", factor=8), "lacks"), (64, 1.0, dict(type="yarn", factor=2, original_max_position_embeddings=64), "zero")])
def test_frequencies_refuse(dims, base, scaling, why):
    from kubeai_b200 import B200Error, ops
    with pytest.raises(B200Error, match=why):
        ops.rotary(dims, base, scaling, device="cpu")


def test_gain_of_yarn():
    from kubeai_b200 import ops
    y = dict(type="yarn", factor=32.0, original_max_position_embeddings=4096)
    assert math.isclose(ops.rotary(128, 1e4, y, device="cpu").gain, 0.1 * math.log(32) + 1)
    assert ops.rotary(128, 1e4, y | dict(attention_factor=1.5), device="cpu").gain == 1.5


def configured(dims, base, scaling):
    """Frequencies and gain as transformers makes them of a configuration, in 32 bits."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    cfg = LlamaConfig(hidden_size=dims, num_attention_heads=1, head_dim=dims, max_position_embeddings=131072, rope_theta=base, rope_scaling=scaling | dict(rope_theta=base))
    f, gain = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    return f.double().numpy(), gain


YARN = dict(rope_type="yarn", factor=32.0, original_max_position_embeddings=4096)


@pytest.mark.parametrize("dims,base,more", [
    (64, 150000.0, dict(truncate=False)), (64, 150000.0, dict(truncate=True)), (128, 10000.0, dict(truncate=False, beta_fast=20.0, beta_slow=2.0)), (128, 1e6, dict(truncate=False, factor=4.0)),
    (64, 10000.0, dict(mscale=1.0, mscale_all_dim=1.0, factor=40.0)), (64, 10000.0, dict(mscale=0.707, mscale_all_dim=1.0, factor=40.0)), (64, 10000.0, dict(mscale=0.707, factor=40.0)),
    (64, 10000.0, dict(mscale_all_dim=0.5)), (64, 10000.0, dict(mscale=0, mscale_all_dim=0)), (128, 10000.0, dict(mscale=1.0, mscale_all_dim=0.707, attention_factor=1.5)),
    (128, 10000.0, dict(attention_factor=None, beta_fast=None, mscale=None, truncate=False)), (128, 10000.0, dict(factor=1.0, mscale=2.0, mscale_all_dim=1.0))])
def test_further_forms_of_yarn(dims, base, more):
    """2^-20 for the 32 bits of the other side (a power, its quotient, two products and a sum), and what its ramp p loses: an end of up to 2^6 is rounded by 2^-19 where the ramp is longer than 2^3, p
    and 1 - p by 2^-24 each, so 1 - p is off by less than 2^-21; a frequency is f (p / factor + 1 - p) and no less than f / factor, so that is 2^-21 of it times the factor."""
    from kubeai_b200 import ops
    want, gain = configured(dims, base, YARN | {k: v for k, v in more.items() if v is not None})
    r = ops.rotary(dims, base, YARN | more, device="cpu")
    assert abs(r.gain - gain) < 1e-6, (r.gain, gain)
    assert np.allclose(r.freqs.numpy(), want, rtol=2.0 ** -20 + 2.0 ** -21 * more.get("factor", 32.0), atol=0)


@pytest.mark.parametrize("dims,base,scaling,why", [
    (64, 1e4, YARN | dict(finetuned=True), "'finetuned'"), (64, 1e4, dict(rope_type="linear", factor=2.0, beta_fast=32), "'beta_fast'"), (64, 1e4, dict(rope_type="linear", factor=2.0, attention_factor=2.0), "'attention_factor'"),
    (128, 1e4, dict(rope_type="default", mrope_section=[16, 24, 24]), "'mrope_section'"), (128, 1e4, dict(short_factor=[1.0], long_factor=[1.0]), "'long_factor', 'short_factor'"),
    (128, 1e4, dict(factor=2.0), "'factor'"), (128, 1e4, dict(rope_theta=5e5), "says otherwise"), (128, 1e4, dict(partial_rotary_factor=0.5), "says otherwise"),
    (64, 1e4, YARN | dict(factor=None), "lacks 'factor'"), (64, 1e4, YARN | dict(factor="many"), "cannot be made of"), (64, 1e4, YARN | dict(beta_fast=-1.0), "cannot be made of"), (64, 1e4, YARN | dict(mscale=[1]), "cannot be made of")])
def test_scalings_that_are_not_handled_are_refused(dims, base, scaling, why):
    from kubeai_b200 import B200Error, ops
    with pytest.raises(B200Error, match=why):
        ops.rotary(dims, base, scaling, device="cpu")


def test_a_scaling_may_say_what_the_call_says():
    from kubeai_b200 import ops
    plain = ops.rotary(64, 1e6, device="cpu")
    same = ops.rotary(64, 1e6, dict(rope_type="default", rope_theta=1e6, partial_rotary_factor=0.5, original_max_position_embeddings=4096, factor=None), device="cpu")
    assert torch.equal(plain.freqs, same.freqs) and plain.gain == same.gain


def test_costs_stay_within_their_bound(tmp_path):
    exe = tmp_path / "beam_costs_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "kubeai_b200" / "csrc"),
                    str(ROOT / "tests" / "native" / "beam_costs_check.cc"), "-o", str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


LONG = dict(S=256, T=768, G=32, q_heads=32, kv_heads=8, ldq=6144, ldo=4096, max_blocks=8192, ld_tables=8192, max_rows=512, num_pages=100)


def test_one_long_portion_among_many_requests_is_taken():
    """256 requests with 768 rows, 512 of them one's: 448 pieces of 16 rows in all where starts ascend, not 128 for each."""
    from kubeai_b200 import lib
    small = lib().b200_op_paged_attn_shared_workspace(C.byref(attn(**LONG | dict(S=254))))
    assert small > 0 and lib().b200_op_paged_attn_shared_workspace(C.byref(attn(**LONG))) == small + 260 * 4      # the starts' copy
    refused("b200_op_paged_attn_shared", attn(**LONG | dict(workspace_bytes=small)), "workspace")
    refused("b200_op_paged_attn_shared", attn(**LONG | dict(max_blocks=1 << 22, ld_tables=1 << 22)), "the pages of all requests")


@pytest.mark.parametrize("scaling", [dict(rope_theta="x"), dict(partial_rotary_factor="half"), dict(partial_rotary_factor=float("nan")), dict(partial_rotary_factor=float("inf"))])
def test_scalings_without_numbers_are_refused(scaling):
    from kubeai_b200 import B200Error, ops
    with pytest.raises(B200Error, match="cannot be made of"):
        ops.rotary(64, 1e4, scaling, device="cpu")
