"""What the Python operations on drafted trees make of their tensors, ahead of the library: on CPU tensors that stand for a GPU's."""
import pytest
import torch


@pytest.fixture
def ops(monkeypatch):
    from kubeai_b200 import ops
    monkeypatch.setattr(ops, "_gpu", lambda t: t.get_device())
    return ops


@pytest.mark.parametrize("rows", [1, 4])
def test_masks_narrower_than_the_vocabulary_are_refused_however_far_apart_they_lie(ops, rows):
    """4008 words for 128256 tokens: the last columns of a buffer have rows 4010 words apart, and 4006 words each."""
    from kubeai_b200 import B200Error
    allow = torch.zeros(4, 4010, dtype=torch.int32)[:rows, 4:]
    with pytest.raises(B200Error, match="allow"):
        ops.constrain(torch.zeros(1, 128256), allow=allow, allow_rows=torch.zeros(1, dtype=torch.int32))


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("shape", [(2, 0), (2, 9), (1, 1), (2,), (2, 1, 1)])
def test_masks_without_words_are_not_no_masks(ops, shape):
    """A tensor of no values has no address, which the library would take for a chain."""
    from kubeai_b200 import B200Error
    with pytest.raises(B200Error, match="masks: "):
        ops.paged_attn_tree(torch.zeros(2, 512).bfloat16(), torch.zeros(1, 2, 1, 16, 128).bfloat16(), ints(1, 1), ints(2), ints(1), ints(*shape), 4, 1, 2)
    with pytest.raises(B200Error, match="masks: "):
        ops.constrain(torch.zeros(2, 10), starts=ints(2), drafts=ints(2), masks=ints(*shape))


def test_rows_may_name_no_mask_where_there_are_none(ops, monkeypatch):
    """A step in which no request has a grammar: no masks, and -1 for every row."""
    from kubeai_b200 import B200Error
    calls = []

    class Library:
        @staticmethod
        def b200_op_constrain(a, stream):
            calls.append(a._obj)
            return 0

    monkeypatch.setattr(ops, "lib", lambda: Library)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda at: 0)
    x = torch.zeros(2, 70)
    ops.constrain(x, allow=ints(0, 3), allow_rows=ints(2) - 1)
    ops.constrain(x, allow=ints(4, 3), allow_rows=ints(2) - 1)
    without, with_masks = calls
    assert not without.allow and not without.allow_rows and with_masks.allow and with_masks.allow_rows and with_masks.allow_count == 4
    for bad in (dict(allow=ints(0, 3)), dict(allow=ints(0, 2), allow_rows=ints(2) - 1), dict(allow=ints(0, 3), allow_rows=ints(1))):
        with pytest.raises(B200Error, match="allow"):
            ops.constrain(x, **bad)
    assert len(calls) == 2


@pytest.mark.parametrize("more", [1 << 31, (1 << 32) + 2])
def test_sizes_that_pass_32_bits_are_refused_and_not_cut_off(ops, more):
    """Of 2^32 + 2 the library would see 2.  (Tensors without memory: nothing follows their addresses.)"""
    from kubeai_b200 import B200Error
    far = lambda rows, n, dtype: torch.empty_strided((rows, n), (more + n, 1), dtype=dtype, device="meta")      # noqa: E731
    q, kv, i, s = torch.zeros(2, 512).bfloat16(), torch.zeros(1, 2, 1, 16, 128).bfloat16(), ints(2), ints(3)
    big = torch.empty(more, dtype=torch.int32, device="meta")
    calls = [
        lambda: ops.step_maps(i, i, i, ints(2, 4), i, ints(1), more),
        lambda: ops.step_maps(i, i, i, far(2, 4, torch.int32), i, ints(1), 2),
        lambda: ops.step_maps(i, i, i, ints(2, 4), big, ints(1), 2),
        lambda: ops.paged_attn_tree(q, kv, ints(2, 4), s, i, None, 4, 1, more),
        lambda: ops.paged_attn_tree(q, kv, ints(2, 4), s, i, None, 4, 1, 2, max_ctx=more),
        lambda: ops.paged_attn_tree(far(2, 512, torch.bfloat16), kv, ints(2, 4), s, i, None, 4, 1, 2),
        lambda: ops.paged_attn_tree(q, kv, ints(2, 4), s, i, None, 4, 1, 2, out=far(2, 512, torch.bfloat16)),
        lambda: ops.constrain(far(2, 8, torch.float32), starts=s),
        lambda: ops.constrain(torch.zeros(2, 8), starts=s, history=big, hist_starts=s),
        lambda: ops.constrain(torch.zeros(2, 8), starts=s, allow=far(2, 1, torch.int32)),
        lambda: ops.constrain(torch.zeros(2, 8), starts=s, out=far(2, 8, torch.float32)),
        lambda: ops.tree_accept(i, i, None, s, i, far(2, 4, torch.int32), None, 2),
        lambda: ops.tree_accept(big, big, None, s, i, ints(2, 4), None, 2),
    ]
    for k, call in enumerate(calls):
        with pytest.raises(B200Error, match="32 bits"):
            call()
            pytest.fail(f"call {k} was taken")
