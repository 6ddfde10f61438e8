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
