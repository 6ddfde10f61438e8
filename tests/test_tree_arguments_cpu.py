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
