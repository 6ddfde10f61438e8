"""Logits whose rows begin and end off the 16 bytes of a copy, one behind the other through the same few buffers."""
import pytest
import torch

from test_tree_step_gpu import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,ld", [(8, 9), (13, 13), (37, 41), (8191, 8193), (8200, 8201), (16397, 16399)])
def test_ragged_rows_follow_one_another(V, ld, dtype):
    """The same bytes of a buffer are a thread's store for one row and a copy's for another."""
    from kubeai_b200 import ops
    rows = 2000 if V < 1000 else 300
    g = torch.Generator(device="cuda").manual_seed(V)
    wide = torch.randint(-1000, 1000, (rows, ld), generator=g, device="cuda").to(dtype)
    x = wide[:, :V]
    best = x.float().amax(1, keepdim=True)
    want = torch.where(x.float() == best, torch.arange(V, device="cuda"), V).amin(1)
    for _ in range(5):
        ids, y = ops.constrain(x, starts=ints([0, rows]), out=dtype)
        assert torch.equal(ids.long(), want) and torch.equal(y, x)
