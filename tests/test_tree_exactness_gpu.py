"""Attention of drafted trees against the same steps in 64 bits, as the kernels of prompt attention are: weights relative to the largest score met so far, which makes
the largest weight exactly 1, rounded to bf16, divided by the rounded weights' sum, and the output rounded to bf16.  Those two roundings are all that a result may be off
by.  (An item of which several ranges have parts has such a largest weight in each, which rounds no worse.)"""
import math

import numpy as np
import pytest
import torch

import tree_step_util as U
from test_attention_exactness_gpu import DEV, bf, check

pytestmark = pytest.mark.gpu


def attention(q, k, v, see, scale):
    """q [rows, heads, 128], k and v [keys, kv heads, 128] in 64 bits, see [rows, keys] -> the exact result and the one with the two roundings."""
    rows, heads = q.shape[:2]
    keys = k.shape[0]
    tiles = -(-keys // 64)
    exact, rounded = torch.empty_like(q), torch.empty_like(q)
    for h in range(heads):
        kv = h * k.shape[1] // heads
        s = (q[:, h] @ k[:, kv].T * scale).masked_fill(~see, -math.inf)
        exact[:, h] = torch.softmax(s, 1) @ v[:, kv]
        pad = torch.nn.functional.pad(s, (0, 64 * tiles - keys), value=-math.inf).reshape(rows, tiles, 64)
        ref = pad.amax(2).cummax(1).values.clamp_min(-1e300)                # the largest score up to each tile of 64 keys
        pr = bf(torch.exp(pad - ref[:, :, None]).float()).double() * torch.exp(ref - s.amax(1, keepdim=True))[:, :, None]
        rounded[:, h] = bf((pr.reshape(rows, -1)[:, :keys] @ v[:, kv] / pr.sum((1, 2))[:, None]).float()).double()
    return exact, rounded


@pytest.mark.parametrize("ctx,rows,tree", [(448, 64, True), (60, 640, False), (2000, 200, True), (1937, 64, False)])
@pytest.mark.parametrize("deviation", [1, 2, 4, 8])
def test_trees(ctx, rows, tree, deviation):
    from kubeai_b200 import ops
    kv_heads, group, requests = 2, 4, 4
    heads, n = kv_heads * group, ctx + rows
    g = torch.Generator(device=DEV).manual_seed(n + deviation)
    pages = -(-n // 16)
    order = torch.randperm(requests * pages, generator=g, device=DEV).reshape(requests, pages)
    kv = bf(torch.randn(requests * pages, 2, kv_heads, 16, 128, generator=g, device=DEV))
    q = bf(torch.randn(requests * rows, heads * 128, generator=g, device=DEV)) * deviation           # a power of two: exact
    sees = [U.ancestors(U.random_tree(np.random.default_rng(s), rows)) if tree else np.tril(np.ones((rows, rows), dtype=bool)) for s in range(requests)]
    masks = torch.tensor(np.concatenate([U.pack(see, 8) for see in sees])).to(DEV) if tree else None
    starts = torch.arange(0, requests * rows + 1, rows, dtype=torch.int32, device=DEV)
    got = ops.paged_attn_tree(q, kv, order.to(torch.int32), starts, torch.full((requests,), ctx, dtype=torch.int32, device=DEV), masks, heads, kv_heads, rows)
    parts = []
    for s, see in enumerate(sees):
        k, v = kv[order[s]].permute(1, 0, 3, 2, 4).reshape(2, pages * 16, kv_heads, 128)[:, :n].double()
        see = torch.cat([torch.ones(rows, ctx, dtype=torch.bool), torch.tensor(see)], 1).to(DEV)
        parts.append(attention(q[s * rows:(s + 1) * rows].reshape(rows, heads, 128).double(), k, v, see, 128 ** -0.5))
    check(got.reshape(-1, heads, 128), torch.cat([a for a, _ in parts]), torch.cat([b for _, b in parts]))
