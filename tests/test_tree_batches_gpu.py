"""Constrained choice over more rows of a request than a CTA holds the choices of, and over as many as a step may have."""
import numpy as np
import pytest
import torch

from test_tree_step_gpu import ints

pytestmark = pytest.mark.gpu

DEV = "cuda"


def lowest_best(y):
    return torch.where(y == y.amax(1, keepdim=True), torch.arange(y.shape[1], device=DEV), y.shape[1]).amin(1)


@pytest.mark.parametrize("V,said", [(40, 30), (6000, 9000)])
def test_a_chain_among_many_requests(V, said):
    """300 requests of which one has 70000 rows: a launch has no room for 256 rows a CTA of every one.  (6000 tokens that are all named: more than a CTA has slots.)"""
    from kubeai_b200 import ops
    S, long, many, dtype = 300, 17, 70000, torch.bfloat16
    rng = np.random.default_rng(V)
    rows = [1] * S
    rows[long] = many
    T, starts = sum(rows), np.concatenate([[0], np.cumsum(rows)])
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn(T, V, generator=g, device=DEV) * 3).to(dtype)
    history = rng.integers(0, V // 2, said) if V < said else rng.integers(0, V, said)
    if V > 4096:
        history[-V:] = rng.permutation(V)
    hist_starts = [0] * (long + 1) + [said] * (S - long)
    drafts = ints(rng.integers(0, V, T))
    rho, pi, phi = 1.25, 0.5, 0.25
    pen = torch.ones(S, 3, device=DEV) * torch.tensor([1.0, 0.0, 0.0], device=DEV)
    pen[long] = torch.tensor([rho, pi, phi], device=DEV)
    out = torch.empty_like(x)
    ids, y = ops.constrain(x, starts=ints(starts), history=ints(history), hist_starts=ints(hist_starts), prompt_lens=ints([said // 3] * S), drafts=drafts, penalties=pen, out=out)
    a, b = int(starts[long]), int(starts[long + 1])
    others = torch.ones(T, dtype=torch.bool, device=DEV)
    others[a:b] = False
    # the other requests have neither penalties nor anything else
    assert torch.equal(y[others], x[others]) and torch.equal(ids[others].long(), lowest_best(x[others].float()))
    prompt = torch.zeros(V, dtype=torch.bool, device=DEV)
    prompt[torch.tensor(history[:said // 3], device=DEV)] = True
    base = torch.bincount(torch.tensor(history[said // 3:], device=DEV), minlength=V).int()
    f = lambda v: torch.full((), v, device=DEV)      # noqa: E731
    for r0 in range(a, b, 5000):                      # the chain so far, and what these rows add to it
        r1 = min(b, r0 + 5000)
        own = torch.zeros(r1 - r0, V, dtype=torch.int32, device=DEV).scatter_(1, drafts[r0:r1, None].long(), 1).cumsum(0, dtype=torch.int32)
        count = own + base
        base = count[-1].clone()
        z = x[r0:r1].float()
        z = torch.where((count > 0) | prompt, torch.where(z > 0, z / f(rho), z * f(rho)), z)
        z = z - f(phi) * count.float()
        z = torch.where(count > 0, z - f(pi), z)
        assert torch.equal(ids[r0:r1].long(), lowest_best(z)), r0
        assert torch.equal(y[r0:r1], z.to(dtype)), r0


def test_as_many_rows_as_pass_a_launch_of_256_each():
    from kubeai_b200 import ops
    T = 65536 * 256 + 77
    x = torch.randint(-100, 100, (T, 8), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    want = lowest_best(x.float())
    ids, none = ops.constrain(x, starts=ints([0, T]))
    assert none is None and torch.equal(ids.long(), want)
    ids, none = ops.constrain(x, starts=ints([0, 5, T - 3, T]))
    assert torch.equal(ids.long(), want)


@pytest.mark.parametrize("S,rows", [(4096, 16), (2000, 40)])
def test_many_requests_of_many_rows(S, rows):
    from kubeai_b200 import ops
    x = torch.randint(-100, 100, (S * rows, 65), generator=torch.Generator(device=DEV).manual_seed(S), device=DEV).float()
    ids, none = ops.constrain(x, starts=torch.arange(0, S * rows + 1, rows, dtype=torch.int32, device=DEV))
    assert torch.equal(ids.long(), lowest_best(x))
