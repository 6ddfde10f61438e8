"""Penalties in steps whose rows carry a part of the prompt: its tokens are the prompt's, whether a request's history has them or its rows."""
import numpy as np
import pytest
import torch

import tree_step_util as U
from test_tree_step_gpu import ints

pytestmark = pytest.mark.gpu


def case(seed, rows, history, prompt, V, tree, low):
    rng = np.random.default_rng(seed)
    T = sum(rows)
    starts = [0, *np.cumsum(rows).tolist()]
    see = [U.ancestors(U.random_tree(rng, n)) if tree else np.tril(np.ones((n, n), dtype=bool)) for n in rows]
    for s, n in enumerate(rows):             # a prompt's rows are a chain that the drafts hang on
        k = min(n, max(0, prompt[s] - history[s]))
        if tree and k:
            see[s] = U.ancestors([*range(-1, k - 1), *(int(rng.integers(k - 1, i)) for i in range(k, n))])
    return dict(rows=rows, starts=starts, see=see, V=V, tree=tree, prompt=prompt, said=[[int(t) for t in rng.integers(0, low, h)] for h in history],
                drafts=[int(t) for t in rng.integers(0, low, T)], x=torch.randn(T, V, generator=torch.Generator().manual_seed(seed)) * 3,
                penalties=np.stack([rng.choice([1.1, 1.3], len(rows)), rng.choice([0.5, -0.3], len(rows)), rng.choice([0.3, 0.01], len(rows))], 1).astype(np.float32))


def run(c):
    from kubeai_b200 import ops
    words = -(-max(c["rows"]) // 32)
    return ops.constrain(c["x"].cuda(), starts=ints(c["starts"]), history=ints(sum(c["said"], [])), hist_starts=ints([0, *np.cumsum([len(h) for h in c["said"]])]), prompt_lens=ints(c["prompt"]),
                         drafts=ints(c["drafts"]), masks=ints(np.concatenate([U.pack(m, words) for m in c["see"]])) if c["tree"] else None, penalties=torch.tensor(c["penalties"]).cuda(), out=torch.float32)


def want(c):
    """Every row as a request of its own, whose text is its request's and what leads to it, the prompt's in front."""
    said, prompt, penalties = [], [], []
    for s, n in enumerate(c["rows"]):
        for i in range(n):
            text = [(k < c["prompt"][s], t) for k, t in enumerate(c["said"][s])] + [(len(c["said"][s]) + j < c["prompt"][s], c["drafts"][c["starts"][s] + j]) for j in np.flatnonzero(c["see"][s][i])]
            said.append([t for p, t in text if p] + [t for p, t in text if not p])
            prompt.append(sum(p for p, _ in text))
            penalties.append(c["penalties"][s])
    T = len(said)
    return U.constrained(c["x"].numpy(), [[r] for r in range(T)], said, prompt, None, [np.ones((1, 1))] * T, np.array(penalties), [[]] * T, np.ones((T, c["V"]), dtype=bool))


@pytest.mark.parametrize("rows,history,prompt,V,tree,low", [
    ([1], [0], [1], 40, False, 8), ([5], [0], [5], 40, False, 4), ([5], [0], [3], 40, True, 4), ([8, 8, 8], [10, 0, 7], [14, 100, 3], 500, False, 12), ([30, 1, 33], [40, 3, 0], [60, 4, 20], 500, True, 12),
    ([256], [9], [150], 300, True, 20), ([700, 3], [50, 0], [400, 2], 331, False, 60), ([40, 60], [0, 9000], [20, 9030], 20011, False, 20011), ([64, 30], [9000, 0], [9040, 0], 20011, True, 20011)])
def test_rows_of_a_prompt_count_as_prompt(rows, history, prompt, V, tree, low):
    c = case(V + sum(rows), rows, history, prompt, V, tree, low)
    ids, y = run(c)
    logits, choices = want(c)
    assert ids.tolist() == choices.tolist() and np.array_equal(y.cpu().numpy(), logits)


def test_a_prompt_in_portions_gives_the_choice_of_one_in_the_history():
    c = case(3, [1], [50], [51], 2000, False, 40)
    c["x"] = c["x"].expand(1, -1).contiguous()
    ids, y = run(c)
    for cut in (0, 1, 20, 49):
        n = 51 - cut
        d = c | dict(rows=[n], starts=[0, n], said=[c["said"][0][:cut]], drafts=c["said"][0][cut:] + c["drafts"], x=c["x"].expand(n, -1).contiguous(), see=[np.tril(np.ones((n, n), dtype=bool))])
        for tree in (False, True):
            got, z = run(d | dict(tree=tree))
            assert got[-1] == ids[0] and torch.equal(z[-1], y[0])
