"""Requests that step_maps turns away, in the operations behind it: nothing of theirs is written, and nothing of anybody else's."""
import numpy as np
import pytest
import torch

import tree_step_util as U
from test_tree_step_gpu import ints

pytestmark = pytest.mark.gpu

HEADS, KVH, V = 8, 2, 300
#      ctx, rows, held, table (what lies behind the pages held was another request's, or never anybody's)
STAYS = (20, 6, 2, [4, 5, 0, 0])
CASES = {"too few pages": ((16, 4, 1, [1, 4, 5, 0]), 1), "fewer pages held than tokens": ((33, 3, 2, [1, 2, 4, 5]), 2), "more rows than masks have bits": ((0, 40, 0, [4, 5, 4, 5]), 2),
         "negative length": ((-1, 2, 1, [4, 5, 0, 0]), 2)}


def step(x, state):
    """maps, attention, the choice and acceptance on `state`, whose lengths, tables and cache they read and write."""
    from kubeai_b200 import ops
    m = ops.step_maps(state["ctx"], x["new"], state["held"], state["tables"], x["free"], state["cursor"], x["T"], parents=x["parents"], words=1, inplace=True)
    y = ops.paged_attn_tree(x["qkv"], state["kv"][0], state["tables"], m.starts, state["ctx"], m.masks, HEADS, KVH, 32, status=m.status)
    kept = torch.full((x["T"], HEADS * 128), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attn_tree(x["qkv"], state["kv"][0], state["tables"], m.starts, state["ctx"], m.masks, HEADS, KVH, 32, out=kept, status=m.status)
    logits = torch.full((x["T"], V), 9.0, device="cuda")
    ids, _ = ops.constrain(x["logits"], starts=m.starts, drafts=x["drafts"], masks=m.masks, penalties=x["penalties"], out=logits, status=m.status)
    a = ops.tree_accept(ids, x["drafts"], x["parents"], m.starts, state["ctx"], state["tables"], state["kv"], 8, status=m.status)
    return dict(m=m, y=y, kept=kept, ids=ids, logits=logits, a=a)


def inputs(away, flag, first):
    """The request that stays and the one that is turned away, in this order or the other; some rows of nobody behind them."""
    both = [STAYS, away] if first else [away, STAYS]
    rows, me = [max(r[1], 0) for r in both], 0 if first else 1
    T = sum(rows) + 3
    rng, g = np.random.default_rng(4), torch.Generator().manual_seed(4)
    at = sum(rows[:me])
    parents = np.concatenate([U.random_tree(rng, n) for n in rows] + [[-1] * 3])
    parents[at:at + 6] = [-1, 0, 0, 1, 2, 4]
    drafts = rng.integers(0, 50, T)
    logits = torch.randn(T, V, generator=g)
    for row in range(T):                       # every row's choice is what its last child drafts
        for j in range(row + 1, T):
            s = next((k for k in range(2) if sum(rows[:k]) <= row and j < sum(rows[:k + 1])), None)
            if s is not None and parents[j] == row - sum(rows[:s]):
                logits[row, drafts[j]] = 50.0 + j
    x = dict(new=ints([r[1] for r in both]), free=ints([3]) if flag == 1 else ints([3, 6, 7]), T=T, parents=ints(parents), drafts=ints(drafts), logits=logits.cuda(),
             penalties=torch.tensor([[1.1, 0.2, 0.1]] * 2).cuda(), qkv=torch.randn(T, (HEADS + 2 * KVH) * 128, generator=g).bfloat16().cuda())
    # (16 pages that nobody has the first of: page 0 of a stale table is another request's all the same)
    state = dict(ctx=ints([r[0] for r in both]), held=ints([r[2] for r in both]), tables=ints([r[3] for r in both]), cursor=ints([1 if flag == 1 else 0]),
                 kv=torch.randn(2, 8, 2, KVH, 16, 128, generator=g).bfloat16().cuda())
    return x, state, me, at


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("name", CASES)
def test_a_request_that_is_turned_away_touches_nothing(name, first):
    away, flag = CASES[name]
    x, state, me, at = inputs(away, flag, first)
    other, before = 1 - me, {k: v.clone() for k, v in state.items()}
    # the same step in which the other request brings no rows, its own behind everybody's
    lone, alone = dict(x), {k: v.clone() for k, v in state.items()}
    lone["new"] = x["new"].clone()
    lone["new"][other] = 0
    alone["ctx"][other], alone["held"][other] = 0, 0
    pick = torch.cat([torch.arange(at, at + 6), torch.tensor([t for t in range(x["T"]) if not at <= t < at + 6])]).cuda()
    for k in ("parents", "drafts", "logits", "qkv"):
        lone[k] = x[k][pick].contiguous()
    want = step(lone, alone)
    # the step itself, captured and replayed
    eager = step(x, {k: v.clone() for k, v in before.items()})
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = step(x, state)
    for _ in range(2):
        for k, v in before.items():
            state[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for out in (got, eager):
            m, a, mine = out["m"], out["a"], torch.zeros(x["T"], dtype=torch.bool, device="cuda")
            mine[at:at + 6] = True
            assert m.status.tolist() == [0 if s == me else flag for s in range(2)]
            assert a.accepted[other] == 0 and (a.path[other] == -1).all() and (a.tokens[other] == -1).all() and a.ctx_lens[other] == away[0] and m.held[other] == away[2]
            assert (out["y"][~mine] == 0).all() and (out["kept"][~mine] == 5).all() and (out["ids"][~mine] == -1).all() and (out["logits"][~mine] == 9).all()
            # the other request: as without it
            assert a.accepted[me] == want["a"].accepted[me] and a.accepted[me] > 2
            for k in ("path", "tokens", "ctx_lens"):
                assert torch.equal(getattr(a, k)[me], getattr(want["a"], k)[me])
            assert torch.equal(out["y"][mine], want["y"][:6]) and torch.equal(out["kept"][mine], out["y"][mine])
            assert torch.equal(out["ids"][mine], want["ids"][:6]) and torch.equal(out["logits"][mine], want["logits"][:6])
        assert torch.equal(state["kv"].view(torch.int16), alone["kv"].view(torch.int16))
        assert torch.equal(state["tables"][other], before["tables"][other])
    changed = (state["kv"].view(torch.int16) != before["kv"].view(torch.int16)).any(-1).any(3).any(2).any(0)      # [pages, 16]
    assert changed.any() and not changed[[p for p in range(8) if p not in (4, 5, 3)]].any()


def test_rows_of_requests_that_are_turned_away_among_many():
    """Zeros in a new output, in rows of some of many requests and behind the last."""
    from kubeai_b200 import ops
    rng = np.random.default_rng(8)
    S = 300
    rows = [int(n) for n in rng.integers(0, 9, S)]
    T, starts = sum(rows) + 40, np.concatenate([[0], np.cumsum(rows)])
    status = rng.choice([0, 0, 4, 1, 2, 5], S)
    qkv, kv = torch.randn(T, 6 * 128, device="cuda").bfloat16(), torch.randn(50, 2, 1, 16, 128, device="cuda").bfloat16()
    tables, ctx = ints(rng.integers(0, 50, (S, 5))), ints(rng.integers(1, 60, S))
    torch.full((T, 512), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = ops.paged_attn_tree(qkv, kv, tables, ints(starts), ctx, None, 4, 1, 8, status=ints(status))
    gone = torch.ones(T, dtype=torch.bool)
    for s in range(S):
        gone[starts[s]:starts[s + 1]] = bool(status[s] & 3)
    assert (got.cpu()[gone] == 0).all()
    # the others as in a call that is told of no status (how the work is cut differs, and with it the last bit of some)
    whole = ops.paged_attn_tree(qkv, kv, tables, ints(starts), ctx, None, 4, 1, 8)
    off = (got.cpu()[~gone].double() - whole.cpu()[~gone].double()).abs()
    # in both forms weights that sum to 1 are rounded to bf16, on values below 6 and in their sum, and the result
    assert (off <= 2 * 2.0 ** -8 * (6 + 2 * whole.cpu()[~gone].double().abs())).all() and whole.cpu()[~gone].any(1).all()


def test_a_status_that_is_not_the_requests_is_refused():
    from kubeai_b200 import B200Error, ops
    i, s, t = ints([1, 1]), ints([0, 1, 2]), ints([[0], [0]])
    q, kv = torch.zeros(2, 512, device="cuda", dtype=torch.bfloat16), torch.zeros(1, 2, 1, 16, 128, device="cuda", dtype=torch.bfloat16)
    for bad in (ints([0]), ints([0, 0, 0]), i.long(), i.cpu()):
        with pytest.raises(B200Error):
            ops.paged_attn_tree(q, kv, t, s, i, None, 4, 1, 1, status=bad)
        with pytest.raises(B200Error):
            ops.constrain(torch.zeros(2, 8, device="cuda"), starts=s, status=bad)
        with pytest.raises(B200Error):
            ops.tree_accept(i, i, None, s, i, t, None, 2, status=bad)
