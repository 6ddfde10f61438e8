"""The operations on drafted trees where lists are long, requests many and lengths at their ends; calls side by side, captured, and again on what they wrote."""
import numpy as np
import pytest
import torch

import tree_step_util as U
from test_tree_step_gpu import (accept_case, attention_case, check_attention, check_constrain, check_maps, constrain_case, ints, run_attention, run_constrain)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ maps
def test_maps_give_no_slot_on_pages_that_cannot_be():
    from kubeai_b200 import ops
    tables = ints([[5, -1, (1 << 27) - 2, (1 << 27) - 1, 1 << 27, (1 << 31) - 1]])
    m = ops.step_maps(ints([0]), ints([96]), ints([6]), tables, ints([]), ints([0]), 96, words=3)
    page = lambda n: [n * 16 + i for i in range(16)]       # noqa: E731
    assert m.slots.tolist() == page(5) + [-1] * 16 + page((1 << 27) - 2) + [-1] * 48 and m.status.tolist() == [0]
    m = ops.step_maps(ints([16]), ints([2]), ints([1]), ints([[3, 0]]), ints([-5]), ints([0]), 2)
    assert m.slots.tolist() == [-1, -1]


def test_maps_again_and_again_in_place():
    """What one call writes the next one reads, while a batch grows."""
    from kubeai_b200 import ops
    rng = np.random.default_rng(3)
    S, width, free = 37, 9, rng.permutation(200)
    ctx, held, tables, cursor = [0] * S, [0] * S, np.full((S, width), -1), 0
    d_held, d_tables, d_cursor, d_free = ints(held), ints(tables), ints([0]), ints(free)
    for step in range(12):
        new = [int(n) for n in rng.integers(0, 18, S)]
        rows = sum(new) + step
        parents = sum((U.random_tree(rng, n) for n in new), []) + [-1] * step
        want = U.maps(ctx, new, held, tables, free, cursor, rows, parents, 1)
        got = ops.step_maps(ints(ctx), ints(new), d_held, d_tables, d_free, d_cursor, rows, parents=ints(parents), words=1, inplace=True)
        for name in ("starts", "positions", "slots", "seqs", "status", "held"):
            assert getattr(got, name).tolist() == list(want[name]), (step, name)
        tables, held, cursor = want["tables"], want["held"], want["cursor"]
        assert np.array_equal(d_tables.cpu().numpy(), tables) and d_cursor.tolist() == [cursor]
        ctx = [c + int(rng.integers(0, n + 1)) if n and not f else c for c, n, f in zip(ctx, new, want["status"])]


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("S,kv_heads,group,masks", [(1, 8, 8, "tree"), (300, 2, 4, "random"), (600, 1, 1, "chain"), (257, 1, 8, "tree"), (90, 3, 2, "random")])
def test_attention_of_many_requests(S, kv_heads, group, masks):
    """More requests than threads, ranges of many items, ranges that share one."""
    rng = np.random.default_rng(S)
    ctx = [int(n) for n in rng.choice([0, 1, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129], S)]
    rows = [int(n) for n in rng.choice([0, 1, 2, 5, 17, 33], S)]
    ctx[S // 2], rows[S // 2], rows[0] = 4000, 40, 2
    c = attention_case(S, ctx, rows, kv_heads, group, masks)
    a = run_attention(c)
    check_attention(c, a)
    check_attention(c, run_attention(c, max_ctx=1))       # lengths that were not known


@pytest.mark.parametrize("rows,group,masks", [(600, 8, "chain"), (256, 8, "random"), (900, 1, "chain"), (129, 2, "tree"), (1024, 2, "chain")])
def test_attention_of_blocks_of_rows(rows, group, masks):
    c = attention_case(rows, [333, 0], [rows, min(rows, 200)], 2, group, masks)
    check_attention(c, run_attention(c))


@pytest.mark.parametrize("n", [1, 2, 47, 48, 49, 191, 192, 193, 320])
def test_attention_where_ranges_end_by_an_items_ends(n):
    """Contexts whose tiles divide into ranges with and without a remainder."""
    c = attention_case(n, [64 * n - 3, 64 * (n // 2 + 1)], [2, 3], 4, 4)
    check_attention(c, run_attention(c))


def test_attention_of_large_scores():
    """Maxima that move by more than the slack from tile to tile, up and down, and scores far below them."""
    c = attention_case(21, [700, 260], [9, 30], 2, 4)
    rng = np.random.default_rng(21)
    for p in range(c["kv"].shape[0]):
        c["kv"][p, 0] *= float(rng.choice([0.01, 1.0, 5.0, 20.0]))
    check_attention(c, run_attention(c))


@pytest.mark.parametrize("extra,ctx", [(1, [40, 70, 3]), (700, [40, 70, 3]), (2900, [40, 1 << 20, 3]), (15, [-1, 70, 3])])
def test_attention_of_a_padded_batch_is_zero_in_rows_that_nobody_owns(extra, ctx):
    """Behind the last request, and those of requests whose lengths are none, in a new output over memory that held something else."""
    from kubeai_b200 import ops
    c = attention_case(50, [40, 70, 3], [10, 21, 30], 2, 4, extra=extra)
    torch.full((c["T"] + extra, c["heads"] * 128), float("nan"), dtype=torch.bfloat16, device="cuda")      # given back at once: what the output is likely to lie on
    got = ops.paged_attn_tree(c["qkv"].cuda(), c["kv"].cuda(), ints(c["tables"]), ints(c["starts"]), ints(ctx), ints(c["bits"]), c["heads"], c["kv_heads"], 30)
    whole = run_attention(c)
    assert (got[c["T"]:] == 0).all() and (whole[c["T"]:] == 0).all()
    for s in range(3):
        rows = slice(c["starts"][s], c["starts"][s + 1])
        if ctx[s] == c["ctx"][s]:
            whole[rows] = got[rows]
        else:
            assert (got[rows] == 0).all()
    check_attention(c, whole)


# ------------------------------------------------------------------ constrain
@pytest.mark.parametrize("rows,V,history,f32", [([1], 128256, 60000, False), ([1], 393216, 200000, True), ([3, 9], 50021, 30000, True), ([70, 70], 20011, 9000, False)])
def test_constrain_with_more_marked_tokens_than_slots(rows, V, history, f32):
    c = constrain_case(V, rows, V, [history] * len(rows), f32, 500, "some" if sum(rows) < 20 else None, "tree")
    check_constrain(c, *run_constrain(c, out=torch.float32))
    ids, none = run_constrain(c)
    check_constrain(c, ids)
    here = c | dict(x=c["x"].cuda())                         # and in place, where pieces follow one another
    again, y = run_constrain(here, out=here["x"])
    assert y is here["x"] and torch.equal(ids, again)
    check_constrain(c, again, y)


def test_constrain_with_every_token_marked():
    for V in (4096, 4097, 8192, 12345):
        c = constrain_case(V, [2, 1], V, [V, 3], True, 3, "some", "chain")
        c["said"][0] = [int(t) for t in np.random.default_rng(V).permutation(V)]
        c["prompt"][0] = V // 2
        check_constrain(c, *run_constrain(c, out=torch.float32))


def test_constrain_of_biases_that_come_twice():
    """More biases than threads, tokens several times over: the last one counts."""
    c = constrain_case(31, [4, 1, 2], 700, [20, 0, 300], True, 2000, None, "tree")
    check_constrain(c, *run_constrain(c, out=torch.float32))
    c = constrain_case(32, [1, 1], 60001, [20, 0], False, 257, "few", None)
    check_constrain(c, *run_constrain(c, out=torch.float32))


@pytest.mark.parametrize("n", [256, 257, 700])
def test_constrain_of_long_chains(n):
    """A chain's rows see more drafts than a CTA has threads."""
    c = constrain_case(n, [n, 3], 331, [40, 0], True, 5, None, "chain")
    check_constrain(c, *run_constrain(c, out=torch.float32))


@pytest.mark.parametrize("S,V", [(700, 5001), (2500, 129), (300, 33000)])
def test_constrain_of_many_requests(S, V):
    rng = np.random.default_rng(S)
    rows = [int(n) for n in rng.choice([0, 1, 1, 2, 5], S)]
    c = constrain_case(S, rows, V, [int(n) for n in rng.integers(0, 40, S)], False, 2, None, "tree")
    check_constrain(c, run_constrain(c)[0])


# ------------------------------------------------------------------ accept
def test_accept_of_more_requests_than_places():
    from kubeai_b200 import ops
    rng = np.random.default_rng(5)
    S = 3000
    c = accept_case(5, [int(n) for n in rng.integers(0, 40, S)], [int(n) for n in rng.integers(0, 12, S)], 2, 1)
    want = U.accepted(c["ids"], c["drafts"], c["parents"], c["starts"], c["ctx"], c["tables"], c["kv"].view(torch.int16).numpy(), 6)
    kv = c["kv"].cuda()
    got = ops.tree_accept(ints(c["ids"]), ints(c["drafts"]), ints(c["parents"]), ints(c["starts"]), ints(c["ctx"]), ints(c["tables"]), kv, 6)
    for name in ("accepted", "path", "tokens", "ctx_lens"):
        assert getattr(got, name).tolist() == want[name], name
    assert np.array_equal(kv.cpu().view(torch.int16).numpy(), want["kv"])


def test_accept_far_into_a_large_cache():
    """Layers and pages behind 2^31 values and 2^32 bytes."""
    from kubeai_b200 import ops
    c = accept_case(12, [10, 3], [30, 30], 2, 2)
    want = U.accepted(c["ids"], c["drafts"], c["parents"], c["starts"], c["ctx"], c["tables"], c["kv"].view(torch.int16).numpy(), 16)
    assert max(want["accepted"]) > 1
    big = torch.zeros(2, 140000, 2, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
    at = np.array([139999 - 37 * i for i in range(c["kv"].shape[1])])
    big[:, torch.tensor(at).cuda()] = c["kv"].cuda()
    got = ops.tree_accept(ints(c["ids"]), ints(c["drafts"]), ints(c["parents"]), ints(c["starts"]), ints(c["ctx"]), ints(at[np.maximum(c["tables"], 0)]), big, 16)
    assert got.path.tolist() == want["path"]
    assert np.array_equal(big[:, torch.tensor(at).cuda()].cpu().view(torch.int16).numpy(), want["kv"])


def test_constrain_far_into_many_rows():
    """Rows behind 2^31 values and 2^32 bytes, in place."""
    from kubeai_b200 import ops
    T, V = 17000, 128256
    x = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    x[T - 1, 100000], x[T - 1, 77], x[T - 2, 128255], x[0, 5] = 2.0, 1.0, 1.0, 1.0
    starts = np.zeros(T + 1, dtype=np.int64)
    starts[T] = 1
    ids, y = ops.constrain(x, bias=(ints(starts), ints([77]), torch.tensor([5.0]).cuda()), out=x)
    ids = ids.tolist()
    assert y is x and ids[T - 1] == 77 and ids[T - 2] == 128255 and ids[0] == 5 and not any(ids[1:T - 2])
    assert x[T - 1, 77] == 6 and x[T - 1, 100000] == 2 and x[T - 2].sum() == 1 and x[T // 2].abs().sum() == 0


# ------------------------------------------------------------------ graphs, streams, devices
def test_two_graphs_replayed_at_once():
    """Each graph has its own workspace: side by side they give what they give alone."""
    from kubeai_b200 import ops
    cases = [attention_case(40 + i, [3000, 20 + i], [30, 64], 2, 4) for i in range(2)]
    alone = [run_attention(c) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    inputs = [(c["qkv"].cuda(), c["kv"].cuda(), ints(c["tables"]), ints(c["starts"]), ints(c["ctx"]), ints(c["bits"])) for c in cases]
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(ops.paged_attn_tree(*inputs[i], 8, 2, 64))
        graphs.append(g)
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for a, b in zip(alone, outs):
        assert torch.equal(a, b)


def test_tensors_that_are_not_laid_out_as_asked_are_refused():
    from kubeai_b200 import B200Error, ops
    i = ints([1, 1])
    wide = ints(np.zeros((4, 4)))
    kv = torch.zeros(4, 2, 1, 16, 128, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(2, 512, device="cuda", dtype=torch.bfloat16)
    s = ints([0, 1, 2])
    bad = [
        lambda: ops.step_maps(wide[:2, 0], i, i, wide[:2], i, ints([0]), 2),                              # lengths with strides
        lambda: ops.step_maps(i, i, i, wide[:2].t(), i, ints([0]), 2),                                    # tables by columns
        lambda: ops.step_maps(i, i, i.long(), wide[:2], i, ints([0]), 2),
        lambda: ops.step_maps(i, i, i, wide[:2], i, ints([0]).cpu(), 2),
        lambda: ops.paged_attn_tree(q, kv.transpose(1, 2), wide[:2], s, i, None, 4, 1, 1),
        lambda: ops.paged_attn_tree(q, kv[:, :, :, :, :64], wide[:2], s, i, None, 4, 1, 1),
        lambda: ops.paged_attn_tree(q.t(), kv, wide[:2], s, i, None, 4, 1, 1),
        lambda: ops.paged_attn_tree(q[:, :384], kv, wide[:2], s, i, None, 4, 1, 1),
        lambda: ops.paged_attn_tree(q, kv, wide[:2], s, i, wide[:2, ::2], 4, 1, 1),
        lambda: ops.paged_attn_tree(q, kv, wide[:2], s, i, None, 4, 1, 1, scale=-0.1),
        lambda: ops.constrain(torch.zeros(8, 2, device="cuda").t()),
        lambda: ops.constrain(torch.zeros(2, 8, device="cuda", dtype=torch.float16)),
        lambda: ops.constrain(torch.zeros(2, 8, device="cuda"), starts=s, penalties=torch.ones(2, 6, device="cuda")[:, ::2]),
        lambda: ops.constrain(torch.zeros(2, 8, device="cuda"), out=torch.zeros(2, 8)),
        lambda: ops.tree_accept(i, i, None, s, i, wide[:2], torch.zeros(2, 4, 2, 1, 128, 16, device="cuda", dtype=torch.bfloat16).transpose(4, 5), 2),
        lambda: ops.tree_accept(i, i, None, s, i, wide[:2], kv, 2),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(B200Error):
            call()
            pytest.fail(f"call {k} was taken")
