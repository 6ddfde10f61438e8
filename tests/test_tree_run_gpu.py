"""The operations on drafted trees as they are used: steps of a small model over a paged cache, one behind the other, captured into a graph and on streams side by side."""
import threading

import numpy as np
import pytest
import torch

import tree_step_util as U

pytestmark = pytest.mark.gpu

HID, HEADS, KVH, VOCAB, LAYERS, PAGES, WIDTH, FF = 512, 8, 2, 500, 2, 64, 12, 1024


def ints(v):
    return torch.tensor(np.asarray(v, dtype=np.int64).astype(np.int32)).cuda()


def weights():
    g = torch.Generator().manual_seed(0)

    def w(n, k, scale=1.0):
        return (torch.randn(n, k, generator=g) * scale / k ** 0.5).bfloat16().cuda()

    ang = torch.arange(512)[:, None] * 10000.0 ** (-torch.arange(64)[None] / 64)
    one = torch.ones(HID, dtype=torch.bfloat16, device="cuda")
    return dict(embed=torch.randn(VOCAB, HID, generator=g).bfloat16().cuda(), head=w(VOCAB + 12, HID, 4.0), cos_sin=torch.cat([ang.cos(), ang.sin()], 1).bfloat16().cuda(), one=one,
                layers=[dict(qkv=w((HEADS + 2 * KVH) * 128, HID), o=w(HID, HEADS * 128), up=w(2 * FF, HID), down=w(HID, FF)) for _ in range(LAYERS)])


def forward(W, ids, m, tables, ctx, kv, masks, max_tree):
    from kubeai_b200 import ops
    res = ops.embed(W["embed"], ids)
    x = torch.zeros_like(res)
    for l, w in enumerate(W["layers"]):
        h = ops.rmsnorm(x, W["one"], 1e-5, residual=res)
        qkv = ops.gemm(h, w["qkv"])
        ops.rope_kvwrite(qkv, m.positions, m.slots, W["cos_sin"], kv[l], HEADS, KVH)
        x = ops.gemm(ops.paged_attn_tree(qkv, kv[l], tables, m.starts, ctx, masks, HEADS, KVH, max_tree), w["o"])
        h = ops.rmsnorm(x, W["one"], 1e-5, residual=res)
        x = ops.gemm(ops.silu_mul(ops.gemm(h, w["up"])), w["down"])
    return ops.gemm(ops.rmsnorm(x, W["one"], 1e-5, residual=res), W["head"])[:, :VOCAB]


class Requests:
    """A batch of conversations on the paged cache."""

    def __init__(self, W, prompts, allow):
        self.W, self.S = W, len(prompts)
        self.kv = torch.full((LAYERS, PAGES, 2, KVH, 16, 128), float("nan"), dtype=torch.bfloat16, device="cuda")      # nothing may read what no step wrote
        self.tables = ints(np.full((self.S, WIDTH), -1))
        self.held, self.cursor, self.ctx = ints([0] * self.S), ints([0]), ints([0] * self.S)
        self.free = ints(np.random.default_rng(3).permutation(PAGES))
        self.said = [[] for _ in prompts]
        self.prompt = [len(p) for p in prompts]
        self.allow = allow
        self.last = [int(v) for v in self.step([list(p) for p in prompts], None, prefill=True)]

    def step(self, rows, parents, prefill=False):
        from kubeai_b200 import ops
        n = [len(r) for r in rows]
        T, drafts = sum(n), ints(sum(rows, []))
        words = 0 if parents is None else 2
        flat = None if parents is None else ints(sum(parents, []))
        m = ops.step_maps(self.ctx, ints(n), self.held, self.tables, self.free, self.cursor, T, parents=flat, words=words, inplace=True)
        assert m.status.tolist() == [0] * self.S
        logits = forward(self.W, drafts, m, self.tables, self.ctx, self.kv, m.masks, max(n))
        counted = sum((self.said[s] for s in range(self.S)), [])
        ids, y = ops.constrain(logits, starts=m.starts, history=ints(counted), hist_starts=ints([0, *np.cumsum([len(h) for h in self.said])]), prompt_lens=ints(self.prompt),
                               drafts=drafts, masks=m.masks, penalties=torch.tensor([[1.3, 0.5, 0.25]] * self.S).cuda(), bias=(ints(range(self.S + 1)), ints([7] * self.S), torch.full((self.S,), -1.5).cuda()),
                               allow=self.allow, allow_rows=ints([0] * T), out=torch.float32)
        top = y.topk(2, dim=1).values
        self.margin = (top[:, 0] - top[:, 1]).tolist()
        if prefill:
            self.said = [list(r) for r in rows]
            self.ctx = self.ctx + ints(n)
            return [ids[sum(n[:s + 1]) - 1] for s in range(self.S)]
        a = ops.tree_accept(ids, drafts, flat, m.starts, self.ctx, self.tables, self.kv, 16)
        self.ctx = a.ctx_lens
        new = []
        for s in range(self.S):
            k, path = a.accepted[s].item(), a.path[s].tolist()
            self.said[s] += [rows[s][i] for i in path[:k]]
            new.append(a.tokens[s].tolist()[:k])
            self.last[s] = new[s][-1]
        assert self.ctx.tolist() == [len(h) for h in self.said]
        return new


@pytest.fixture(scope="module")
def W():
    return weights()


PROMPTS = [[int(v) for v in np.random.default_rng(5 + i).integers(0, VOCAB, n)] for i, n in enumerate((5, 17, 40))]


def allowed():
    mask = np.ones((1, VOCAB), dtype=bool)
    mask[0, 100:140] = False
    return ints(U.pack(mask, -(-VOCAB // 32)))


def test_drafted_trees_give_the_tokens_of_single_steps(W):
    one = Requests(W, PROMPTS, allowed())
    alone, sure = [[t] for t in one.last], [[True] for _ in PROMPTS]
    for _ in range(28):
        new = one.step([[t] for t in one.last], [[-1]] * 3)
        for s in range(3):
            alone[s] += new[s]
            sure[s].append(one.margin[s] > 0.25)       # closer ones may go the other way by the rounding of the products' bf16 results
    rng = np.random.default_rng(9)
    many = Requests(W, PROMPTS, allowed())
    assert many.last == [a[0] for a in alone]
    done, steps = [1] * 3, 0
    while min(done) < 20:
        rows, parents, right = [], [], []
        for s in range(3):
            told = alone[s][done[s]:done[s] + int(rng.integers(0, 5))]      # what the drafter gets right
            tree, drafts, on = [-1], [many.last[s]], [0]
            for t in told:
                for _ in range(int(rng.integers(0, 3))):                    # siblings and their children that are wrong
                    tree.append(int(rng.integers(0, len(tree))))
                    drafts.append(int(rng.integers(0, VOCAB)))
                tree.append(on[-1])
                on.append(len(drafts))
                drafts.append(t)
            rows.append(drafts), parents.append(tree), right.append(told)
        new = many.step(rows, parents)
        steps += 1
        for s in range(3):
            want = alone[s][done[s]:done[s] + len(new[s])]
            upto = next((k for k, t in enumerate(want) if not sure[s][done[s] + k]), len(want))
            assert new[s][:upto] == want[:upto], (s, done[s], new[s], want)
            if upto < len(want) and new[s] != want:
                pytest.fail(f"request {s}: a choice within rounding of another at token {done[s] + upto}; the tokens behind it cannot be compared")
            assert len(new[s]) > len(right[s]) or not all(sure[s][done[s]:done[s] + len(right[s])])
            done[s] += len(new[s])
    assert steps < 15 and not many.kv[:, many.tables[0, 0].long(), :, :, 0].isnan().any()


def test_a_step_captured_into_a_graph(W):
    from kubeai_b200 import ops
    S, T = 3, 24
    rng = np.random.default_rng(1)
    kv = torch.randn(LAYERS, PAGES, 2, KVH, 16, 128, device="cuda", dtype=torch.bfloat16)
    ctx, held, cursor = ints([30, 0, 100]), ints([2, 0, 7]), ints([9])
    tables = ints(np.concatenate([rng.permutation(9), np.full(S * WIDTH - 9, 63)]).reshape(S, WIDTH))
    tables[2, :7] = ints([3, 4, 5, 6, 7, 8, 62])
    free, new, parents, ids = ints(np.arange(PAGES)), ints([8, 8, 4]), ints([-1, 0, 0, 1, 2, 2, 3, 0] * 2 + [-1, 0, 1, 2] + [0] * 4), ints(rng.integers(0, VOCAB, T))

    def pass_over(state):
        m = ops.step_maps(state["ctx"], state["new"], state["held"], state["tables"], free, state["cursor"], T, parents=parents, words=1, inplace=True)
        logits = forward(W, state["ids"], m, state["tables"], state["ctx"], state["kv"], m.masks, 8)
        pick, y = ops.constrain(logits, starts=m.starts, drafts=state["ids"], masks=m.masks, penalties=pen, out=torch.float32)
        a = ops.tree_accept(pick, state["ids"], parents, m.starts, state["ctx"], state["tables"], state["kv"], 8)
        return [*m, y, pick, *a]

    pen = torch.tensor([[1.2, 0.5, 0.1]] * S).cuda()
    state = dict(ctx=ctx, held=held, cursor=cursor, tables=tables, kv=kv, new=new, ids=ids)
    first = {k: v.clone() for k, v in state.items()}
    eager = {k: v.clone() for k, v in first.items()}
    pass_over({k: v.clone() for k, v in first.items()})
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        outs = pass_over(state)
    for round in range(3):
        for k in ("ctx", "new", "ids"):       # other lengths and tokens, the same rows
            v = first[k] + (round if k == "ctx" else 0)
            v = v if k != "ids" else (v + 17 * round) % VOCAB
            v = v if k != "new" else ints([8 - round, 8, 4])
            state[k].copy_(v), eager[k].copy_(v)
        for k in ("held", "cursor", "tables", "kv"):
            state[k].copy_(first[k]), eager[k].copy_(first[k])
        graph.replay()
        want = pass_over(eager)
        torch.cuda.synchronize()
        rows = int(want[0][-1])
        for i, (a, b) in enumerate(zip(outs, want)):
            if a.dim() == 2 and a.shape == (T, VOCAB):
                a, b = a[:rows], b[:rows]
            assert torch.equal(a, b), (round, i)
        for k in ("held", "cursor", "tables"):
            assert torch.equal(state[k], eager[k])
        assert torch.equal(state["kv"].nan_to_num(), eager["kv"].nan_to_num())


def test_calls_on_streams_side_by_side():
    """Each thread its own stream and inputs, at the same time; what each gives is what it gives alone."""
    from kubeai_b200 import ops

    def make(seed):
        rng = np.random.default_rng(seed)
        rows, ctx = [20, 33, 64], [700 + 100 * seed, 40, 3000]
        tables, at = np.zeros((3, 200), dtype=np.int64), 0
        for s in range(3):
            need = U.pages(ctx[s] + rows[s])
            tables[s, :need] = np.arange(at, at + need)
            at += need
        parents = sum((U.random_tree(rng, n) for n in rows), [])
        g = torch.Generator().manual_seed(seed)
        kv = torch.randn(2, at, 2, 2, 16, 128, generator=g).bfloat16().cuda()
        starts, drafts = [0, *np.cumsum(rows)], rng.integers(0, 99, sum(rows))
        return dict(kv=kv, tables=ints(tables), starts=ints(starts), ctx=ints(ctx), new=ints(rows), parents=ints(parents), drafts=ints(drafts), held=ints([U.pages(c) for c in ctx]),
                    free=ints(np.arange(at, at + 40)), cursor=ints([0]), qkv=torch.randn(sum(rows), 12 * 128, generator=g).bfloat16().cuda(),
                    logits=(torch.randn(sum(rows), 50021, generator=g) * 3).cuda(), T=sum(rows))

    def pass_over(c):
        tables, kv = c["tables"].clone(), c["kv"].clone()
        m = ops.step_maps(c["ctx"], c["new"], c["held"], tables, c["free"], c["cursor"], c["T"], parents=c["parents"], words=2)
        y = ops.paged_attn_tree(c["qkv"], kv[0], c["tables"], m.starts, c["ctx"], m.masks, 8, 2, 64)
        ids, z = ops.constrain(c["logits"], starts=m.starts, drafts=c["drafts"], masks=m.masks, out=torch.float32, penalties=torch.full((3, 3), 0.75, device="cuda"))
        a = ops.tree_accept(ids % 99, c["drafts"], c["parents"], m.starts, c["ctx"], c["tables"], kv, 16)
        return [*m, tables, y, ids, z, *a, kv]

    cases = [make(s) for s in range(4)]
    alone = [pass_over(c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    got[i] = pass_over(cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:       # noqa: BLE001 - reported by the test's thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for want, have in zip(alone, got):
        for i, (a, b) in enumerate(zip(want, have)):
            assert torch.equal(a, b), i
