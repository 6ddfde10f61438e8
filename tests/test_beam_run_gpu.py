"""Decode steps of beams, as they would be run: rows get places, queries and keys norms and positions, beams that share their pages are attended together, the best candidates of all go on, and
tables, texts and the cache follow them."""
import math

import numpy as np
import pytest
import torch

import beam_step_util as plain

pytestmark = pytest.mark.gpu
D, PAGE, BF16 = 128, 16, 2.0 ** -8      # BF16: half a step, relative to the value


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


class Model:
    def __init__(self, kvh=2, group=4, layers=2, V=1200, hidden=256, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")      # noqa: E731
        self.kvh, self.heads, self.layers, self.V = kvh, kvh * group, layers, V
        self.embed = normal(V, hidden).bfloat16()
        self.qkv = [(normal(hidden, (self.heads + 2 * kvh) * D) * hidden ** -0.5).bfloat16() for _ in range(layers)]
        self.down = [(normal(self.heads * D, hidden) * (self.heads * D) ** -0.5).bfloat16() for _ in range(layers)]
        self.up = (normal(hidden, V) * 2 * hidden ** -0.5).bfloat16()
        self.norms = [(1 + 0.1 * normal(D)).bfloat16() for _ in range(2 * layers)]


class Beams:
    """What a replica keeps of its requests: every one has its prompt in the cache, on pages that its beams share but for the last one where it is not full."""

    def __init__(self, model, prompts, B, room, seed=1, pad=0):
        from kubeai_b200 import ops
        rng, gen = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed)
        self.m, self.S, self.B, self.pad = model, len(prompts), B, pad
        R = self.S * B
        width = max(map(plain.pages, prompts)) + plain.pages(room) + 1
        tables, held, at = np.full((R, width), -1), np.zeros(R, dtype=int), 0
        for s, n in enumerate(prompts):
            whole = n // PAGE
            tables[s * B:(s + 1) * B, :whole] = np.arange(at, at + whole)
            at += whole
            for b in range(B if n % PAGE else 0):
                tables[s * B + b, whole] = at
                at += 1
            held[s * B:(s + 1) * B] = plain.pages(n)
        self.pages = at + R * (plain.pages(room) + 1)
        names = rng.permutation(self.pages)
        self.tables = ints(np.where(tables >= 0, names[tables], -1))
        self.free, self.cursor, self.held = ints(names[at:]), ints([0]), ints(held)
        self.kv = torch.randn(model.layers, self.pages, 2, model.kvh, PAGE, D, generator=gen, device="cuda").bfloat16()
        for s, n in enumerate(prompts):      # the beams' copies of a last page are alike
            if n % PAGE:
                mine = self.tables[s * B:(s + 1) * B, n // PAGE].long()
                self.kv[:, mine] = self.kv[:, mine[:1]]
        self.ctx = ints(np.repeat(prompts, B))
        self.tokens = ints(rng.integers(0, model.V, (self.S, 1)).repeat(B, 1))
        self.scores = torch.full((self.S, B), -math.inf, device="cuda")
        self.scores[:, 0] = 0
        self.shared = ints([n // PAGE * PAGE for n in prompts])
        self.texts = torch.zeros(R, room, dtype=torch.int32, device="cuda")
        self.text_lens = ints([0] * R)
        self.group_starts, self.new = ints(np.arange(self.S + 1) * B), ints([1] * R)
        self.turn = ops.rotary(base=5e5)
        self.most = max(prompts) + room

    NAMES = "tables free cursor held kv ctx tokens scores shared texts text_lens".split()

    def state(self):
        return {n: getattr(self, n).clone() for n in self.NAMES}

    def put(self, state):
        for n in self.NAMES:
            getattr(self, n).copy_(state[n])

    def step(self, seen=None):
        """A step of all beams; what the operations were given and answered goes to `seen`."""
        from kubeai_b200 import ops
        m, R = self.m, self.S * self.B
        T = R + self.pad
        maps = ops.step_maps(self.ctx, self.new, self.held, self.tables, self.free, self.cursor, T)
        rows = torch.cat([self.tokens.view(-1), self.tokens.new_zeros(self.pad)])
        x = m.embed[rows.clamp(min=0).long()]
        attended = []
        for i in range(m.layers):
            qkv = x @ m.qkv[i]
            q = ops.norm_rope_kvwrite(qkv, maps.positions, maps.slots, self.kv[i], m.heads, m.kvh, self.turn.freqs, self.turn.gain, m.norms[2 * i], m.norms[2 * i + 1])
            y = ops.paged_attn_shared(q, self.kv[i], self.tables, maps.starts, self.ctx, self.group_starts, self.shared, m.heads, m.kvh, 1, max_ctx=self.most, status=maps.status)
            attended.append((q, y))
            x = x + y @ m.down[i]
        logits = x @ m.up
        best = ops.beam_select(logits[:R], self.scores, ends=ints([7, 11]) if seen is not None else None)
        after = self.ctx + 1
        moved = ops.beam_reorder(best.parents, best.tokens, after, self.tables, self.kv, self.texts, self.text_lens)
        if seen is not None:
            seen.update(maps=maps, attended=attended, logits=logits, best=best, moved=moved)
        self.held, self.cursor, self.ctx = maps.held, maps.cursor, after
        self.tables, self.shared, self.texts, self.text_lens = moved.block_tables, moved.shared, moved.texts, moved.text_lens
        self.tokens, self.scores = best.tokens, best.scores


def of_tables(kv, tables, ctx):
    """Every row's keys and values in order: [layers, 2, heads, tokens, 128]."""
    return [kv[:, row[:plain.pages(n)]].transpose(0, 2, 3, 1, 4, 5).reshape(kv.shape[0], 2, kv.shape[3], -1, D)[:, :, :, :n] for row, n in zip(tables, ctx)]


@pytest.mark.parametrize("prompts,B,steps,pad", [([40], 4, 20, 0), ([16, 333, 5], 4, 18, 0), ([100, 31], 8, 36, 3), ([0, 17], 1, 17, 0), ([640, 48, 47, 49], 32, 6, 5)])
def test_beams_over_page_boundaries(prompts, B, steps, pad):
    m = Model()
    r = Beams(m, prompts, B, steps + 2, pad=pad)
    S, R = r.S, r.S * B
    host = lambda t: t.cpu().numpy()      # noqa: E731
    exact = lambda t: t.double().cpu().numpy()      # noqa: E731
    lists = of_tables(exact(r.kv), host(r.tables), host(r.ctx))      # every beam's keys and values, as the plain form has them
    texts = [[] for _ in range(R)]
    for _ in range(steps):
        scores, seen = r.scores.clone(), {}
        alive = np.isfinite(host(r.scores)).reshape(-1)
        r.step(seen)
        # rows have places, each its own
        slots = host(seen["maps"].slots)
        assert (host(seen["maps"].status) == 0).all() and (slots[:R] >= 0).all() and len(set(slots[:R])) == R and (slots[R:] == -1).all()
        kv = exact(r.kv)
        assert all(bool((y[R:] == 0).all()) for _, y in seen["attended"])
        best, moved = seen["best"], seen["moved"]
        # ---- the choice, on the logits as they are
        x = exact(seen["logits"])[:R].reshape(S, B, m.V)
        found, goes, gap = plain.selected(x, exact(scores), 2 * B, {7, 11})
        for want, c, p, v in ((found, best.found_scores, best.found_parents, best.found_tokens), (goes, best.scores, best.parents, best.tokens)):
            w = np.array([[e[0] for e in row] for row in want])
            fine = np.isfinite(w)
            assert (np.abs(exact(c)[fine] - w[fine]) <= 2.0 ** -24 * np.abs(w[fine]) + 2.0 ** -20).all() and (exact(c)[~fine] == w[~fine]).all()
            if gap > 1e-6:      # what decides is exact to the sum's error
                assert p.tolist() == [[e[1] for e in row] for row in want] and v.tolist() == [[e[2] for e in row] for row in want]
        # ---- the beams that go on: their texts, and in the cache their parents' keys and values with the step's own behind them
        parents, tokens = host(best.parents), host(best.tokens)
        now = of_tables(kv, host(r.tables), host(r.ctx))
        new_texts, rows = [], {}
        for s in range(S):
            assert (parents[s] >= 0).all()
            for b in range(B):
                new_texts.append(texts[s * B + parents[s, b]] + [int(tokens[s, b])])
        for at in range(R):
            p = at // B * B + parents.reshape(-1)[at]
            assert (now[at][:, :, :, :-1] == lists[p]).all()
            step = now[at][:, :, :, -1]
            assert p not in rows or (rows[p] == step).all()      # all heirs have the same row
            rows[p] = step
        texts = new_texts
        for at in range(R):
            assert host(r.texts)[at, :len(texts[at])].tolist() == texts[at] and int(host(r.text_lens)[at]) == len(texts[at])
        # ---- attention, of the beams that had heirs (the others' rows may have been overwritten since)
        for p, step in rows.items():
            if not alive[p]:
                continue
            for i, (q, y) in enumerate(seen["attended"]):
                k, v = (np.concatenate([lists[p][i, j], step[i, j][:, None]], 1) for j in (0, 1))
                q_p, y_p = exact(q[p]).reshape(m.heads, D), exact(y[p]).reshape(m.heads, D)
                for h in range(m.heads):
                    z = k[h // (m.heads // m.kvh)] @ q_p[h] * D ** -0.5
                    w = np.exp(z - z.max())
                    w /= w.sum()
                    mine = v[h // (m.heads // m.kvh)]
                    want, size = w @ mine, w @ np.abs(mine)
                    assert (np.abs(y_p[h] - want) <= (2 * BF16 + 2.0 ** -12) * size + BF16 * np.abs(want) + 1e-30).all()
        lists = now
        # ---- pages: a page that is not full has one owner, what beams share is shared from the start, and what nobody has any more is nobody's
        tables, c = host(r.tables), host(r.ctx)
        last = [int(tables[b, c[b] // PAGE]) for b in range(R) if c[b] % PAGE]
        everywhere = [int(p) for b in range(R) for p in tables[b, :c[b] // PAGE]]
        assert len(set(last)) == len(last) and not set(last) & set(everywhere)
        gone = [int(p) for p in host(moved.released).reshape(-1) if p >= 0]
        assert len(set(gone)) == len(gone) and not set(gone) & (set(everywhere) | set(last))
        for s in range(S):
            n = int(host(r.shared)[s])
            assert n % PAGE == 0 and n <= c[s * B] and (tables[s * B:(s + 1) * B, :n // PAGE] == tables[s * B, :n // PAGE]).all()
        # the pages that were released go to those that are free
        if gone:
            r.free, r.cursor = torch.cat([r.free[int(r.cursor):], ints(gone)]), ints([0])


def answers(r):
    return [t.clone() for t in (r.tables, r.texts, r.text_lens, r.scores, r.tokens, r.shared, r.held, r.cursor, r.kv)]


def run(r, steps):
    for _ in range(steps):
        r.step()
    return answers(r)


def same(a, b):
    return all(torch.equal(x.view(torch.int16) if x.dtype is torch.bfloat16 else x, y.view(torch.int16) if y.dtype is torch.bfloat16 else y) for x, y in zip(a, b))


def test_steps_in_a_graph_and_on_two_streams_at_once():
    m = Model(seed=3)
    makers = [lambda: Beams(m, [70, 300, 16], 4, 24, seed=5), lambda: Beams(m, [1000, 15], 24, 24, seed=6)]
    want = [run(make(), 20) for make in makers]
    # twice more, at the same time on two streams
    beams, sides = [make() for make in makers], [torch.cuda.Stream() for _ in makers]
    torch.cuda.synchronize()
    for _ in range(20):
        for r, side in zip(beams, sides):
            with torch.cuda.stream(side):
                r.step()
    torch.cuda.synchronize()
    for r, w in zip(beams, want):
        assert same(answers(r), w)
    # both in graphs of four steps, captured one behind the other and replayed in turn
    graphs = []
    for make in makers:
        r = make()
        start = r.state()
        r.step()
        r.put(start)
        kept = r.state()      # what a graph reads and writes: copied in front of every replay, as a program would hand its state on
        for n in Beams.NAMES:
            setattr(r, n, kept[n])
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            for _ in range(4):
                r.step()
            after = r.state()
        graphs.append((g, start, kept, after, r))      # (what the graph reads lives as long as it)
    for turn in range(5):
        for g, start, kept, after, _ in graphs:
            for n in Beams.NAMES:
                kept[n].copy_((after if turn else start)[n])
            g.replay()
    torch.cuda.synchronize()
    for (_, _, _, after, _), w in zip(graphs, want):
        got = [after[n] for n in "tables texts text_lens scores tokens shared held cursor kv".split()]
        assert same(got, w)
