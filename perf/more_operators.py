"""The device side of a decode step whose requests share their beginnings, beams above all: what is measured of it, its plain forms and its values in 64 bits.

Four operators of kubeai_b200.ops stand between the projections of such a step:

  norm_rope_kvwrite   norms of queries and keys for each head, rotary positions in the same pass, keys and values into the paged cache
  paged_attn_shared   attention over the paged cache for groups of requests whose first pages are the same: those pass once for a group
  beam_select         log-probabilities of the beams' logits, and the best candidates over beams and vocabulary
  beam_reorder        block tables, texts and partly filled pages of the beams that go on

Lengths belong to a case and are ragged; a seed makes values, pages, scores and parents.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE, D = 16, 128
VOCAB, LAYERS, QH, KVH = 128256, 32, 32, 8      # the layer sizes that the engine's default configuration names
EPS = 1e-6
ENDS = (2, 9)                                   # tokens that end a text


def listed():
    return [
        # one request's four beams, a token each: what a launch costs
        dict(name="rotate, 4 rows", op="rotate", rows=4, far=500, kv_heads=KVH, group=4, dims=128, interleaved=False, norm="one", scaling="none", idle=0),
        # a prompt step: whole heads, the frequencies of a long context, a norm's weights shared by the heads
        dict(name="rotate, 8191 rows", op="rotate", rows=8191, far=131072, kv_heads=KVH, group=4, dims=128, interleaved=False, norm="one", scaling="llama3", idle=0),
        # interleaved pairs of three quarters of a head, weights for each head, a batch padded for a captured graph
        dict(name="rotate, 999 rows, interleaved", op="rotate", rows=999, far=1000000, kv_heads=4, group=2, dims=96, interleaved=True, norm="each", scaling="yarn", idle=25),
        # one request's beams behind its prompt
        dict(name="attention, 1 x 4 beams", op="attn", groups=1, members=4, shared=450, own=40, most=1, kv_heads=KVH, group=4),
        # a busy replica whose requests have one system prompt
        dict(name="attention, 128 behind 2048", op="attn", groups=1, members=128, shared=2048, own=500, most=1, kv_heads=KVH, group=4),
        # beams of sixteen requests, odd lengths
        dict(name="attention, 16 x 8 beams", op="attn", groups=16, members=8, shared=4001, own=250, most=1, kv_heads=KVH, group=4),
        # questions of up to 32 tokens about two long documents
        dict(name="attention, 2 x 24 questions", op="attn", groups=2, members=24, shared=16001, own=130, most=32, kv_heads=KVH, group=4),
        # one request's four beams: the choice of the next ones
        dict(name="select, 1 x 4 beams", op="select", seqs=1, beams=4, k=8, vocab=VOCAB, fp32=False, pad=0, first=False),
        # a busy replica
        dict(name="select, 64 x 8 beams", op="select", seqs=64, beams=8, k=16, vocab=VOCAB, fp32=False, pad=0, first=False),
        # logits that a penalty changed, in fp32, an odd vocabulary in wider rows
        dict(name="select, 13 x 5 beams, fp32", op="select", seqs=13, beams=5, k=15, vocab=99991, fp32=True, pad=9, first=False),
        # one request's four beams in 32 layers
        dict(name="reorder, 1 x 4 beams", op="reorder", seqs=1, beams=4, shared=450, own=40, layers=LAYERS, kv_heads=KVH, text=True),
        # a busy replica, last pages filled to every degree
        dict(name="reorder, 64 x 8 beams", op="reorder", seqs=64, beams=8, shared=100, own=45, layers=LAYERS, kv_heads=KVH, text=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotate", "attn", "attn", "select", "select", "reorder"])
    kv_heads, group = rng.choice([(8, 4), (8, 4), (4, 4), (1, 8), (5, 2), (8, 1)])
    if op == "rotate":
        return dict(op=op, rows=_log_int(rng, 1, 8000), far=_log_int(rng, 16, 1000000), kv_heads=kv_heads, group=group, dims=rng.choice([128, 128, 64, 96, 20]), interleaved=rng.random() < 0.4,
                    norm=rng.choice(["one", "each", "none"]), scaling=rng.choice(["none", "linear", "llama3", "yarn"]), idle=rng.choice([0, 0, 1, 17]))
    if op == "attn":
        shared, most = _log_int(rng, 1, 16000), rng.choice([1, 1, 1, _log_int(rng, 2, 32)])
        mine = max(most, _log_int(rng, 1, 600))
        members = _log_int(rng, 1, max(1, min(96, 64000 // mine)))
        groups = _log_int(rng, 1, max(1, min(16, 64000 // (members * mine), 64000 // shared, 800000 // (members * (shared + mine)))))
        return dict(op=op, groups=groups, members=members, shared=shared, own=mine, most=most, kv_heads=kv_heads, group=group)
    if op == "select":
        beams = _log_int(rng, 1, 16)
        return dict(op=op, seqs=_log_int(rng, 1, max(1, 256 // beams)), beams=beams, k=rng.choice([beams, 2 * beams, 3 * beams]), vocab=_log_int(rng, 60, 128256), fp32=rng.random() < 0.4,
                    pad=rng.choice([0, 8, 3]), first=rng.random() < 0.2)
    return dict(op=op, seqs=_log_int(rng, 1, 64), beams=_log_int(rng, 1, 12), shared=_log_int(rng, 1, 100), own=_log_int(rng, 1, 60), layers=_log_int(rng, 1, 24), kv_heads=kv_heads,
                text=rng.random() < 0.7)


# ------------------------------------------------------------------ lengths of a case
def _spread(n, lo, hi):
    """n lengths between lo and hi, the largest first, the others in no order."""
    v = [lo + (hi - lo) * ((i * 37) % n) // max(1, n - 1) for i in range(n)]
    return [hi] + v[1:]


def _rows(case):
    return _spread(case["groups"] * case["members"], 1, case["most"])


def _tokens(case):
    """Tokens of every request behind what its group shares, this step's rows among them."""
    return [max(n, k) for n, k in zip(_spread(case["groups"] * case["members"], min(case["most"], case["own"]), case["own"]), _rows(case))]


def _shared(case):
    return _spread(case["groups"], max(1, case["shared"] // 2), case["shared"])


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _generated(case):
    """Tokens that each request's beams have behind the prompt."""
    return _spread(case["seqs"], max(1, case["own"] // 4), case["own"])


def _room(case):
    return max(p + n for p, n in zip(_spread(case["seqs"], max(1, case["shared"] // 2), case["shared"]), _generated(case))) + 8


def work(case):
    if case["op"] == "rotate":
        live, qh, kvh = case["rows"] - case["idle"] * (case["idle"] < case["rows"]), case["kv_heads"] * case["group"], case["kv_heads"]
        weights = dict(one=2 * D * 2, each=(qh + kvh) * D * 2, none=0)[case["norm"]]
        return dict(bytes=2 * live * (qh + 2 * kvh) * D * 2 + 8 * case["rows"] + weights + 8 * (case["dims"] // 2), flops=live * (qh + kvh) * D * 8)
    if case["op"] == "attn":
        n, mine, kvh = _rows(case), _tokens(case), case["kv_heads"]
        heads, T = kvh * case["group"], sum(n)
        front = [p for p in _shared(case) for _ in range(case["members"])]
        keys = sum(_shared(case)) + sum(mine)
        return dict(bytes=keys * kvh * 2 * D * 2 + 2 * T * heads * D * 2, flops=4 * D * heads * sum(k * (p + m) for k, p, m in zip(n, front, mine)))
    if case["op"] == "select":
        rows, size = case["seqs"] * case["beams"], 4 if case["fp32"] else 2
        return dict(bytes=rows * case["vocab"] * size + 4 * rows + case["seqs"] * 12 * (case["k"] + case["beams"]), flops=3 * rows * case["vocab"])
    front, mine, B = _spread(case["seqs"], max(1, case["shared"] // 2), case["shared"]), _generated(case), case["beams"]
    lens = [p + n for p, n in zip(front, mine)]
    rows = case["seqs"] * B
    width = max(map(_pages, lens)) + 1
    # of B parents drawn at random, B (1 - 1/e) are others'; the rest of the beams are copies
    copies = 0 if B == 1 else B * ((1 - 1 / B) ** B)
    moved = sum(copies * (n % PAGE) for n in lens) * case["layers"] * 2 * case["kv_heads"] * D * 2
    texts = (2 * B * sum(lens) * 4) if case["text"] else 0
    return dict(bytes=int(2 * moved) + 3 * rows * width * 4 + texts + 16 * rows, flops=0)


# ------------------------------------------------------------------ inputs
def _ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).to(DEV)


def _freqs(case):
    """Radians a position of each rotated pair, and what the rotated values are multiplied by; the scalings as model configurations name them."""
    dims = case["dims"]
    f = 500000.0 ** (-np.arange(0, dims, 2, dtype=np.float64) / dims)
    if case["scaling"] == "linear":
        return f / 8, 1.0
    if case["scaling"] == "llama3":
        factor, low, high, length = 8.0, 1.0, 4.0, 8192
        turns = length * f / (2 * math.pi)
        part = np.clip((turns - low) / (high - low), 0, 1)
        return f / factor * (1 - part) + f * part, 1.0
    if case["scaling"] == "yarn":
        factor, fast, slow, length = 32.0, 32.0, 1.0, 4096
        at = lambda turns: dims * math.log(length / (2 * math.pi * turns)) / (2 * math.log(500000.0))      # noqa: E731
        lo, hi = max(0, math.floor(at(fast))), min(dims - 1, math.ceil(at(slow)))
        part = np.clip((np.arange(dims // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * part + f * (1 - part), 0.1 * math.log(factor) + 1
    return f, 1.0


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV, dtype=torch.bfloat16)      # noqa: E731
    return dict(rotate=_prepare_rotate, attn=_prepare_attn, select=_prepare_select, reorder=_prepare_reorder)[case["op"]](case, rng, gen, normal) | dict(case=case)


def _prepare_rotate(case, rng, gen, normal):
    T, kvh, heads = case["rows"], case["kv_heads"], case["kv_heads"] * case["group"]
    slots = rng.permutation(_pages(T + 40) * PAGE)[:T]
    if 0 < case["idle"] < T:
        slots[T - case["idle"]:] = -1                      # rows behind the batch have no place
    f, gain = _freqs(case)
    norm = lambda n: (1 + 0.2 * torch.randn(*((n, D) if case["norm"] == "each" else (D,)), generator=gen, device=DEV)).bfloat16() if case["norm"] != "none" else None      # noqa: E731
    # heads of different sizes, as projections give them
    size = torch.rand(heads + 2 * kvh, 1, generator=gen, device=DEV) * 3 + 0.1
    qkv = (torch.randn(T, heads + 2 * kvh, D, generator=gen, device=DEV) * size).bfloat16().view(T, -1)
    return dict(qkv=qkv, positions=_ints(rng.integers(0, case["far"], T)), slots=_ints(slots), kv=normal(_pages(T + 40), 2, kvh, PAGE, D), q_norm=norm(heads), k_norm=norm(kvh),
                freqs=torch.tensor(f, dtype=torch.float64).to(DEV), gain=gain)


def _prepare_attn(case, rng, gen, normal):
    n, mine, front, kvh, heads = _rows(case), _tokens(case), _shared(case), case["kv_heads"], case["kv_heads"] * case["group"]
    S, M = len(n), case["members"]
    lens = [front[s // M] + m for s, m in enumerate(mine)]
    whole = [front[s // M] // PAGE for s in range(S)]      # the shared tokens' last page, where it is not full, is everybody's own
    need = sum(p // PAGE for p in front) + sum(_pages(t) - w for t, w in zip(lens, whole))
    order, tables, at = rng.permutation(need), np.zeros((S, max(map(_pages, lens))), dtype=np.int64), 0
    for g, p in enumerate(front):
        tables[g * M:(g + 1) * M, :p // PAGE] = order[at:at + p // PAGE]
        at += p // PAGE
    for s in range(S):
        k = _pages(lens[s]) - whole[s]
        tables[s, whole[s]:whole[s] + k] = order[at:at + k]
        at += k
    kv = normal(need, 2, kvh, PAGE, D)
    # the tokens of a shared page that is not full are the same ones in every request
    for g, p in enumerate(front):
        if p % PAGE:
            kv[torch.tensor(tables[g * M:(g + 1) * M, p // PAGE]).to(DEV), :, :, :p % PAGE] = normal(1, 2, kvh, p % PAGE, D)
    return dict(qkv=normal(sum(n), (heads + 2 * kvh) * D), kv=kv, tables=_ints(tables), starts=_ints(np.concatenate([[0], np.cumsum(n)])), ctx=_ints([t - k for t, k in zip(lens, n)]),
                group_starts=_ints(np.arange(case["groups"] + 1) * M), shared=_ints(front), max_ctx=max(lens))


def _prepare_select(case, rng, gen, normal):
    S, B, V = case["seqs"], case["beams"], case["vocab"]
    rows = torch.randn(S * B, V + case["pad"], generator=gen, device=DEV) * 2.5
    # a few tokens are likely
    liked = torch.randint(0, V, (S * B, 6), generator=gen, device=DEV)
    rows.scatter_add_(1, liked, torch.rand(S * B, 6, generator=gen, device=DEV) * 9)
    # a text may end anywhere
    ends = [e for e in ENDS if e < V]
    rows[:, ends] += torch.rand(S * B, len(ends), generator=gen, device=DEV) * 12
    scores = -torch.rand(S, B, generator=gen, device=DEV).cumsum(1) * 4 - 10
    if case["first"]:
        scores[:, 1:] = -math.inf                          # behind the prompt all beams are the same one
    return dict(logits=(rows if case["fp32"] else rows.bfloat16())[:, :V], scores=scores, ends=_ints(ends))


def _prepare_reorder(case, rng, gen, normal):
    S, B, kvh = case["seqs"], case["beams"], case["kv_heads"]
    front, mine = _spread(S, max(1, case["shared"] // 2), case["shared"]), _generated(case)
    lens = [p + n for p, n in zip(front, mine)]
    width = max(map(_pages, lens)) + 1
    tables, at = np.full((S * B, width), -1, dtype=np.int64), 0
    for s in range(S):
        for c in range(_pages(lens[s])):
            # the prompt's pages are everybody's; of those behind it the older ones belong to fewer beams; one that is not full has one owner
            kinds = 1 if (c + 1) * PAGE <= front[s] else B if (c + 1) * PAGE > lens[s] else min(B, 1 + c % 3)
            tables[s * B:(s + 1) * B, c] = at + np.arange(B) * kinds // B
            at += kinds
    tables[tables >= 0] = rng.permutation(at)[tables[tables >= 0]]
    parents = rng.integers(0, B, (S, B))
    parents[:, -1] = np.where(rng.random(S) < 0.1, -1, parents[:, -1])      # fewer candidates than beams
    if B == 1:
        parents[:] = 0
    text = _ints(rng.integers(0, VOCAB, (S * B, _room(case)))) if case["text"] else None
    return dict(parents=_ints(parents), tokens=_ints(rng.integers(0, VOCAB, (S, B))), ctx=_ints(np.repeat(lens, B)), tables=_ints(tables), kv=normal(case["layers"], at, 2, kvh, PAGE, D),
                texts=text, text_lens=_ints(np.repeat(lens, B)) if case["text"] else None)


# ------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _own(st)
    return dict(rotate=_plain_rotate, attn=_plain_attn, select=_plain_select, reorder=_plain_reorder)[st["case"]["op"]](st)


def _own(st):
    from kubeai_b200 import ops
    case = st["case"]
    if case["op"] == "rotate":
        q = ops.norm_rope_kvwrite(st["qkv"], st["positions"], st["slots"], st["kv"], case["kv_heads"] * case["group"], case["kv_heads"], st["freqs"], gain=st["gain"], q_norm=st["q_norm"],
                                  k_norm=st["k_norm"], eps=EPS, interleaved=case["interleaved"])
        return dict(q=q, kv=st["kv"])
    if case["op"] == "attn":
        return ops.paged_attn_shared(st["qkv"], st["kv"], st["tables"], st["starts"], st["ctx"], st["group_starts"], st["shared"], case["kv_heads"] * case["group"], case["kv_heads"],
                                     case["most"], max_ctx=st["max_ctx"])
    if case["op"] == "select":
        b = ops.beam_select(st["logits"], st["scores"], case["k"], ends=st["ends"])
        return dict(parents=b.parents, tokens=b.tokens, scores=b.scores, found_parents=b.found_parents, found_tokens=b.found_tokens, found_scores=b.found_scores)
    r = ops.beam_reorder(st["parents"], st["tokens"], st["ctx"], st["tables"], st["kv"], texts=st["texts"], text_lens=st["text_lens"])
    return dict(tables=r.block_tables, shared=r.shared, released=r.released, kv=st["kv"], **(dict(texts=r.texts, text_lens=r.text_lens) if st["texts"] is not None else {}))


# ------------------------------------------------------------------ plain forms
def _plain_rotate(st):
    case, kv, T = st["case"], st["kv"], st["case"]["rows"]
    kvh, heads, n = case["kv_heads"], case["kv_heads"] * case["group"], case["dims"] // 2
    x = st["qkv"].view(T, heads + 2 * kvh, D)
    q, k = x[:, :heads].float(), x[:, heads:heads + kvh].float()
    if st["q_norm"] is not None:
        q, k = (t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * w.float() for t, w in ((q, st["q_norm"]), (k, st["k_norm"])))
    # angles of far positions in 64 bits
    angle = st["positions"].double()[:, None] * st["freqs"]
    cos, sin = ((t * st["gain"]).float()[:, None] for t in (torch.cos(angle), torch.sin(angle)))

    def rotated(t):
        if case["interleaved"]:
            a, b = t[..., 0:2 * n:2], t[..., 1:2 * n:2]
            pairs = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = t[..., :n], t[..., n:2 * n]
            pairs = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([pairs, t[..., 2 * n:]], -1).bfloat16()

    q, k = rotated(q), rotated(k)
    slots = st["slots"].long()
    row = (slots >= 0).nonzero()[:, 0]
    page, at = slots[row] // PAGE, slots[row] % PAGE
    kv[page, 0, :, at] = k[row]
    kv[page, 1, :, at] = x[row, heads + kvh:]
    return dict(q=q.reshape(T, heads * D), kv=kv)


def _plain_attn(st):
    case, starts, ctx = st["case"], st["starts"].long(), st["ctx"].long()
    kvh, G, S, T, most = case["kv_heads"], case["group"], len(st["ctx"]), st["qkv"].shape[0], case["most"]
    seq = torch.searchsorted(starts[1:].contiguous(), torch.arange(T, device=DEV), right=True)
    i = torch.arange(T, device=DEV) - starts[seq]
    q = torch.zeros(S, most, kvh, G, D, device=DEV)      # every request as wide as the widest
    q[seq, i] = st["qkv"][:, :kvh * G * D].float().view(T, kvh, G, D)
    k, v = (st["kv"][:, w][st["tables"].long()].transpose(2, 3).reshape(S, -1, kvh, D).float() for w in (0, 1))      # [request, key, head, dimension]
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(S, kvh, G * most, D), k.permute(0, 2, 3, 1)).view(S, kvh, G, most, -1) * D ** -0.5
    seen = torch.arange(k.shape[1], device=DEV) <= ctx[:, None, None] + torch.arange(most, device=DEV)[:, None]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
    y = torch.matmul(p.view(S, kvh, G * most, -1), v.transpose(1, 2)).view(S, kvh, G, most, D) / p.sum(-1, keepdim=True)
    return y.permute(0, 3, 1, 2, 4)[seq, i].reshape(T, kvh * G * D).bfloat16()


def _plain_select(st):
    S, B = st["scores"].shape
    V, k = st["logits"].shape[1], st["case"]["k"]
    x = st["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    total = torch.exp((x - top).double()).sum(1, keepdim=True)      # in 64 bits: what lies close together keeps its order
    best, token = (t[:, :k] for t in torch.sort(x, dim=1, descending=True, stable=True))
    c = (best.double() - (top.double() + torch.log(total))).view(S, B, -1) + st["scores"].double()[:, :, None]
    c, order = torch.sort(c.flatten(1), dim=1, descending=True, stable=True)
    c, order = c[:, :k], order[:, :k]
    real = c > -math.inf
    token = torch.where(real, token.reshape(S, -1).gather(1, order), -1)
    parent = torch.where(real, order // min(k, V), -1)
    if c.shape[1] < k:      # fewer tokens than candidates asked for
        room = (0, k - c.shape[1])
        c, token, parent, real = (torch.nn.functional.pad(t, room, value=f) for t, f in ((c, -math.inf), (token, -1), (parent, -1), (real, False)))
    # those that do not end go on, in order
    on = real & ~(token[:, :, None] == st["ends"][None, None, :]).any(-1)
    place = torch.where(on & (on.cumsum(1) <= B), on.cumsum(1) - 1, B)
    pick = lambda t, rest: torch.full((S, B + 1), rest, dtype=t.dtype, device=DEV).scatter_(1, place, t)[:, :B]      # noqa: E731
    return dict(parents=pick(parent, -1).int(), tokens=pick(token, -1).int(), scores=pick(c.float(), -math.inf), found_parents=parent.int(), found_tokens=token.int(), found_scores=c.float())


def _plain_reorder(st):
    tables, kv, ctx = st["tables"].long(), st["kv"], st["ctx"].long()
    S, B = st["parents"].shape
    parents, ctx, width = st["parents"].long(), ctx.view(S, B)[:, 0], tables.shape[1]
    b = torch.arange(B, device=DEV)
    # a beam that is none follows the request's first one
    real = parents >= 0
    lead = parents.gather(1, real.int().argmax(1, keepdim=True))
    p = torch.where(real, parents, lead)
    same = p[:, :, None] == p[:, None, :]
    extra = (same & (b[None, :] < b[:, None])).any(2)                # not its parent's first child
    childless = ~(p[:, :, None] == b).any(1)
    free = torch.argsort(childless.int(), dim=1, descending=True, stable=True)      # childless beams first, in order
    heir = torch.where(extra, free.gather(1, (extra.cumsum(1) - 1).clamp(min=0)), p)      # whose partly filled page a beam takes
    old = tables.view(S, B, width)
    col = torch.arange(width, device=DEV)
    full, part = ctx // PAGE, ctx % PAGE
    new = old.gather(1, p[:, :, None].expand(S, B, width))
    last = (col == full[:, None]) & (part > 0)[:, None]
    new = torch.where(last[:, None], old.gather(1, heir[:, :, None].expand(S, B, width)), new)
    new = torch.where((col < (full + (part > 0))[:, None])[:, None], new, old)
    # whole pages that no beam names any more, each once
    kept = (old[:, :, None] == new[:, None, :]).any(2)
    earlier = ((old[:, :, None] == old[:, None, :]) & (b[None, :] < b[:, None])[None, :, :, None]).any(2)
    gone = ~kept & ~earlier & (col < full[:, None])[:, None]
    alike = (new == new[:, :1]).all(1) & (col < full[:, None])
    shared = alike.int().cumprod(1).sum(1) * PAGE
    s, i = extra.nonzero(as_tuple=True)
    src, dst = (old[s, t[s, i], full[s].clamp(max=width - 1)] for t in (p, heir))
    row = torch.arange(PAGE, device=DEV)[None, :] < part[s, None]
    at, r = row.nonzero(as_tuple=True)
    kv[:, dst[at], :, :, r] = kv[:, src[at], :, :, r]
    out = dict(tables=new.reshape(S * B, width).int(), shared=shared.int(), released=torch.where(gone, old, -1).reshape(S * B, width).int(), kv=kv)
    if st["texts"] is not None:
        texts = st["texts"].view(S, B, -1).gather(1, p[:, :, None].expand(S, B, st["texts"].shape[1]))
        end = torch.arange(texts.shape[2], device=DEV) == st["text_lens"].view(S, B).gather(1, p)[:, :, None]
        out["texts"] = torch.where(end & real[:, :, None], st["tokens"][:, :, None], texts).view(S * B, -1)
        out["text_lens"] = (st["text_lens"].view(S, B).gather(1, p) + real).view(-1).int()
    return out


# ------------------------------------------------------------------ the definitions, row by row
def exact(case, seed):
    st = prepare(case, seed)
    return dict(rotate=_exact_rotate, attn=_exact_attn, select=_exact_select, reorder=_exact_reorder)[case["op"]](st)


def _exact_rotate(st):
    case = st["case"]
    kvh, heads, n = case["kv_heads"], case["kv_heads"] * case["group"], case["dims"] // 2
    kv = st["kv"].double()
    out = torch.empty(case["rows"], heads * D, dtype=torch.float64, device=DEV)
    first, second = (torch.arange(n, device=DEV) * 2, torch.arange(n, device=DEV) * 2 + 1) if case["interleaved"] else (torch.arange(n, device=DEV), torch.arange(n, device=DEV) + n)
    turn = torch.polar(torch.full((case["rows"], n), st["gain"], dtype=torch.float64, device=DEV), torch.outer(st["positions"].double(), st["freqs"]))
    slots = st["slots"].long()
    there = slots >= 0
    page, at = slots[there] // PAGE, slots[there] % PAGE
    for h in range(heads + 2 * kvh):
        x = st["qkv"][:, h * D:(h + 1) * D].double()
        if h < heads + kvh:
            w = st["q_norm"] if h < heads else st["k_norm"]
            if w is not None:
                w = w.double() if w.dim() == 1 else w[h if h < heads else h - heads].double()
                x = w * x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / D + EPS)
            z = torch.complex(x[:, first].contiguous(), x[:, second].contiguous()) * turn
            x[:, first], x[:, second] = z.real, z.imag
        if h < heads:
            out[:, h * D:(h + 1) * D] = x
        else:
            kv[page, int(h >= heads + kvh), (h - heads) % kvh, at] = x[there]
    return dict(q=out, kv=kv)


def _exact_attn(st):
    case, starts, ctx = st["case"], st["starts"].tolist(), st["ctx"].tolist()
    kvh, G = case["kv_heads"], case["group"]
    out = torch.zeros(starts[-1], kvh * G, D, dtype=torch.float64, device=DEV)
    for s, c in enumerate(ctx):
        a, b = starts[s], starts[s + 1]
        n = b - a
        pages = st["tables"][s, :_pages(c + n)].long()
        k, v = (st["kv"][pages, w].transpose(0, 1).reshape(kvh, -1, D)[:, :c + n].double() for w in (0, 1))
        q = st["qkv"][a:b, :kvh * G * D].double().view(n, kvh, G, D).permute(1, 2, 0, 3)
        hidden = torch.ones(n, c + n, dtype=torch.bool, device=DEV).triu(c + 1)
        p = torch.softmax((q @ k.mT[:, None] / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
        out[a:b] = (p @ v[:, None]).permute(2, 0, 1, 3).reshape(n, kvh * G, D)
    return out.view(starts[-1], -1)


def _exact_select(st):
    case = st["case"]
    S, B, V, k = case["seqs"], case["beams"], case["vocab"], case["k"]
    x = st["logits"].double()
    share = x - torch.logsumexp(x, 1, keepdim=True)
    ends, found, goes = set(st["ends"].tolist()), [], []
    for s in range(S):
        c = (share[s * B:(s + 1) * B] + st["scores"][s].double()[:, None]).flatten()
        at = torch.topk(c, min(len(c), k + 200)).indices      # more than are wanted: ties go to the lowest index
        value, at = c[at].cpu().numpy(), at.cpu().numpy()
        order = np.lexsort((at, -value))[:k]
        best = [(float(v), int(i) // V, int(i) % V) if v > -math.inf else (-math.inf, -1, -1) for v, i in zip(value[order], at[order])]
        best += [(-math.inf, -1, -1)] * (k - len(best))
        found.append(best)
        on = [f for f in best if f[1] >= 0 and f[2] not in ends][:B]
        goes.append(on + [(-math.inf, -1, -1)] * (B - len(on)))
    whole = lambda rows, j: _ints([[r[j] for r in row] for row in rows])      # noqa: E731
    value = lambda rows: torch.tensor([[r[0] for r in row] for row in rows], dtype=torch.float64).to(DEV)      # noqa: E731
    return dict(parents=whole(goes, 1), tokens=whole(goes, 2), scores=value(goes), found_parents=whole(found, 1), found_tokens=whole(found, 2), found_scores=value(found))


def _exact_reorder(st):
    case, kv = st["case"], st["kv"]
    B, old, ctx = case["beams"], st["tables"].cpu().numpy(), st["ctx"].tolist()
    new, released, shared, moves = old.copy(), np.full_like(old, -1), [], []
    texts = st["texts"].cpu().numpy().copy() if case["text"] else None
    lens = []
    for s, named in enumerate(st["parents"].tolist()):
        rows, full, part = range(s * B, (s + 1) * B), ctx[s * B] // PAGE, ctx[s * B] % PAGE
        lead = next(p for p in named if p >= 0)
        parents = [p if p >= 0 else lead for p in named]
        spare = [b for b in range(B) if b not in parents]
        for i, p in enumerate(parents):
            new[rows[i], :full] = old[rows[p], :full]
            if part:
                heir = p if p not in parents[:i] else spare.pop(0)
                new[rows[i], full] = old[rows[heir], full]
                if heir != p:
                    moves.append((old[rows[p], full], old[rows[heir], full], part))
            if texts is not None:
                texts[rows[i]] = st["texts"][rows[p]].cpu().numpy()
                lens.append(int(st["text_lens"][rows[p]]))
                if named[i] >= 0:
                    texts[rows[i], lens[-1]] = int(st["tokens"][s, i])
                    lens[-1] += 1
        for c in range(full):
            stays, seen = set(new[list(rows), c].tolist()), set()
            for r in rows:
                page = int(old[r, c])
                if page not in stays and page not in seen:
                    released[r, c] = page
                seen.add(page)
        alike = [len(set(new[list(rows), c].tolist())) == 1 for c in range(full)] + [False]
        shared.append(alike.index(False) * PAGE)
    for src, dst, part in moves:
        kv[:, dst, :, :, :part] = kv[:, src, :, :, :part]
    out = dict(tables=_ints(new), shared=_ints(shared), released=_ints(released), kv=kv)
    return out | (dict(texts=_ints(texts), text_lens=_ints(lens)) if texts is not None else {})
