"""The device side of a verification step of drafted tokens: what is measured of it, its plain forms and its values in 64 bits.

A step runs the tokens that a drafter proposed for each of a batch of requests, as a tree that hangs on the request's last token.
Four operators of kubeai_b200.ops take it from the requests' lengths to their new ones:

  step_maps         pages, block tables, slots, positions and ancestor masks of the step's rows, made on the GPU
  paged_attn_tree   attention of the rows over the paged cache and over their ancestors in the tree
  constrain         repetition, presence and frequency penalties, biases and grammar masks on the rows' logits, and the choice
  tree_accept       the path of drafts that the choices confirm, and its cache rows moved to where they stay

Lengths belong to a case and are ragged; a seed makes values, trees, pages and lists.  A request's row 0 is its last token, which is
not in the cache yet; the other rows are drafts, a parent always in front of its children.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE, D = 16, 128
VOCAB, LAYERS, QH, KVH = 128256, 32, 32, 8      # the layer sizes that the engine's default configuration names
PATH = 16                                       # rows of an accepted path at most


def listed():
    return [
        # one user, a small tree: what a launch costs
        dict(name="maps, 1 request", op="maps", seqs=1, ctx=450, most=8, tree=True, pad=0),
        # a full replica, drafted trees of up to 64 rows, in a batch padded for a captured graph
        dict(name="maps, 128 trees", op="maps", seqs=128, ctx=2048, most=64, tree=True, pad=77),
        # a step of many prompt portions: pages by the hundred, no trees
        dict(name="maps, 512 prompt portions", op="maps", seqs=512, ctx=1500, most=127, tree=False, pad=0),
        # a conversation of one user: few keys, eight rows
        dict(name="attention, 1 x 450", op="attn", seqs=1, ctx=450, most=8, kv_heads=KVH, group=4, chain=False),
        # a busy replica, trees of up to 16 rows over ragged contexts
        dict(name="attention, 64 x 2048", op="attn", seqs=64, ctx=2048, most=16, kv_heads=KVH, group=4, chain=False),
        # two long documents, chains of 32 rows without a mask
        dict(name="attention, 2 x 32001", op="attn", seqs=2, ctx=32001, most=32, kv_heads=KVH, group=4, chain=True),
        # the widest trees, over which the products weigh as much as the keys
        dict(name="attention, 48 x 1999 wide", op="attn", seqs=48, ctx=1999, most=64, kv_heads=KVH, group=4, chain=False),
        # the choice for one request's next token, with its penalties
        dict(name="constrain, 1 row", op="constrain", seqs=1, most=1, vocab=VOCAB, history=450, bias=4, grammar=0, fp32=False, keep=False),
        # one row each of a replica's requests, half of them under a grammar
        dict(name="constrain, 128 rows", op="constrain", seqs=128, most=1, vocab=VOCAB, history=4000, bias=30, grammar=2, fp32=False, keep=False),
        # trees of up to 32 rows, every row with the drafts that lead to it; the logits kept for a sampler, an odd vocabulary in fp32
        dict(name="constrain, 16 trees, fp32", op="constrain", seqs=16, most=32, vocab=99991, history=1000, bias=10, grammar=3, fp32=True, keep=True),
        # one user: the path and its rows in 32 layers
        dict(name="accept, 1 request", op="accept", seqs=1, ctx=450, most=8, layers=LAYERS, kv_heads=KVH),
        # a busy replica
        dict(name="accept, 64 requests", op="accept", seqs=64, ctx=63, most=48, layers=LAYERS, kv_heads=KVH),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["maps", "attn", "attn", "constrain", "constrain", "accept"])
    if op == "maps":
        return dict(op=op, seqs=_log_int(rng, 1, 512), ctx=_log_int(rng, 1, 8000), most=_log_int(rng, 1, 64), tree=rng.random() < 0.7, pad=rng.choice([0, 1, 300]))
    if op == "attn":
        kv_heads, group = rng.choice([(8, 4), (8, 4), (4, 4), (1, 8), (5, 2), (8, 1)])
        most = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 16, 32000)
        seqs = _log_int(rng, 1, max(1, min(64, 64 * 2048 // ctx, 48 * 2000 * 64 // (ctx * most))))
        return dict(op=op, seqs=seqs, ctx=ctx, most=most, kv_heads=kv_heads, group=group, chain=rng.random() < 0.3)
    if op == "constrain":
        most = rng.choice([1, 1, rng.randint(2, 32)])
        return dict(op=op, seqs=_log_int(rng, 1, 128 // (1 if most == 1 else 16)), most=most, vocab=_log_int(rng, 100, 131072), history=_log_int(rng, 1, 8000),
                    bias=rng.choice([0, 7, 300]), grammar=rng.choice([0, 1, 2]), fp32=rng.random() < 0.4, keep=rng.random() < 0.4)
    return dict(op=op, seqs=_log_int(rng, 1, 48), ctx=_log_int(rng, 1, 70), most=_log_int(rng, 1, 64), layers=_log_int(rng, 1, 32), kv_heads=rng.choice([1, 4, 8]))


# ------------------------------------------------------------------ lengths of a case
def _spread(n, lo, hi):
    """n lengths between lo and hi, the largest first, the others in no order."""
    v = [lo + (hi - lo) * ((i * 37) % n) // max(1, n - 1) for i in range(n)]
    return [hi] + v[1:]


def _rows(case):
    return _spread(case["seqs"], 1, case["most"])


def _contexts(case):
    return _spread(case["seqs"], case["ctx"] // 8, case["ctx"])


def _pages(lens):
    return [(n + PAGE - 1) // PAGE for n in lens]


def work(case):
    n = _rows(case)
    T, S = sum(n), case["seqs"]
    if case["op"] == "maps":
        ctx = _contexts(case)
        new = sum(_pages([c + k for c, k in zip(ctx, n)])) - sum(_pages(ctx))
        words = (case["most"] + 31) // 32 if case["tree"] else 0
        return dict(bytes=4 * (7 * S + 2 * new + (4 if case["tree"] else 3) * (T + case["pad"]) + words * (T + case["pad"])), flops=0)
    if case["op"] == "attn":
        ctx, heads = _contexts(case), case["kv_heads"] * case["group"]
        keys = sum(c + k for c, k in zip(ctx, n))
        return dict(bytes=keys * case["kv_heads"] * 2 * D * 2 + 2 * T * heads * D * 2, flops=4 * D * heads * sum(c * k for c, k in zip(ctx, n)))
    if case["op"] == "constrain":
        V, size = case["vocab"], 4 if case["fp32"] else 2
        masks = sum(_under_grammar(case, r) for r in range(T)) * ((V + 31) // 32) * 4
        return dict(bytes=T * V * size * (2 if case["keep"] else 1) + masks + 4 * sum(_histories(case)) + 8 * S * case["bias"] + 4 * T, flops=0)
    # a third of the tree's depth is confirmed, about ln(rows); all of the path but its first row moves
    moved = sum(min(PATH, 1 + int(math.log(k))) - 1 for k in n)
    return dict(bytes=2 * moved * case["layers"] * 2 * case["kv_heads"] * D * 2 + 4 * (3 * T + S * (4 + 2 * PATH)), flops=0)


def _histories(case):
    return _spread(case["seqs"], case["history"] // 8, case["history"])


def _under_grammar(case, row):
    return case["grammar"] > 0 and row % case["grammar"] == 0


# ------------------------------------------------------------------ inputs
def _ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32).to(DEV)


def _trees(rng, n):
    """Parents of the rows of each tree, one tree behind the other: any row in front, so that depths go like a drafter's trees."""
    return np.concatenate([np.where(np.arange(k) == 0, -1, (rng.random(k) * np.arange(k)).astype(np.int64)) for k in n])


def _ancestors(parents, starts, bits):
    """Truth values [rows, bits]: which rows of its own request lead to a row, itself among them."""
    T = len(parents)
    seq = np.searchsorted(starts, np.arange(T), side="right") - 1
    first = starts[seq]
    up = np.where(parents < 0, T, first + parents)
    seen = np.zeros((T + 1, bits), dtype=bool)
    seen[np.arange(T), np.arange(T) - first] = True
    up = np.append(up, T)
    for _ in range(max(1, bits - 1).bit_length()):
        seen |= seen[up]
        up = up[up]
    return seen[:T]


def _packed(truth):
    """Truth values [rows, bits] as int32 words [rows, bits / 32]."""
    rows, bits = truth.shape
    full = np.zeros((rows, (bits + 31) // 32 * 32), dtype=np.uint8)
    full[:, :bits] = truth
    return np.packbits(full, axis=1, bitorder="little").view(np.int32)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = _rows(case)
    starts = np.concatenate([[0], np.cumsum(n)])
    st = dict(case=case, starts=_ints(starts), n=n)
    parents = _trees(rng, n)
    st["parents"] = _ints(parents)
    if case["op"] == "maps":
        ctx = _contexts(case)
        held, need = _pages(ctx), _pages([c + k for c, k in zip(ctx, n)])
        total = sum(need)
        order = rng.permutation(total + 8)
        width = max(need)
        tables = np.zeros((case["seqs"], width), dtype=np.int64)
        at = 0
        for s, h in enumerate(held):
            tables[s, :h] = order[at:at + h]
            at += h
        padded = np.append(parents, np.full(case["pad"], -1))
        return st | dict(ctx=_ints(ctx), new=_ints(n), held=_ints(held), tables=_ints(tables), free=_ints(np.append(order[:3], order[at:])), cursor=_ints([3]),
                         rows=int(starts[-1]) + case["pad"], parents=_ints(padded) if case["tree"] else None, words=(case["most"] + 31) // 32 if case["tree"] else 0)
    if case["op"] == "attn":
        ctx, heads, kvh = _contexts(case), case["kv_heads"] * case["group"], case["kv_heads"]
        need = _pages([c + k for c, k in zip(ctx, n)])
        order, tables = rng.permutation(sum(need)), np.zeros((case["seqs"], max(need)), dtype=np.int64)
        at = 0
        for s, h in enumerate(need):
            tables[s, :h] = order[at:at + h]
            at += h
        words = (case["most"] + 31) // 32
        return st | dict(ctx=_ints(ctx), tables=_ints(tables), masks=None if case["chain"] else _ints(_packed(_ancestors(parents, starts, words * 32))),
                         qkv=torch.randn(int(starts[-1]), (heads + 2 * kvh) * D, generator=gen, device=DEV).bfloat16(),
                         kv=torch.randn(sum(need), 2, kvh, PAGE, D, generator=gen, device=DEV, dtype=torch.bfloat16),
                         max_tree=case["most"], max_ctx=case["ctx"])
    if case["op"] == "constrain":
        S, V, T = case["seqs"], case["vocab"], int(starts[-1])
        hist = _histories(case)
        # text repeats itself: tokens by a power of a uniform number, and the logits lean towards what was said
        text = ((rng.random(sum(hist)) ** 3) * V).astype(np.int64)
        words = (case["most"] + 31) // 32
        logits = torch.randn(T, V, generator=gen, device=DEV) * 2.5
        seq = np.repeat(np.arange(S), n)
        hist_starts = np.concatenate([[0], np.cumsum(hist)])
        liked = [(r, text[hist_starts[s] + rng.integers(0, hist[s], 3)]) for r, s in enumerate(seq) if hist[s]]
        if liked:
            at = torch.tensor(np.repeat([r for r, _ in liked], 3)).to(DEV), torch.tensor(np.concatenate([t for _, t in liked])).to(DEV)
            logits[at] = logits[at] + 6
        some = min(case["bias"], V)
        first, step = rng.integers(0, V, S), max(1, V // max(1, some))
        ids = (first[:, None] + np.arange(some)[None, :] * step) % V      # no token twice
        index = np.array([r if _under_grammar(case, r) else -1 for r in range(T)])
        allow = None
        if case["grammar"]:
            allow = torch.randint(-2**31, 2**31 - 1, (T, (V + 31) // 32), generator=gen, device=DEV, dtype=torch.int32)
            allow &= torch.randint(-2**31, 2**31 - 1, allow.shape, generator=gen, device=DEV, dtype=torch.int32)
        return st | dict(logits=logits if case["fp32"] else logits.bfloat16(), history=_ints(text), hist_starts=_ints(hist_starts), prompt_lens=_ints([h // 3 for h in hist]),
                         drafts=_ints(rng.integers(0, V, T)), masks=_ints(_packed(_ancestors(parents, starts, words * 32))),
                         penalties=torch.tensor(np.stack([rng.choice([1.0, 1.1, 1.25], S), rng.choice([0.0, 0.5, -0.25], S), rng.choice([0.0, 0.125, 0.3], S)], 1), dtype=torch.float32).to(DEV),
                         bias=(_ints(np.arange(S + 1) * some), _ints(ids.reshape(-1)), torch.tensor(rng.uniform(-5, 5, S * some), dtype=torch.float32).to(DEV)) if some else None,
                         allow=allow, allow_rows=_ints(index) if case["grammar"] else None)
    ctx, kvh, T = _contexts(case), case["kv_heads"], int(starts[-1])
    need = _pages([c + k for c, k in zip(ctx, n)])
    order, tables = rng.permutation(sum(need)), np.zeros((case["seqs"], max(need)), dtype=np.int64)
    at = 0
    for s, h in enumerate(need):
        tables[s, :h] = order[at:at + h]
        at += h
    # the drafter is right along the way to some row of the tree
    drafts, ids = rng.integers(0, VOCAB, T), rng.integers(0, VOCAB, T)
    for s, k in enumerate(n):
        row = int(rng.integers(0, k))
        while row > 0:
            above = int(parents[starts[s] + row])
            ids[starts[s] + above] = drafts[starts[s] + row]
            row = above
    return st | dict(ctx=_ints(ctx), tables=_ints(tables), drafts=_ints(drafts), ids=_ints(ids),
                     kv=torch.randn(case["layers"], sum(need), 2, kvh, PAGE, D, generator=gen, device=DEV, dtype=torch.bfloat16))


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if own:
        return _own(st)
    return dict(maps=_plain_maps, attn=_plain_attn, constrain=_plain_constrain, accept=_plain_accept)[case["op"]](st)


def _own(st):
    from kubeai_b200 import ops
    op = st["case"]["op"]
    if op == "maps":
        m = ops.step_maps(st["ctx"], st["new"], st["held"], st["tables"], st["free"], st["cursor"], st["rows"], parents=st["parents"], words=st["words"])
        return dict(tables=st["tables"], starts=m.starts, positions=m.positions, slots=m.slots, seqs=m.seqs, held=m.held, cursor=m.cursor, status=m.status,
                    **(dict(masks=m.masks) if st["words"] else {}))
    if op == "attn":
        heads = st["case"]["kv_heads"] * st["case"]["group"]
        return ops.paged_attn_tree(st["qkv"], st["kv"], st["tables"], st["starts"], st["ctx"], st["masks"], heads, st["case"]["kv_heads"], st["max_tree"], max_ctx=st["max_ctx"])
    if op == "constrain":
        ids, out = ops.constrain(st["logits"], starts=st["starts"], history=st["history"], hist_starts=st["hist_starts"], prompt_lens=st["prompt_lens"],
                                 drafts=st["drafts"], masks=st["masks"], penalties=st["penalties"], bias=st["bias"], allow=st["allow"], allow_rows=st["allow_rows"],
                                 out=torch.float32 if st["case"]["keep"] else None)
        return dict(ids=ids, logits=out) if st["case"]["keep"] else dict(ids=ids)
    a = ops.tree_accept(st["ids"], st["drafts"], st["parents"], st["starts"], st["ctx"], st["tables"], st["kv"], PATH)
    return dict(accepted=a.accepted, path=a.path, tokens=a.tokens, ctx=a.ctx_lens, kv=st["kv"])


# ------------------------------------------------------------------ plain forms
def _request_of(starts, rows):
    """The request of each of `rows` rows; the number of requests for rows behind the last one."""
    return torch.searchsorted(starts[1:].contiguous(), torch.arange(rows, device=DEV), right=True)


def _bits(words):
    """int32 [rows, words] as truth values [rows, 32 words]."""
    return ((words[:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).bool().flatten(1)


def _plain_maps(st):
    ctx, new, held, tables, T, words = (st["ctx"].long(), st["new"].long(), st["held"].long(), st["tables"], st["rows"], st["words"])
    S = len(ctx)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    need = ((ctx + new + PAGE - 1) // PAGE - held).clamp(min=0)
    off = need.cumsum(0) - need
    fits = st["cursor"].long() + off + need <= len(st["free"])
    need = need * fits
    # the new pages, one row of the grid for each request
    k = torch.arange(tables.shape[1], device=DEV)[None, :] - held[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    page = st["free"].long()[(st["cursor"].long() + off[:, None] + k).clamp(0, len(st["free"]) - 1)]
    tables.copy_(torch.where(fresh, page, tables.long()).int())
    seq = _request_of(starts, T)
    real = seq < S
    s = seq.clamp(max=S - 1)
    i = torch.arange(T, device=DEV) - starts[s]
    at = (ctx[s] + i).clamp(0, tables.shape[1] * PAGE - 1)
    slots = torch.where(real & fits[s], tables.long()[s, at // PAGE] * PAGE + at % PAGE, -1)
    out = dict(tables=tables, starts=starts.int(), slots=slots.int(), seqs=torch.where(real, seq, -1).int(), held=(held + need).int(),
               cursor=(st["cursor"] + need.sum()).int(), status=(~fits).int())
    depth = i
    if words:
        # ancestors: what a row sees, and what its parent sees, and so on, twice as far each time
        up = torch.where(real & (st["parents"] >= 0), starts[s] + st["parents"].long(), T)
        up = torch.cat([up, up.new_full((1,), T)])
        seen = torch.zeros(T + 1, words * 32, dtype=torch.bool, device=DEV)
        seen[:T].scatter_(1, i.clamp(0, words * 32 - 1)[:, None], real[:, None])
        for _ in range((words * 32 - 1).bit_length()):
            seen, up = seen | seen[up], up[up]
        seen = seen[:T] & real[:, None]
        depth = seen.sum(1) - 1
        value = (seen.view(T, words, 32).long() << torch.arange(32, device=DEV)).sum(2)
        out["masks"] = torch.where(value >= 2**31, value - 2**32, value).int()
    out["positions"] = torch.where(real & fits[s], ctx[s] + depth, 0).int()
    return out


def _plain_attn(st):
    case, starts, ctx = st["case"], st["starts"].long(), st["ctx"].long()
    kvh, G, S, T = case["kv_heads"], case["group"], case["seqs"], st["qkv"].shape[0]
    seq = _request_of(starts, T)
    i, most = torch.arange(T, device=DEV) - starts[seq], case["most"]
    # every request as wide as the widest
    q = torch.zeros(S, most, kvh, G, D, device=DEV)
    q[seq, i] = st["qkv"][:, :kvh * G * D].float().view(T, kvh, G, D)
    k, v = (st["kv"][:, w][st["tables"].long()].transpose(2, 3).reshape(S, -1, kvh, D).float() for w in (0, 1))      # [request, key, head, dimension]
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(S, kvh, G * most, D), k.permute(0, 2, 3, 1)).view(S, kvh, G, most, -1) * D ** -0.5
    key = torch.arange(k.shape[1], device=DEV)
    j = key[None, :] - ctx[:, None]                                  # a key's number among the drafts
    if st["masks"] is None:
        drafted = (j[:, None, :] >= 0) & (j[:, None, :] <= torch.arange(most, device=DEV)[None, :, None])
    else:
        bits = torch.zeros(S, most, st["masks"].shape[1] * 32, dtype=torch.bool, device=DEV)
        bits[seq, i] = _bits(st["masks"])
        inside = (j >= 0) & (j < bits.shape[2])
        drafted = bits.gather(2, j.clamp(0, bits.shape[2] - 1)[:, None, :].expand(S, most, -1)) & inside[:, None, :]
    seen = (j < 0)[:, None, :] | drafted
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(S, kvh, G * most, -1), v.transpose(1, 2)).view(S, kvh, G, most, D) / torch.where(total == 0, 1.0, total)
    return y.permute(0, 3, 1, 2, 4)[seq, i].reshape(T, kvh * G * D).bfloat16()


def _plain_constrain(st):
    x, starts = st["logits"].float(), st["starts"].long()
    T, V = x.shape
    S = st["case"]["seqs"]
    seq = _request_of(starts, T)
    # how often a request said a token, and a row's ancestors draft it
    ends = st["hist_starts"].long()
    at = torch.arange(len(st["history"]), device=DEV)
    who = torch.searchsorted(ends[1:].contiguous(), at, right=True)
    said = at - ends[who] >= st["prompt_lens"].long()[who]
    anywhere, count = torch.zeros(S, V, device=DEV), torch.zeros(S, V, device=DEV)
    cell = who, st["history"].long()
    anywhere.index_put_(cell, torch.ones(len(at), device=DEV), accumulate=True)
    count.index_put_(cell, said.float(), accumulate=True)
    anywhere, count = anywhere[seq], count[seq]
    row, j = _bits(st["masks"]).nonzero(as_tuple=True)
    cell = row, st["drafts"].long()[starts[seq[row]] + j]
    ones = torch.ones(len(row), device=DEV)
    anywhere.index_put_(cell, ones, accumulate=True)
    count.index_put_(cell, ones, accumulate=True)
    rho, pi, phi = st["penalties"][seq].unbind(1)
    x = torch.where(anywhere > 0, torch.where(x > 0, x / rho[:, None], x * rho[:, None]), x)
    x = x - phi[:, None] * count
    x = x - pi[:, None] * (count > 0)
    if st["bias"] is not None:
        b = torch.zeros(S, V, device=DEV)
        b_starts, b_ids, b_values = st["bias"]
        b[_request_of(b_starts.long(), len(b_ids)), b_ids.long()] = b_values
        x = x + b[seq]
    allowed = torch.ones(T, V, dtype=torch.bool, device=DEV)
    if st["allow"] is not None:
        index = st["allow_rows"].long()
        allowed = _bits(st["allow"][index.clamp(min=0)])[:, :V] | (index < 0)[:, None]
    x = torch.where(allowed, x, -math.inf)
    best = x.amax(1, keepdim=True)
    ids = torch.where(allowed & (x == best), torch.arange(V, device=DEV), V).amin(1)
    ids = torch.where(ids == V, -1, ids).int()
    return dict(ids=ids, logits=x) if st["case"]["keep"] else dict(ids=ids)


def _plain_accept(st):
    ids, drafts, parents, starts, ctx, kv = (st["ids"].long(), st["drafts"].long(), st["parents"].long(), st["starts"].long(), st["ctx"].long(), st["kv"])
    S, T = len(ctx), len(ids)
    seq = _request_of(starts, T)
    i = torch.arange(T, device=DEV) - starts[seq]
    path = torch.full((S, PATH), -1, dtype=torch.long, device=DEV)
    path[:, 0] = 0
    # the next row of a path: the lowest one whose parent is the path's last and whose draft is what was chosen there; a step needs the one before
    for k in range(1, PATH):
        last = path[:, k - 1]
        wanted = torch.where(last >= 0, ids[starts[:-1] + last.clamp(min=0)], -1)
        hit = (parents == last[seq]) & (drafts == wanted[seq]) & (last[seq] >= 0) & (i > 0)
        nxt = torch.full((S,), T, dtype=torch.long, device=DEV).scatter_reduce_(0, seq, torch.where(hit, i, T), "amin")
        path[:, k] = torch.where(nxt < T, nxt, -1)
    real = path >= 0
    accepted = real.sum(1)
    tokens = torch.where(real, ids[starts[:-1, None] + path.clamp(min=0)], -1)
    # the path's rows, read whole before any is written
    s, k = real.nonzero(as_tuple=True)
    src, dst = ctx[s] + path[s, k], ctx[s] + k
    page = st["tables"].long()
    kv[:, page[s, dst // PAGE], :, :, dst % PAGE] = kv[:, page[s, src // PAGE], :, :, src % PAGE]
    return dict(accepted=accepted.int(), path=path.int(), tokens=tokens.int(), ctx=(ctx + accepted).int(), kv=kv)


# ------------------------------------------------------------------ the definitions, request by request
def exact(case, seed):
    st = prepare(case, seed)
    return dict(maps=_exact_maps, attn=_exact_attn, constrain=_exact_constrain, accept=_exact_accept)[case["op"]](st)


def _leading(parents, i):
    """The rows from row i up to the tree's root."""
    way = [i]
    while parents[way[-1]] >= 0:
        way.append(parents[way[-1]])
    return way


def _exact_maps(st):
    ctx, new, held, free = (st[k].tolist() for k in ("ctx", "new", "held", "free"))
    cursor, tables, words, T = st["cursor"].item(), st["tables"].cpu().numpy().copy(), st["words"], st["rows"]
    parents = st["parents"].tolist() if words else None
    rows, masks, starts, status = [], [], [0], []
    for s, (c, n) in enumerate(zip(ctx, new)):
        pages = -(-(c + n) // PAGE)
        while held[s] < pages:
            tables[s, held[s]] = free[cursor]
            held[s], cursor = held[s] + 1, cursor + 1
        tree = parents[starts[-1]:starts[-1] + n] if words else list(range(-1, n - 1))
        for i in range(n):
            way = _leading(tree, i) if words else range(i + 1)
            rows.append((c + len(way) - 1, int(tables[s, (c + i) // PAGE]) * PAGE + (c + i) % PAGE, s))
            if words:
                masks.append(np.isin(np.arange(words * 32), way))
        starts.append(starts[-1] + n)
        status.append(0)
    rows += [(0, -1, -1)] * (T - len(rows))
    positions, slots, seqs = zip(*rows)
    out = dict(tables=_ints(tables), starts=_ints(starts), positions=_ints(positions), slots=_ints(slots), seqs=_ints(seqs), held=_ints(held), cursor=_ints([cursor]), status=_ints(status))
    if words:
        masks += [np.zeros(words * 32, dtype=bool)] * (T - len(masks))
        out["masks"] = _ints(_packed(np.array(masks)))
    return out


def _exact_attn(st):
    case, starts, ctx = st["case"], st["starts"].tolist(), st["ctx"].tolist()
    kvh, G = case["kv_heads"], case["group"]
    heads = kvh * G
    out = torch.zeros(starts[-1], heads, D, dtype=torch.float64, device=DEV)
    for s, c in enumerate(ctx):
        a, b = starts[s], starts[s + 1]
        n = b - a
        pages = st["tables"][s, :(c + n + PAGE - 1) // PAGE].long()
        see = torch.ones(n, c + n, dtype=torch.bool, device=DEV)
        if st["masks"] is None:
            see[:, c:] = torch.ones(n, n, device=DEV).tril().bool()
        else:
            words = st["masks"][a:b].cpu().numpy().astype(np.uint32)
            see[:, c:] = torch.tensor((words[:, np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32)) & 1).bool().to(DEV)
        for h in range(kvh):
            k, v = (st["kv"][pages, w, h].reshape(-1, D)[:c + n].double() for w in (0, 1))
            q = st["qkv"][a:b, h * G * D:(h + 1) * G * D].double().view(n, G, D).transpose(0, 1)
            p = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill(~see, -math.inf), -1)
            out[a:b, h * G:(h + 1) * G] = (p @ v).transpose(0, 1)
    return out.view(starts[-1], heads * D)


def _exact_constrain(st):
    starts, hist, prompt = st["starts"].tolist(), st["hist_starts"].tolist(), st["prompt_lens"].tolist()
    T, V = st["logits"].shape
    x = st["logits"].double()
    text, drafts, parents = st["history"].cpu().numpy(), st["drafts"].tolist(), st["parents"].tolist()
    allow = st["allow"]
    index = st["allow_rows"].tolist() if allow is not None else [-1] * T
    for s, (rho, pi, phi) in enumerate(st["penalties"].double().tolist()):
        all_of, said = text[hist[s]:hist[s + 1]], text[hist[s] + prompt[s]:hist[s + 1]]
        any0, count0 = np.bincount(all_of, minlength=V), np.bincount(said, minlength=V)
        for r in range(starts[s], starts[s + 1]):
            way = [drafts[starts[s] + j] for j in _leading(parents[starts[s]:starts[s + 1]], r - starts[s])]
            more = np.bincount(way, minlength=V)
            seen = torch.tensor(any0 + more > 0).to(DEV)
            count = torch.tensor((count0 + more).astype(np.float64)).to(DEV)
            y = x[r]
            y = torch.where(seen, torch.where(y > 0, y / rho, y * rho), y) - phi * count - pi * (count > 0)
            if st["bias"] is not None:
                a, b = st["bias"][0][s:s + 2].tolist()
                y[st["bias"][1][a:b].long()] += st["bias"][2][a:b].double()
            if index[r] >= 0:
                bits = np.unpackbits(allow[index[r]].cpu().numpy().view(np.uint8), bitorder="little")[:V]
                y = y.masked_fill(torch.tensor(bits == 0).to(DEV), -math.inf)
            x[r] = y
    value, ids = x.max(1)
    ids = torch.where(x == value[:, None], torch.arange(V, device=DEV), V).amin(1)
    ids = torch.where(value == -math.inf, -1, ids).int()
    return dict(ids=ids, logits=x) if st["case"]["keep"] else dict(ids=ids)


def _exact_accept(st):
    ids, drafts, parents, starts, ctx = (st[k].tolist() for k in ("ids", "drafts", "parents", "starts", "ctx"))
    tables, kv = st["tables"].tolist(), st["kv"]
    was = kv.clone()
    paths, tokens = [], []
    for s, c in enumerate(ctx):
        a, n = starts[s], starts[s + 1] - starts[s]
        path = [0]
        while len(path) < PATH:
            nxt = [i for i in range(path[-1] + 1, n) if parents[a + i] == path[-1] and drafts[a + i] == ids[a + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        for k, i in enumerate(path):
            if i != k:
                kv[:, tables[s][(c + k) // PAGE], :, :, (c + k) % PAGE] = was[:, tables[s][(c + i) // PAGE], :, :, (c + i) % PAGE]
        paths.append(path + [-1] * (PATH - len(path)))
        tokens.append([ids[a + i] for i in path] + [-1] * (PATH - len(path)))
    accepted = [sum(i >= 0 for i in p) for p in paths]
    return dict(accepted=_ints(accepted), path=_ints(paths), tokens=_ints(tokens), ctx=_ints([c + k for c, k in zip(ctx, accepted)]), kv=kv)
