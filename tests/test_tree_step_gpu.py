"""The four operations of a verification step of drafted tokens, each against its plain form, and a run of them together."""
import numpy as np
import pytest
import torch

import tree_step_util as U

pytestmark = pytest.mark.gpu


def ints(v, device="cuda"):
    return torch.tensor(np.asarray(v, dtype=np.int64).astype(np.int32)).to(device)


def tables_for(rng, lens, spare=0):
    """Shuffled pages for sequences of these lengths: tables (unused entries name no page), and how many pages there are."""
    need = [U.pages(n) for n in lens]
    order = rng.permutation(sum(need) + spare)
    tables, at = np.full((len(lens), max([1, *need])), -7), 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at:at + n]
        at += n
    return tables, sum(need) + spare


# ------------------------------------------------------------------ maps
def check_maps(ctx, new, held, tables, free, cursor, rows, parents=None, words=0, inplace=False):
    from kubeai_b200 import ops
    want = U.maps(ctx, new, held, tables, free, cursor, rows, parents, words)
    d_tables, d_held, d_cursor = ints(tables), ints(held), ints([cursor])
    got = ops.step_maps(ints(ctx), ints(new), d_held, d_tables, ints(free), d_cursor, rows, parents=None if parents is None else ints(parents), words=words, inplace=inplace)
    for name in ("starts", "positions", "slots", "seqs", "status", "held"):
        assert getattr(got, name).tolist() == list(want[name]), name
    assert got.cursor.tolist() == [want["cursor"]]
    assert np.array_equal(d_tables.cpu().numpy(), want["tables"])
    if words:
        assert np.array_equal(got.masks.cpu().numpy(), want["masks"])
    if inplace:
        assert d_held.tolist() == list(want["held"]) and d_cursor.tolist() == [want["cursor"]]
    else:
        assert d_held.tolist() == list(held) and d_cursor.tolist() == [cursor]
    return got


@pytest.mark.parametrize("S,most,tree,words,pad,inplace", [
    (1, 1, False, 0, 0, False), (1, 1, True, 1, 0, True), (1, 32, True, 1, 3, False), (1, 33, True, 2, 0, False), (3, 256, True, 8, 5, True), (2, 256, False, 8, 0, False),
    (31, 64, True, 2, 100, False), (257, 40, True, 2, 0, True), (1025, 3, False, 1, 9000, False), (8192, 2, False, 0, 0, False), (2, 9000, False, 0, 17, False), (5, 300, True, 0, 0, False)])
def test_maps_of_ragged_batches(S, most, tree, words, pad, inplace):
    rng = np.random.default_rng(S * 1000 + most)
    new = [int(v) for v in rng.integers(0, most + 1, S)]
    new[0] = most
    ctx = [int(v) for v in rng.integers(0, 100, S)]
    ctx[-1] = 0 if S > 1 else 16 * 3 - 1
    held = [U.pages(c) + int(rng.integers(0, 3)) for c in ctx]          # pages of drafts that were turned down are still held
    width = max(max(held), max(U.pages(c + n) for c, n in zip(ctx, new))) + 1
    total = sum(max(0, U.pages(c + n) - h) for c, n, h in zip(ctx, new, held))
    tables = rng.integers(0, 1 << 20, (S, width))
    parents = sum((U.random_tree(rng, n) for n in new), []) + [int(v) for v in rng.integers(-9, 9, pad)] if tree else None
    check_maps(ctx, new, held, tables, rng.permutation(total + 7) + (1 << 20), 4, sum(new) + pad, parents, words, inplace)


def test_maps_of_requests_that_do_not_fit():
    # ctx, rows, held: fits | negative rows | negative ctx | more than the table | fewer pages held than ctx needs | fits, nothing to do | tree too large | fits
    cases = [(5, 3, 1), (5, -2, 1), (-1, 2, 0), (100, 29, 7), (33, 1, 2), (16, 0, 1), (0, 33, 1), (15, 2, 1)]
    ctx, new, held = map(list, zip(*cases))
    rng = np.random.default_rng(0)
    got = check_maps(ctx, new, held, rng.integers(0, 99, (8, 8)), np.arange(100, 140), 0, sum(max(n, 0) for n in new) + 2, words=1)
    assert got.status.tolist() == [0, 2, 2, 2, 2, 0, 2, 0]


def test_maps_when_pages_or_rows_run_out():
    rng = np.random.default_rng(1)
    tables = rng.integers(0, 99, (6, 8))
    got = check_maps([0, 0, 0, 20, 0, 0], [16, 40, 1, 5, 0, 16], [0, 0, 0, 2, 0, 0], tables, np.arange(100, 103), 0, 78)
    assert got.status.tolist() == [0, 1, 1, 0, 0, 1] and got.cursor.tolist() == [1]
    got = check_maps([0, 0, 0], [4, 4, 4], [0, 0, 0], tables[:3], np.arange(100, 110), 2, 9)
    assert got.status.tolist() == [0, 0, 2] and got.starts.tolist() == [0, 4, 8, 9]
    check_maps([3], [40], [1], tables[:1], np.arange(0), 0, 40)            # no pages at all
    check_maps([3, 3], [4, 0], [1, 1], tables[:2], np.arange(0), 0, 4)     # none needed
    check_maps([3], [40], [1], tables[:1], np.arange(5), 5, 40)            # all taken


def test_maps_count_a_parent_behind_its_child_as_none():
    got = check_maps([7, 7], [4, 4], [1, 1], np.arange(8).reshape(2, 4), np.arange(10, 14), 0, 8, parents=[-1, 1, 0, -5, -1, 0, 1, 1 << 30], words=1)
    assert got.status.tolist() == [4, 4]


def test_maps_of_nothing():
    from kubeai_b200 import ops
    e = ints([])
    m = ops.step_maps(e, e, e, ints(np.zeros((0, 4))), e, ints([0]), 0)
    assert m.starts.tolist() == [0] and m.cursor.tolist() == [0]
    m = ops.step_maps(e, e, e, ints(np.zeros((0, 4))), e, ints([0]), 3, words=2)
    assert m.slots.tolist() == [-1] * 3 and not m.masks.any()


def test_maps_keep_to_their_columns_of_a_wider_table():
    from kubeai_b200 import ops
    wide = torch.full((3, 10), -3, dtype=torch.int32, device="cuda")
    ops.step_maps(ints([0, 0, 0]), ints([20, 1, 33]), ints([0, 0, 0]), wide[:, :4], ints(range(50, 60)), ints([0]), 54)
    assert wide.tolist() == [[50, 51] + [-3] * 8, [52] + [-3] * 9, [53, 54, 55] + [-3] * 7]


# ------------------------------------------------------------------ attention
def attention_case(seed, ctx, rows, kv_heads, group, masks="tree", words=None, poison=True, extra=0, wide=0, pages_at=None):
    """Inputs on the GPU and the truth values of the masks.  poison: NaN wherever the cache holds nothing."""
    rng = np.random.default_rng(seed)
    heads, T = kv_heads * group, sum(rows)
    tables, num = tables_for(rng, [c + n for c, n in zip(ctx, rows)], spare=2)
    starts = [0, *np.cumsum(rows).tolist()]
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(num, 2, kv_heads, 16, 128, generator=g).bfloat16()
    if poison:
        used = torch.zeros(num, 16, dtype=torch.bool)
        for s, n in enumerate(c + n for c, n in zip(ctx, rows)):
            for p in range(n):
                used[int(tables[s, p // 16]), p % 16] = True
        kv.masked_fill_(~used[:, None, None, :, None], float("nan"))
    qkv = torch.randn(T + extra, (heads + 2 * kv_heads) * 128 + wide, generator=g).bfloat16()
    see, words = [], words or max(1, -(-max([1, *rows]) // 32))
    for n in rows:
        if masks == "tree":
            see.append(U.ancestors(U.random_tree(rng, n)))
        elif masks == "random":       # any rows, none at all among them
            m = rng.random((n, n)) < 0.4
            m[::3] = False
            see.append(m)
        else:
            see.append(np.tril(np.ones((n, n), dtype=bool)))
    bits = None
    if masks != "chain":
        bits = np.concatenate([U.pack(m, words) for m in see] + [np.full((extra, words), -1, dtype=np.int32)])
    return dict(qkv=qkv, kv=kv, tables=tables, starts=starts, ctx=list(ctx), rows=list(rows), see=see, bits=bits, heads=heads, kv_heads=kv_heads, T=T)


def run_attention(c, max_ctx=0, out=None, max_tree=None):
    from kubeai_b200 import ops
    return ops.paged_attn_tree(c["qkv"].cuda(), c["kv"].cuda(), ints(c["tables"]), ints(c["starts"]), ints(c["ctx"]), None if c["bits"] is None else ints(c["bits"]),
                               c["heads"], c["kv_heads"], max_tree or max([1, *c["rows"]]), max_ctx=max_ctx, out=out)


def check_attention(c, got):
    q = c["qkv"][:c["T"], :c["heads"] * 128].double().numpy().reshape(-1, c["heads"], 128)
    kv = np.nan_to_num(c["kv"].double().numpy(), nan=0.0)
    want, size = U.attention(q, kv, c["tables"], c["starts"], c["ctx"], c["see"])
    got = got[:c["T"]].double().cpu().numpy().reshape(want.shape)
    # a weight rounded to bf16 (2^-8 of it) times its value, the result rounded to bf16 (2^-8 of it), and a 64th of the first for the 32-bit sums and exponentials
    tol = 2.0 ** -8 * (size * (1 + 1 / 64) + np.abs(want)) + 1e-30
    off = np.abs(got - want) / tol
    assert np.isfinite(got).all() and off.max() <= 1, f"off by {off.max():.3f} of the bound at {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.parametrize("ctx,rows,kv_heads,group,masks", [
    ([0], [1], 1, 4, "tree"), ([1], [1], 1, 1, "chain"), ([15], [2], 2, 4, "tree"), ([63], [1], 1, 8, "tree"), ([64], [1], 2, 2, "tree"), ([60], [5], 8, 4, "tree"),
    ([0], [64], 2, 4, "tree"), ([0], [200], 1, 4, "chain"), ([130], [65], 1, 4, "tree"), ([129], [256], 2, 4, "tree"), ([300], [33], 1, 8, "random"), ([77], [129], 1, 1, "random"),
    ([0], [31], 1, 4, "random"), ([1000], [16], 2, 4, "tree"), ([1023], [9], 8, 4, "tree"), ([5000], [3], 1, 8, "random"), ([9001], [64], 1, 4, "tree"), ([70], [63], 3, 2, "random"),
    ([450, 0, 17, 64, 1, 900], [8, 3, 0, 64, 1, 33], 2, 4, "tree"), ([5, 2000, 63, 128], [1, 40, 20, 0], 1, 8, "random"), ([16 * n for n in range(40)], [1 + n % 7 for n in range(40)], 2, 4, "tree"),
    ([33] * 5, [16, 17, 15, 1, 0], 4, 1, "chain"), ([100, 3], [128, 130], 1, 2, "chain")])
def test_attention(ctx, rows, kv_heads, group, masks):
    c = attention_case(len(ctx) + sum(rows), ctx, rows, kv_heads, group, masks)
    check_attention(c, run_attention(c))
    check_attention(c, run_attention(c, max_ctx=max(ctx)))


def test_attention_splits_are_the_same_bits_each_time():
    c = attention_case(3, [7000, 40], [40, 64], 2, 4)
    a, b = run_attention(c), run_attention(c)
    assert torch.equal(a, b)


def test_attention_of_masks_with_words_to_spare():
    c = attention_case(5, [100, 31], [33, 5], 1, 4, "random", words=8)
    check_attention(c, run_attention(c))
    check_attention(c, run_attention(c, max_tree=256))


def test_attention_leaves_other_rows_as_they_were_and_takes_strides():
    from kubeai_b200 import ops
    c = attention_case(6, [40, 70], [10, 21], 2, 4, extra=9, wide=64)
    out = torch.full((c["T"] + 9, c["heads"] * 128 + 24), 5.0, dtype=torch.bfloat16, device="cuda")
    got = run_attention(c, out=out)
    assert got is out and (out[c["T"]:] == 5).all() and (out[:, c["heads"] * 128:] == 5).all()
    check_attention(c, out[:, :c["heads"] * 128])
    # requests whose lengths are no requests are left out, the others are not
    starts, ctx = ints(c["starts"]), ints([40, 1 << 20])
    out.fill_(5)
    ops.paged_attn_tree(c["qkv"].cuda(), c["kv"].cuda(), ints(c["tables"]), starts, ctx, ints(c["bits"]), c["heads"], c["kv_heads"], 21, out=out)
    assert (out[10:] == 5).all() and not (out[:10, :c["heads"] * 128] == 5).all()
    for bad in ([0, 10, 9], [0, -1, 31], [0, 10, 41], [5, 3, 3]):
        out.fill_(5)
        ops.paged_attn_tree(c["qkv"].cuda(), c["kv"].cuda(), ints(c["tables"]), ints(bad), ints([40, -1]), ints(c["bits"]), c["heads"], c["kv_heads"], 21, out=out)
        assert (out[10:] == 5).all()


def test_attention_of_more_rows_than_the_tree_may_have_is_left_out():
    c = attention_case(7, [10, 10], [4, 9], 1, 4)
    got = run_attention(c, max_tree=8)
    assert (got[4:] == 0).all()
    c = c | dict(rows=[4, 0], starts=[0, 4, 4], T=4)
    check_attention(c, got)


@pytest.mark.parametrize("ctx,rows,kind", [([100], [40], "tree"), ([64], [64], "random"), ([0], [12], "random"), ([3000], [70], "tree")])
def test_what_a_row_does_not_see_has_no_part_in_it(ctx, rows, kind):
    """NaN and infinities in K and V of drafts reach the rows that see them and no others."""
    c = attention_case(8, ctx, rows, 2, 4, kind)
    n, bad = rows[0], [2, 5, min(11, rows[0] - 1)]
    for j, value in zip(bad, (float("nan"), float("inf"), float("-inf"))):
        p = ctx[0] + j
        c["kv"][int(c["tables"][0, p // 16]), 1, :, p % 16, 7:9] = value
        c["kv"][int(c["tables"][0, p // 16]), 0, :, p % 16, 3] = float("nan") if j == 2 else 1.0
    got = run_attention(c).float().cpu().view(n, c["heads"], 128)
    sees = c["see"][0][:, bad]
    clean = ~sees.any(1)
    assert clean.any() and not clean.all()
    # rows that see none of them: as without them
    d = c | dict(kv=c["kv"].nan_to_num(nan=0.0, posinf=0.0, neginf=0.0))
    want = run_attention(d).float().cpu().view(n, c["heads"], 128)
    assert torch.equal(got[torch.tensor(clean)], want[torch.tensor(clean)])
    for i in np.flatnonzero(~clean):
        if sees[i, 0]:
            assert got[i].isnan().all(), i                       # a key that is no number
        else:
            inf = {(True, False): float("inf"), (False, True): float("-inf")}.get((bool(sees[i, 1]), bool(sees[i, 2])))
            assert (got[i][:, 7:9] == inf).all() if inf is not None else got[i][:, 7:9].isnan().all(), i
            assert got[i][:, :7].isfinite().all() and got[i][:, 9:].isfinite().all(), i


def test_attention_reads_a_page_that_is_not_there_as_zeros():
    c = attention_case(9, [40, 20], [6, 6], 1, 4)
    c["tables"][0, 1], c["tables"][1, 0] = 1 << 28, -1
    got = run_attention(c)
    kv = torch.cat([c["kv"], torch.zeros(1, 2, 1, 16, 128, dtype=torch.bfloat16)])
    tables = c["tables"].copy()
    tables[0, 1] = tables[1, 0] = len(kv) - 1
    check_attention(c | dict(kv=kv, tables=tables), got)


def test_attention_far_into_a_large_cache():
    """Pages behind 2^31 values and 2^32 bytes."""
    from kubeai_b200 import ops
    c = attention_case(10, [200], [20], 8, 4)
    pages = c["kv"].shape[0]
    big = torch.zeros(72000, 2, 8, 16, 128, dtype=torch.bfloat16, device="cuda")
    at = np.array([71999 - 37 * i for i in range(pages)])
    big[torch.tensor(at).cuda()] = c["kv"].cuda()
    got = ops.paged_attn_tree(c["qkv"].cuda(), big, ints(at[c["tables"]]), ints(c["starts"]), ints(c["ctx"]), ints(c["bits"]), 32, 8, 20)
    assert torch.equal(got, run_attention(c))


def test_calls_of_no_requests_or_rows():
    from kubeai_b200 import ops
    c = attention_case(12, [5], [3], 1, 4)
    e, kv, none = ints([]), c["kv"].cuda(), ints(np.zeros((0, 4)))
    assert (ops.paged_attn_tree(c["qkv"].cuda(), kv, none, ints([0]), e, None, 4, 1, 3) == 0).all()
    assert (ops.paged_attn_tree(c["qkv"].cuda(), kv, ints(c["tables"]), ints([0, 3]), ints([5]), None, 4, 1, 0) == 0).all()
    assert ops.paged_attn_tree(c["qkv"].cuda()[:0], kv, ints(c["tables"]), ints([0, 0]), ints([5]), None, 4, 1, 3).shape == (0, 512)
    assert ops.constrain(torch.zeros(3, 9, device="cuda"), starts=ints([0]))[0].tolist() == [-1] * 3
    assert ops.constrain(torch.zeros(0, 9, device="cuda"))[0].shape == (0,)
    a = ops.tree_accept(e, e, None, ints([0]), e, none, None, 3)
    assert a.path.shape == (0, 3)
    a = ops.tree_accept(e, e, e, ints([0, 0]), ints([7]), ints([[1]]), None, 3)
    assert a.accepted.tolist() == [0] and a.ctx_lens.tolist() == [7] and a.path.tolist() == [[-1] * 3]


# ------------------------------------------------------------------ constrain
def constrain_case(seed, rows, V, history, f32, bias=0, grammar=None, drafts="tree", penalties=True, ld=0, repeat=False):
    rng = np.random.default_rng(seed)
    S, T = len(rows), sum(rows)
    rows_of = [list(range(sum(rows[:s]), sum(rows[:s + 1]))) for s in range(S)]
    x = torch.randn(T, V + ld, generator=torch.Generator().manual_seed(seed)) * 3
    x = x if f32 else x.bfloat16()
    low = 4 if repeat else V
    said = [[int(t) for t in rng.integers(-1 if V > 3 else 0, low + 1, h)] for h in history]      # some tokens that there are not
    see = [U.ancestors(U.random_tree(rng, n)) if drafts == "tree" else np.tril(np.ones((n, n), dtype=bool)) for n in rows]
    c = dict(x=x, rows=rows, rows_of=rows_of, V=V, said=said, prompt=[len(h) // 3 for h in said], see=see, drafts=[int(t) for t in rng.integers(0, low, T)] if drafts else None,
             penalties=np.stack([rng.choice([1.0, 1.1, 0.8], S), rng.choice([0.0, 0.5, -0.3], S), rng.choice([0.0, 0.3, 0.01], S)], 1).astype(np.float32) if penalties else None,
             bias=[[(int(t), float(np.float32(v))) for t, v in zip(rng.integers(0, V, bias), rng.normal(0, 4, bias))] for _ in range(S)], tree=drafts == "tree")
    allowed = np.ones((T, V), dtype=bool)
    if grammar == "some":
        allowed = rng.random((T, V)) < 0.2
        allowed[::4] = True
        allowed[1::5] = False
    elif grammar == "few":
        allowed = rng.random((T, V)) < 3.0 / V
    return c | dict(allowed=allowed, grammar=grammar)


def run_constrain(c, out=None, pick=True):
    from kubeai_b200 import ops
    x = c["x"].cuda()[:, :c["V"]]
    words = max(1, -(-max([1, *c["rows"]]) // 32))
    bias = None
    if any(c["bias"]):
        flat = [e for b in c["bias"] for e in b]
        bias = ints([0, *np.cumsum([len(b) for b in c["bias"]])]), ints([t for t, _ in flat]), torch.tensor([v for _, v in flat], dtype=torch.float32).cuda()
    allow = allow_rows = None
    if c["grammar"]:
        allow = ints(U.pack(c["allowed"], -(-c["V"] // 32)))
        free = c["allowed"].all(1)
        allow_rows = ints(np.where(free, -1, np.arange(len(free))))
    return ops.constrain(x, starts=ints([0, *np.cumsum(c["rows"])]), history=ints(sum(c["said"], [])), hist_starts=ints([0, *np.cumsum([len(h) for h in c["said"]])]),
                         prompt_lens=ints(c["prompt"]), drafts=None if c["drafts"] is None else ints(c["drafts"]),
                         masks=ints(np.concatenate([U.pack(m, words) for m in c["see"]])) if c["tree"] else None,
                         penalties=None if c["penalties"] is None else torch.tensor(c["penalties"]).cuda(), bias=bias, allow=allow, allow_rows=allow_rows, out=out, pick=pick)


def check_constrain(c, ids, y=None):
    args = c["rows_of"], c["said"], c["prompt"], c["drafts"], c["see"], c["penalties"], c["bias"], c["allowed"]
    x = c["x"][:, :c["V"]].float().numpy()
    want, want_ids = U.constrained(x, *args)
    if ids is not None:
        assert ids.tolist() == want_ids.tolist()
    if y is None:
        return
    if y.dtype is torch.float32:
        assert np.array_equal(y.cpu().numpy(), want, equal_nan=True)
    else:
        assert torch.equal(y.cpu().nan_to_num(nan=77.0), torch.tensor(want).bfloat16().nan_to_num(nan=77.0))
    # and in 64 bits: a quotient or product, two differences and a product, a sum, each rounded to 2^-24 of at most the largest of them (and bf16 to 2^-8)
    exact, _ = U.constrained(x, *args, exact=True)
    fine = np.isfinite(exact)
    size = np.abs(exact) + np.abs(x) * 1.3 + 30
    tol = 6 * 2.0 ** -24 * size + (2.0 ** -8 * np.abs(exact) if y.dtype is torch.bfloat16 else 0)
    assert (np.abs(y.double().cpu().numpy() - exact)[fine] <= tol[fine]).all()


@pytest.mark.parametrize("rows,V,history,f32,bias,grammar,drafts", [
    ([1], 1, [0], True, 0, None, None), ([1], 7, [3], False, 2, None, None), ([1], 128256, [450], False, 4, None, "tree"), ([1, 1, 1], 1000, [0, 50, 700], False, 0, "some", None),
    ([5, 0, 33], 999, [100, 20, 0], True, 9, "some", "tree"), ([64], 32001, [300], False, 300, None, "tree"), ([3, 2], 131073, [40, 4000], True, 5, "some", "tree"),
    ([40], 50, [500], False, 3, None, "chain"), ([2, 2, 2, 2], 8193, [9, 9, 9, 9], True, 1, "few", "chain"), ([1] * 130, 4097, [30] * 130, False, 2, "some", None),
    ([1], 262144, [2000], False, 20, "some", None), ([2], 393216, [100], True, 10, None, "tree"), ([300], 33, [5], True, 2, "some", "chain"), ([1, 1], 31, [4, 4], False, 0, "few", None)])
def test_constrain(rows, V, history, f32, bias, grammar, drafts):
    c = constrain_case(V + len(rows), rows, V, history, f32, bias, grammar, drafts)
    ids, none = run_constrain(c)
    assert none is None
    check_constrain(c, ids)
    check_constrain(c, *run_constrain(c, out=torch.float32))
    none, y = run_constrain(c, out=torch.bfloat16, pick=False)
    assert none is None
    check_constrain(c, None, y)


def test_constrain_counts_what_stands_often():
    """Thousands of the same few tokens, in the history and among the drafts."""
    c = constrain_case(1, [40, 3], 5000, [9000, 1], True, 30, None, "tree", repeat=True)
    check_constrain(c, *run_constrain(c, out=torch.float32))


@pytest.mark.parametrize("f32,ld", [(True, 1), (False, 3), (False, 8)])
def test_constrain_in_place_on_rows_of_a_wider_buffer(f32, ld):
    from kubeai_b200 import ops
    c = constrain_case(2, [4, 7], 1001, [30, 60], f32, 6, "some", "tree", ld=ld)
    wide = c["x"].cuda()
    x = wide[:, :1001]
    rest = wide[:, 1001:].clone()
    words = 1
    flat = [e for b in c["bias"] for e in b]
    free = c["allowed"].all(1)
    ids, y = ops.constrain(x, starts=ints([0, 4, 11]), history=ints(sum(c["said"], [])), hist_starts=ints([0, 30, 90]), prompt_lens=ints(c["prompt"]), drafts=ints(c["drafts"]),
                           masks=ints(np.concatenate([U.pack(m, words) for m in c["see"]])), penalties=torch.tensor(c["penalties"]).cuda(),
                           bias=(ints([0, 6, 12]), ints([t for t, _ in flat]), torch.tensor([v for _, v in flat], dtype=torch.float32).cuda()),
                           allow=ints(U.pack(c["allowed"], 32)), allow_rows=ints(np.where(free, -1, np.arange(11))), out=x)
    assert y is x and torch.equal(wide[:, 1001:], rest)
    check_constrain(c, ids, y)


def test_choice_of_ties_infinities_and_nothing():
    from kubeai_b200 import ops
    nan, inf = float("nan"), float("inf")
    rows = [[1.0, 3.0, 3.0, 2.0], [nan, -inf, nan, -inf], [-inf] * 4, [nan, -5.0, nan, -5.0], [-0.0, 0.0, -1.0, 0.0], [inf, nan, inf, 0.0], [1.0, 2.0, 3.0, 4.0], [2.0, 2.0, 2.0, 2.0]]
    x = torch.tensor(rows).cuda()
    allow = ints([[0b0000], [0b1110]])
    ids, y = ops.constrain(x, allow=allow, allow_rows=ints([-1, -1, -1, -1, -1, -1, 0, 1]), out=torch.float32)
    assert ids.tolist() == [1, 0, 0, 1, 0, 0, -1, 1]
    assert (y[6] == -inf).all() and y[7].tolist() == [-inf, 2.0, 2.0, 2.0] and y[0].tolist() == rows[0]
    assert ops.constrain(x.bfloat16(), allow=allow, allow_rows=ints([-1, 7, -9, -1, -1, -1, 0, 1]))[0].tolist() == [1, 0, 0, 1, 0, 0, -1, 1]      # masks there are not: none
    wide = torch.full((3, 100003), -2.0, device="cuda", dtype=torch.bfloat16)
    wide[0, 99000] = wide[0, 51] = wide[1, 100002] = wide[2, 8192] = wide[2, 16384] = 7.0
    assert ops.constrain(wide)[0].tolist() == [51, 100002, 8192]
    assert ops.constrain(torch.full_like(wide, nan))[0].tolist() == [0, 0, 0]


def test_constrain_leaves_rows_that_no_request_owns():
    from kubeai_b200 import ops
    x = torch.randn(6, 500, device="cuda")
    out = torch.full_like(x, 9.0)
    ids, _ = ops.constrain(x, starts=ints([0, 2, 4]), out=out)
    assert ids.tolist() == x.argmax(1)[:4].tolist() + [-1, -1] and (out[4:] == 9).all() and torch.equal(out[:4], x[:4])
    ids, _ = ops.constrain(x, starts=ints([3, 2, 99]))
    assert ids.tolist() == [-1] * 6


# ------------------------------------------------------------------ accept
def accept_case(seed, ctx, rows, layers, heads, right=0.7, chain=False):
    rng = np.random.default_rng(seed)
    T = sum(rows)
    tables, num = tables_for(rng, [c + n for c, n in zip(ctx, rows)], spare=1)
    parents = sum((list(range(-1, n - 1)) if chain else U.random_tree(rng, n) for n in rows), [])
    starts = [0, *np.cumsum(rows).tolist()]
    drafts, ids = rng.integers(0, 50, T), rng.integers(-1, 50, T)
    for s, n in enumerate(rows):          # the choice at a row is often what one of its children drafts
        for i in range(n - 1, 0, -1):
            p = parents[starts[s] + i]
            if p >= 0 and rng.random() < right:
                ids[starts[s] + p] = drafts[starts[s] + i]
    kv = torch.randn(layers, num, 2, heads, 16, 128, generator=torch.Generator().manual_seed(seed)).bfloat16()
    return dict(ids=ids, drafts=drafts, parents=parents, starts=starts, ctx=list(ctx), tables=tables, kv=kv)


@pytest.mark.parametrize("ctx,rows,layers,heads,path", [
    ([0], [1], 1, 1, 1), ([7], [8], 2, 8, 4), ([15, 16, 0, 100], [20, 1, 0, 64], 3, 2, 16), ([3] * 70, [1 + n % 40 for n in range(70)], 2, 1, 8), ([30], [256], 1, 4, 256),
    ([5, 900], [2000, 2048], 1, 1, 64), ([1, 2], [16, 31], 32, 8, 16)])
@pytest.mark.parametrize("chain", [False, True])
def test_accept(ctx, rows, layers, heads, path, chain):
    from kubeai_b200 import ops
    c = accept_case(sum(rows) + layers, ctx, rows, layers, heads, right=0.98 if chain else 0.7, chain=chain)
    want = U.accepted(c["ids"], c["drafts"], c["parents"], c["starts"], c["ctx"], c["tables"], c["kv"].view(torch.int16).numpy(), path)
    kv = c["kv"].cuda()
    got = ops.tree_accept(ints(c["ids"]), ints(c["drafts"]), None if chain else ints(c["parents"]), ints(c["starts"]), ints(c["ctx"]), ints(c["tables"]), kv, path)
    for name in ("accepted", "path", "tokens", "ctx_lens"):
        assert getattr(got, name).tolist() == want[name], name
    assert np.array_equal(kv.cpu().view(torch.int16).numpy(), want["kv"])
    # without a cache to move in
    again = ops.tree_accept(ints(c["ids"]), ints(c["drafts"]), None if chain else ints(c["parents"]), ints(c["starts"]), ints(c["ctx"]), ints(c["tables"]), None, path)
    assert again.path.tolist() == want["path"]


def test_accept_of_what_is_no_request_and_of_pages_that_are_not_there():
    from kubeai_b200 import ops
    c = accept_case(4, [10, 12, 3], [9, 9, 9], 2, 1, chain=True, right=1.0)
    tables = c["tables"].copy()
    tables[0, 1] = 1 << 27          # positions 16 .. 18 of request 0
    kv = c["kv"].cuda()
    ctx = [10, 1 << 30, -1]
    got = ops.tree_accept(ints(c["ids"]), ints(c["drafts"]), None, ints(c["starts"]), ints(ctx), ints(tables), kv, 16)
    assert got.accepted.tolist()[1:] == [0, 0] and got.ctx_lens.tolist()[1:] == ctx[1:] and (got.path[1:] == -1).all()
    assert torch.equal(kv.cpu().view(torch.int16), c["kv"].view(torch.int16))      # a chain's rows are where they stay
    # a tree whose path jumps over rows: moves from or to that page are left out
    parents, drafts, ids = [-1, 0, 0, 1, 2, 4, 4, 6, 6], list(range(9)), [2, 9, 4, 9, 6, 9, 8, 9, 9]
    got = ops.tree_accept(ints(ids), ints(drafts), ints(parents), ints([0, 9]), ints([10]), ints(tables[:1]), kv, 16)
    assert got.path.tolist()[0][:5] == [0, 2, 4, 6, 8] and got.accepted.tolist() == [5]
    want = c["kv"].clone()
    page, src = int(tables[0, 0]), [10, 12, 14]        # 16 and 18 lie on the page that is not there
    for k in (1, 2):
        want[:, page, :, :, 10 + k] = c["kv"][:, page, :, :, src[k]]
    assert torch.equal(kv.cpu().view(torch.int16), want.view(torch.int16))


def test_accept_in_some_layers_of_a_larger_cache():
    from kubeai_b200 import ops
    c = accept_case(11, [10, 3], [30, 30], 4, 2)
    want = U.accepted(c["ids"], c["drafts"], c["parents"], c["starts"], c["ctx"], c["tables"], c["kv"].view(torch.int16).numpy(), 16)
    kv = c["kv"].cuda()
    ops.tree_accept(ints(c["ids"]), ints(c["drafts"]), ints(c["parents"]), ints(c["starts"]), ints(c["ctx"]), ints(c["tables"]), kv[::2], 16)
    got = kv.cpu().view(torch.int16).numpy()
    assert np.array_equal(got[::2], want["kv"][::2]) and np.array_equal(got[1::2], c["kv"].view(torch.int16).numpy()[1::2])
