"""Attention of groups of requests, parts of more than 32 rows (row = token * group + head): the tensor cores' form, with one row tile (up to 128 rows) and with two, in whole items and in cut ones."""
import numpy as np
import pytest
import torch

from test_beam_step_gpu import D, PAGE, Batch, dev, near_attention

pytestmark = pytest.mark.gpu


def chains(rows, kvh=2, group=4, shared=64, own=20, seed=0):
    """Requests with so many rows each, behind shared pages and `own` tokens more or fewer."""
    return Batch([(len(rows), shared)], [n + own + 7 * s % 30 for s, n in enumerate(rows)], rows, kvh, group, seed=seed)


# one row tile (17 and 32 tokens of 4 heads), two (33 and 64), more than a block of 256 rows, and groups of so many rows
KINDS = {
    "17 tokens": lambda seed: chains([17, 9], seed=seed),
    "32 tokens": lambda seed: chains([32, 32], seed=seed),
    "33 tokens": lambda seed: chains([33, 50, 20], seed=seed),
    "64 tokens": lambda seed: chains([64], seed=seed),
    "100 tokens": lambda seed: chains([100, 70], seed=seed),
    "40 tokens of 8 heads": lambda seed: chains([40], kvh=1, group=8, seed=seed),
    "300 tokens of 1 head": lambda seed: chains([300], kvh=3, group=1, seed=seed),
    "behind 3000": lambda seed: chains([17, 64, 33], kvh=1, shared=3008, own=1500, seed=seed),
    "12 beams": lambda seed: Batch([(12, 400)], [1 + 5 * s for s in range(12)], [1] * 12, 2, 4, seed=seed),
    "70 beams": lambda seed: Batch([(70, 1600)], [1 + s % 40 for s in range(70)], [1] * 70, 1, 4, seed=seed),
}
kinds = pytest.mark.parametrize("kind", list(KINDS))


def token_of(b, s, p):
    """Where position p of request s lies: page and place."""
    return int(b.tables[s, p // PAGE]), p % PAGE


def check(b, **kw):
    """Every value against 64 bits: those that are a number within the rounding's bounds, the others the same infinity or NaN."""
    got = b.call(**kw).double().cpu().numpy().reshape(b.T, b.heads, D)
    with np.errstate(all="ignore"):
        want, size = b.want(kw.get("scale", D ** -0.5))
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    near_attention(torch.tensor(np.where(fine, got, 0)), np.where(fine, want, 0), np.where(fine, size, 0))
    return got


@kinds
def test_equal_values_come_out_as_they_are(kind):
    """Weights are rounded to bf16 and divided by the sum of the rounded ones, so what all values have in common has no part of their rounding: 3000 products and sums in fp32 are off by 2^-12 at
    most, and a bf16 value's neighbours are 2^-8 away.  One key outweighs the others by a factor that differs from row to row: the others' weights are all rounded the same way."""
    b = KINDS[kind](1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    b.kv[:, 0] = 0
    b.kv[:, 0, :, :, 0] = 1                            # every key's score is the query's first value ...
    for s in range(b.S):
        page, at = token_of(b, s, 5)
        b.kv[page, 0, :, at, 1] = 1                    # ... and one key has the second one more
    values = (1 + torch.rand(b.kvh, D, generator=gen, device="cuda")).bfloat16()
    b.kv[:, 1] = values[:, None]
    b.q = torch.zeros_like(b.q).view(b.T, b.heads, D)
    b.q[:, :, 0] = torch.randn(b.T, b.heads, generator=gen, device="cuda").bfloat16()
    b.q[:, :, 1] = (torch.rand(b.T, b.heads, generator=gen, device="cuda") * 40).bfloat16()
    b.q = b.q.view(b.T, -1)
    want = values.repeat_interleave(b.heads // b.kvh, 0).view(1, -1).expand(b.T, -1)
    got = b.call()
    assert torch.equal(got, want), (int((got != want).sum()), got.numel())


@kinds
@pytest.mark.parametrize("spread", [1, 8])
def test_scores_that_lie_near_and_far(kind, spread):
    """Score deviations of 1 and of 8, where few keys have a row's whole weight."""
    b = KINDS[kind](3)
    b.q = (b.q.float() * spread).bfloat16()
    check(b)


@kinds
@pytest.mark.parametrize("scale", [1e-6, 1.0, 30.0])
def test_scales(kind, scale):
    b = KINDS[kind](4)
    b.q = (b.q * (1 if scale < 1 else 2.0 ** -5)).bfloat16()
    check(b, scale=scale)


@kinds
def test_odd_values_that_no_row_sees(kind):
    """NaN and infinities behind the last token, in the rest of its page, and in pages of nobody."""
    b = KINDS[kind](5)
    want, size = b.want()
    used = np.zeros(b.pages, dtype=bool)
    for s in range(b.S):
        end = b.lens[s]
        used[b.tables[s, :-(-end // PAGE)]] = True
        if end % PAGE:
            page = int(b.tables[s, end // PAGE])
            b.kv[page, 0, :, end % PAGE:] = float("nan")
            b.kv[page, 1, :, end % PAGE:] = float("inf")
    b.kv[dev(~used, torch.bool)] = float("nan")
    near_attention(b.call(), want, size)


@kinds
@pytest.mark.parametrize("at", ["values", "keys", "both ends"])
def test_odd_values_that_some_rows_see(kind, at):
    """In the middle of a request's own rows: rows in front of it have no part of it, those behind it the infinity or NaN."""
    b = KINDS[kind](6)
    for s in range(b.S):
        n, first = b.rows[s], b.lens[s] - b.rows[s]
        places = [first + n // 2] if at != "both ends" else [first, first + n - 1]
        for p in places:
            page, i = token_of(b, s, p)
            if at == "keys":
                b.kv[page, 0, 0, i, 3] = float("nan")
            else:
                b.kv[page, 1, :, i, 5] = float("inf")
                b.kv[page, 1, :, i, 70] = float("-inf")
                b.kv[page, 1, 0, i, 9] = float("nan")
        if at == "values" and n > 4:                   # another sign further on: rows that see both have none
            page, i = token_of(b, s, first + n - 2)
            b.kv[page, 1, :, i, 70] = float("inf")
    check(b)


def test_odd_values_in_items_one_behind_the_other():
    """A CTA's items of one and of two row tiles in turn, short and with odd values in each: behind one of two tiles comes one without scores for the second group, and another with odd values."""
    rows = [64, 9, 40, 17, 12, 64, 20, 33] * 10
    b = Batch([(8, 16)] * 10, [n + 2 + 11 * s % 60 for s, n in enumerate(rows)], rows, 4, 4, seed=7)
    for s in range(0, b.S, 3):
        first = b.lens[s] - b.rows[s]
        for k, dim in ((1, 3), (b.rows[s] // 2, 40), (b.rows[s] - 1, 100)):
            page, i = token_of(b, s, first + k)
            b.kv[page, 1, :, i, dim] = float("inf") if s % 2 else float("nan")
    check(b)


@kinds
def test_pages_that_the_cache_does_not_have_read_as_zeros(kind):
    b = KINDS[kind](8)
    b.tables[:, 1] = b.pages + 5                       # a shared one
    for s in range(b.S):
        b.tables[s, (b.lens[s] - 1) // PAGE] = (-1, b.pages, 1 << 30, -2 ** 31)[s % 4]      # everybody's last
    check(b)


@kinds
def test_the_same_bits_in_a_graph_and_on_two_streams(kind):
    b, c = KINDS[kind](9), KINDS[kind](10)
    from kubeai_b200 import ops
    maps = [[dev(v) for v in (x.tables, x.starts, x.ctx, x.group_starts, x.shared)] for x in (b, c)]
    call = lambda x, m: ops.paged_attn_shared(x.q, x.kv, *m, x.heads, x.kvh, max(x.rows), max_ctx=max(x.ctx))      # noqa: E731
    first = [call(x, m).clone() for x, m in zip((b, c), maps)]
    sides = [torch.cuda.Stream() for _ in maps]
    torch.cuda.synchronize()
    again = []
    for _ in range(4):
        for x, m, f, side in zip((b, c), maps, first, sides):
            with torch.cuda.stream(side):
                again.append((call(x, m), f))
    torch.cuda.synchronize()
    assert all(torch.equal(y, f) for y, f in again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = [call(x, m) for x, m in zip((b, c), maps)]
    for _ in range(3):
        for y in kept:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, f) for y, f in zip(kept, first))


# 256 requests of 768 rows, of which one has 512: most rows times requests would pass 32 bits
def portion(ctx, own, seed, groups=8):
    rows = [512] + [2] * 128 + [0] * 127
    return Batch([(32, ctx)] * groups, [own + n + s % 9 for s, n in enumerate(rows)], rows, 8, 4, seed=seed, width=8192)


def test_one_long_portion_among_many_requests():
    b = portion(32, 3, 11)
    want, size = b.want()
    near_attention(b.call(), want, size)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(b.q)
    from kubeai_b200 import ops
    maps = [dev(v) for v in (b.tables, b.starts, b.ctx, b.group_starts, b.shared)]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.paged_attn_shared(b.q, b.kv, *maps, b.heads, b.kvh, 512, out=out)
    for _ in range(2):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        near_attention(out, want, size)
    # no groups
    near_attention(b.call(group_starts=dev([0]), shared=dev(np.zeros(0))), want, size)


@pytest.mark.parametrize("starts", [[0, 512] * 128 + [0], [768] + [0] * 256, [0, 512, 511] + [768] * 254, [-1] + [768] * 256, [0] * 256 + [769]])
def test_a_long_portion_without_order_is_nobodys(starts):
    b = portion(32, 3, 12)
    assert not b.call(starts=dev(starts)).any()
    kept = torch.full_like(b.q, 7.0)
    assert (b.call(starts=dev(starts), out=kept) == 7).all()
