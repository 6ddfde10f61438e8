"""The operations of a step whose requests share their beginnings, against their plain forms in 64 bits."""
import math

import numpy as np
import pytest
import torch

import beam_step_util as plain

pytestmark = pytest.mark.gpu
D, PAGE, BF16 = 128, 16, 2.0 ** -8      # BF16: half a step, relative to the value


def dev(v, dtype=torch.int32):
    return torch.as_tensor(np.asarray(v)).to(dtype).cuda()


def wide(t):
    """The values as leading columns of a wider buffer, whose others are NaN or 77."""
    t = t if t.dim() == 2 else t.view(len(t), -1)
    big = torch.full((t.shape[0] + 2, t.shape[1] + 24), float("nan") if t.is_floating_point() else 77, dtype=t.dtype, device=t.device)
    big[:t.shape[0], :t.shape[1]] = t
    return big[:t.shape[0], :t.shape[1]]


# ------------------------------------------------------------------ norm and rotation
def near_rotated(got, want, size):
    """One rounding to bf16, and in front of it in fp32 two products of a norm's factor, a weight and a cosine whose angle was reduced exactly: 16 half steps of 2^-24 of each."""
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert (np.abs(got - want) <= BF16 * np.abs(want) + 2.0 ** -20 * size + 1e-40).all(), np.abs(got - want).max()


def turned(T, heads, kvh, dims, interleaved, norm, far, f32=False, seed=0, in_place=False, rows_apart=False, eps=1e-6, gain=1.0):
    from kubeai_b200 import ops
    rng, gen = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(T, (heads + 2 * kvh) * D, generator=gen, device="cuda") * 3).bfloat16()
    if rows_apart:
        qkv = wide(qkv)
    pages = T // PAGE + 3
    slots = rng.permutation(pages * PAGE)[:T]
    slots[::5] = -1
    if T > 3:
        slots[3] = pages * PAGE                       # a page that the cache does not have
    kv = torch.randn(pages, 2, kvh, PAGE, D, generator=gen, device="cuda").bfloat16() if kvh else torch.zeros(pages, 2, 0, PAGE, D, device="cuda").bfloat16()
    positions = rng.integers(0, far, T)
    positions[0] = far - 1
    freqs = 10000.0 ** (-np.arange(0, dims, 2) / max(dims, 1))
    w = lambda n: None if norm == "none" else torch.randn(*((n, D) if norm == "each" else (D,)), generator=gen, device="cuda").to(torch.float32 if f32 else torch.bfloat16)      # noqa: E731
    qw, kw = w(heads), w(kvh)
    was, before = kv.clone(), qkv.clone()
    out = ops.norm_rope_kvwrite(qkv, dev(positions), dev(slots), kv, heads, kvh, dev(freqs, torch.float64), gain=gain, q_norm=qw, k_norm=kw, eps=eps, interleaved=interleaved, out=qkv if in_place else None)
    x = before.double().cpu().numpy().reshape(T, heads + 2 * kvh, D)
    wide_of = lambda w: None if w is None else w.double().cpu().numpy()      # noqa: E731
    q, qs = plain.rotated(x[:, :heads], wide_of(qw), eps, positions, freqs, gain, interleaved)
    k, ks = plain.rotated(x[:, heads:heads + kvh], wide_of(kw), eps, positions, freqs, gain, interleaved)
    near_rotated(out[:, :heads * D].reshape(T, heads, D), q, qs)
    if in_place:
        assert out.data_ptr() == qkv.data_ptr() and torch.equal(qkv[:, heads * D:], before[:, heads * D:])
    else:
        assert torch.equal(qkv, before)
    keep = (slots >= 0) & (slots < pages * PAGE)
    page, off = slots[keep] // PAGE, slots[keep] % PAGE
    near_rotated(kv[page, 0, :, off], k[keep], ks[keep])
    assert torch.equal(kv[page, 1, :, off].double().cpu(), torch.tensor(x[keep][:, heads + kvh:]))
    rest = torch.ones(pages, PAGE, dtype=torch.bool, device="cuda")
    rest[page, off] = False
    assert torch.equal(kv.transpose(2, 3).transpose(1, 2)[rest], was.transpose(2, 3).transpose(1, 2)[rest])


@pytest.mark.parametrize("T,heads,kvh", [(1, 32, 8), (4, 8, 1), (33, 5, 5), (257, 64, 8), (3, 1, 1), (2, 0, 3), (2, 3, 0), (9, 100, 7)])
def test_rotation_of_head_layouts(T, heads, kvh):
    turned(T, heads, kvh, 128, False, "one", 4000)


@pytest.mark.parametrize("dims", [0, 2, 6, 8, 20, 64, 72, 96, 100, 126, 128])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_of_parts_of_a_head(dims, interleaved):
    turned(7, 6, 2, dims, interleaved, "each", 1000, rows_apart=True, gain=1.25)


@pytest.mark.parametrize("norm,f32", [("none", False), ("one", False), ("one", True), ("each", False), ("each", True)])
@pytest.mark.parametrize("in_place", [False, True])
def test_norms_and_places(norm, f32, in_place):
    turned(19, 8, 2, 64, False, norm, 1000, f32=f32, in_place=in_place, rows_apart=in_place)


@pytest.mark.parametrize("far", [1, 2, 1 << 20, 1 << 30, (1 << 31) - 1])
def test_angles_of_far_positions(far):
    """In 64 bits a position of 2^31 leaves 2^-22 of the angle; the tolerance's 2^-20 of the values has room for it."""
    turned(11, 4, 2, 128, False, "none", far)


def test_norm_of_zeros_and_of_one_norm_alone():
    from kubeai_b200 import ops
    kv, z, f = torch.zeros(1, 2, 1, PAGE, D).bfloat16().cuda(), torch.zeros(1, 3 * D).bfloat16().cuda(), dev([1.0], torch.float64)
    w = torch.ones(D).bfloat16().cuda()
    assert not ops.norm_rope_kvwrite(z, dev([5]), dev([2]), kv, 1, 1, f, q_norm=w, k_norm=w).any() and not kv.any()
    x = torch.randn(1, 3 * D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    q = ops.norm_rope_kvwrite(x, dev([0]), dev([2]), kv, 1, 1, f, k_norm=w)
    assert torch.equal(q, x[:, :D]) and torch.equal(kv[0, 1, 0, 2], x[0, 2 * D:]) and not torch.equal(kv[0, 0, 0, 2], x[0, D:2 * D])


def test_values_pass_as_they_are():
    from kubeai_b200 import ops
    kv, f = torch.zeros(1, 2, 1, PAGE, D).bfloat16().cuda(), dev([1.0], torch.float64)
    x = torch.zeros(1, 3 * D).bfloat16().cuda()
    x[0, 2 * D:] = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0] * 32).bfloat16()
    ops.norm_rope_kvwrite(x, dev([0]), dev([7]), kv, 1, 1, f)
    assert torch.equal(kv[0, 1, 0, 7].view(torch.int16), x[0, 2 * D:].view(torch.int16))


# ------------------------------------------------------------------ attention
def near_attention(got, out, size):
    """Weights are rounded to bf16 and divided by the sum of the rounded ones (twice half a step of the magnitudes), scores are fp32 sums of 128 products (2^-12 of a weight at these sizes), and
    the output is rounded once."""
    got = got.double().cpu().numpy().reshape(out.shape)
    off = np.abs(got - out) - ((2 * BF16 + 2.0 ** -12) * size + BF16 * np.abs(out) + 1e-30)
    assert (off <= 0).all(), (off.max(), np.argwhere(off > 0)[:5])


class Batch:
    """A step: groups of requests (members, shared tokens), each member's own tokens and rows; tables on random pages."""

    def __init__(self, groups, own, rows, kvh, group, seed=0, extra_pages=0, width=0):
        rng, gen = np.random.default_rng(seed), torch.Generator(device="cuda").manual_seed(seed)
        self.kvh, self.heads = kvh, kvh * group
        self.group_starts = np.concatenate([[0], np.cumsum([m for m, _ in groups])])
        self.shared = [p for _, p in groups]
        self.lens, at, names = [], 0, []
        S = int(self.group_starts[-1])
        for g, (m, p) in enumerate(groups):
            common = list(range(at, at + p // PAGE))
            at += p // PAGE
            for s in range(self.group_starts[g], self.group_starts[g + 1]):
                n = plain.pages(p + own[s]) - p // PAGE
                names.append(common + list(range(at, at + n)))
                self.lens.append(p + own[s])
                at += n
        self.pages = at + extra_pages
        order = rng.permutation(self.pages)
        width = max([width, 1] + [len(n) for n in names])
        self.tables = np.full((S, width), 1 << 30)
        for s, n in enumerate(names):
            self.tables[s, :len(n)] = order[n]
        self.rows, self.S, self.T = list(rows), S, sum(rows)
        self.starts = np.concatenate([[0], np.cumsum(rows)])
        self.ctx = [t - n for t, n in zip(self.lens, rows)]
        self.kv = torch.randn(self.pages, 2, kvh, PAGE, D, generator=gen, device="cuda").bfloat16()
        # a page's shared tokens are the same in all members' copies
        for g, (m, p) in enumerate(groups):
            if p % PAGE and m > 1:
                mine = dev(self.tables[self.group_starts[g]:self.group_starts[g + 1], p // PAGE], torch.long)
                self.kv[mine, :, :, :p % PAGE] = self.kv[mine[0], :, :, :p % PAGE].clone()
        self.q = torch.randn(self.T, self.heads * D, generator=gen, device="cuda").bfloat16()

    def call(self, max_rows=None, **kw):
        from kubeai_b200 import ops
        kw = dict(max_ctx=max(self.ctx + [0])) | kw
        return ops.paged_attn_shared(kw.pop("qkv", self.q), self.kv, kw.pop("tables", dev(self.tables)), kw.pop("starts", dev(self.starts)), kw.pop("ctx", dev(self.ctx)),
                                     kw.pop("group_starts", dev(self.group_starts)), kw.pop("shared", dev(self.shared)), self.heads, self.kvh, max(self.rows + [1]) if max_rows is None else max_rows, **kw)

    def want(self, scale=D ** -0.5):
        return plain.attention(self.q.double().cpu().numpy().reshape(self.T, self.heads, D), self.kv.double().cpu().numpy(), self.tables, self.starts, self.ctx, scale)

    def check(self, **kw):
        near_attention(self.call(**kw), *self.want(kw.get("scale", D ** -0.5)))


@pytest.mark.parametrize("kvh,group", [(8, 4), (1, 8), (2, 1), (3, 2), (1, 1), (4, 8)])
@pytest.mark.parametrize("shared", [0, 15, 16, 100, 333])
def test_beams_behind_a_prompt(kvh, group, shared):
    Batch([(4, shared), (3, shared // 2)], [1, 5, 16, 17, 40, 2, 33], [1] * 7, kvh, group, seed=shared).check()


@pytest.mark.parametrize("rows", [[1, 2, 3], [5, 1, 4], [17, 33, 64], [0, 2, 0]])
@pytest.mark.parametrize("group", [1, 4, 8])
def test_several_rows_of_a_request(rows, group):
    Batch([(3, 70)], [max(r, n) for r, n in zip(rows, (1, 40, 77))], rows, 2, group, seed=sum(rows)).check()


@pytest.mark.parametrize("members", [1, 2, 5, 40, 130])
def test_groups_of_many_requests(members):
    own = [1 + (i * 7) % 50 for i in range(members)]
    Batch([(members, 200)], own, [1] * members, 2, 4, seed=members).check()


@pytest.mark.parametrize("shared,own", [(5000, 3), (3, 5000), (2049, 2049), (16, 1), (1, 1)])
def test_long_and_short_parts(shared, own):
    Batch([(4, shared)], [own, own // 2 + 1, 1, own], [1] * 4, 1, 4, seed=shared).check()


@pytest.mark.parametrize("S,rows", [(257, [1]), (700, [0, 1, 3, 1]), (1500, [1, 0, 0])])
def test_more_requests_than_lie_in_shared_memory(S, rows):
    groups = [(7, 32)] * (S // 7) + ([(S % 7, 16)] if S % 7 else [])
    b = Batch(groups, [4 + s % 5 for s in range(S)], [rows[s % len(rows)] for s in range(S)], 2, 2, seed=S)
    out = torch.full((b.T, b.heads * D), 3.0, device="cuda").bfloat16()
    status = [2 if s % 11 == 5 else 0 for s in range(S)]      # some have no place in the cache
    got = b.call(status=dev(status), out=out)
    want, size = b.want()
    for s, no in enumerate(status):
        if no:
            want[b.starts[s]:b.starts[s + 1]], size[b.starts[s]:b.starts[s + 1]] = 3.0, 0.0
    assert got.data_ptr() == out.data_ptr()
    near_attention(got, want, size)


def test_long_chains_behind_a_document():
    Batch([(3, 3000), (2, 1000)], [40, 64, 70, 33, 90], [33, 64, 1, 7, 50], 2, 4, seed=3).check()


def test_groups_may_be_empty_or_leave_requests_out():
    b = Batch([(1, 40), (3, 64), (2, 100), (2, 0)], [5, 6, 7, 8, 9, 10, 11, 12], [1, 2, 1, 3, 1, 1, 2, 1], 2, 4, seed=4)
    want = b.want()
    for gs, shared in (([1, 1, 4, 4, 6], [0, 64, 10 ** 6, 100]), ([0, 0, 0], [5, 5]), ([8, 8], [64]), ([2, 4], [64]), ([0, 1, 4, 6, 8], [40, 64, 100, 0])):
        near_attention(b.call(group_starts=dev(gs), shared=dev(shared)), *want)
    near_attention(b.call(group_starts=dev([0]), shared=dev(np.zeros(0))), *want)


@pytest.mark.parametrize("gs,shared", [([4, 1, 6], [64, 64]), ([0, 99], [64]), ([-1, 4], [64]), ([1, 4], [-5]), ([1, 4], [10 ** 9]), ([1, 4], [-2 ** 31]), ([1, 4], [66])])
def test_groups_that_are_none_share_nothing_wrong(gs, shared):
    """Named tokens beyond what the first request has, group starts that descend or pass the requests: all still see their own tables.  (Two of three requests have what is named.)"""
    b = Batch([(1, 40), (3, 64), (2, 100)], [5, 6, 7, 8, 9, 10], [1, 2, 1, 3, 1, 1], 2, 4, seed=5)
    if shared[0] == 10 ** 9:      # whole pages that the first one has, which the others do not: a promise that the call makes
        b.ctx[1] = 64
        b.lens[1] = 66
    near_attention(b.call(group_starts=dev(gs), shared=dev(shared)), *b.want())


def test_a_member_with_fewer_tokens_than_are_shared_is_attended_alone():
    b = Batch([(3, 96)], [4, 5, 6], [1, 1, 1], 2, 4, seed=6)
    b.ctx[2], b.lens[2] = 50, 51
    b.check()


def test_what_is_left_out_stays_as_it_was():
    b = Batch([(3, 64), (3, 64)], [5, 6, 7, 8, 9, 10], [1, 2, 1, 3, 1, 1], 2, 4, seed=7)
    want, size = b.want()
    starts, ctx = b.starts, list(b.ctx)
    for s, kw in ((1, dict(status=dev([0, 1, 0, 0, 0, 0]))), (0, dict(status=dev([2, 0, 0, 0, 0, 0]))), (3, dict(max_rows=2)), (4, dict(ctx=dev(ctx[:4] + [-1] + ctx[5:]))), (3, dict(ctx=dev(ctx[:3] + [10 ** 6] + ctx[4:])))):
        for out in (None, torch.full_like(b.q, 7.0), wide(torch.full_like(b.q, 7.0))):
            got = b.call(out=out, **kw)
            mine = np.ones(b.T, dtype=bool)
            mine[starts[s]:starts[s + 1]] = False
            near_attention(got[dev(mine, torch.bool)], want[mine], size[mine])
            assert (got[dev(~mine, torch.bool)] == (0.0 if out is None else 7.0)).all()


def test_padded_rows_and_wide_buffers():
    b = Batch([(2, 48), (2, 20)], [3, 4, 5, 30], [1, 1, 2, 1], 2, 4, seed=8)
    want, size = b.want()
    padded = torch.cat([torch.full((3, b.q.shape[1]), float("nan"), device="cuda").bfloat16(), b.q, torch.full((6, b.q.shape[1]), float("nan"), device="cuda").bfloat16()])
    out = wide(torch.full_like(padded, 5.0))
    got = b.call(qkv=wide(padded), out=out, starts=dev(b.starts + 3))
    near_attention(got[3:3 + b.T], want, size)
    assert (got[:3] == 5).all() and (got[3 + b.T:] == 5).all()
    fresh = b.call(qkv=wide(padded), starts=dev(b.starts + 3))
    assert not fresh[:3].any() and not fresh[3 + b.T:].any() and torch.equal(fresh[3:3 + b.T], got[3:3 + b.T])


def test_starts_that_descend_leave_their_requests_out():
    b = Batch([(4, 64)], [5, 6, 7, 8], [2, 1, 1, 2], 2, 4, seed=9)
    want, size = b.want()
    starts = b.starts.copy()
    starts[2] = 1                                     # request 1 has rows 2 .. 1, request 2 rows 1 .. 4
    got = b.call(starts=dev(starts), max_rows=2)
    near_attention(got[[0, 4, 5]], want[[0, 4, 5]], size[[0, 4, 5]])
    assert not got[2:4].any()


def test_odd_values_in_what_a_row_does_not_see():
    """Behind the last token, in rows behind a row's own, and in other pages: NaN and infinities of those have no part; a row that sees an infinity has it."""
    b = Batch([(3, 64)], [5, 9, 20], [3, 2, 1], 2, 4, seed=10)
    want, size = b.want()
    for s in range(3):
        end = b.lens[s]
        b.kv[int(b.tables[s, (end - 1) // PAGE]), :, :, (end - 1) % PAGE + 1:] = float("nan")
    near_attention(b.call(), want, size)
    last = b.lens[0] - 1                              # the last of three rows: seen by itself alone
    b.kv[int(b.tables[0, last // PAGE]), 1, :, last % PAGE, 5] = float("inf")
    b.kv[int(b.tables[0, last // PAGE]), 1, :, last % PAGE, 9] = float("nan")
    got = b.call().view(b.T, b.heads, D)
    near_attention(got[[0, 1, 3, 4, 5]], want[[0, 1, 3, 4, 5]], size[[0, 1, 3, 4, 5]])
    assert (got[2, :, 5] == math.inf).all() and got[2, :, 9].isnan().all()
    rest = [c for c in range(D) if c not in (5, 9)]
    near_attention(got[2][:, rest], want[2][:, rest], size[2][:, rest])


def test_pages_that_the_cache_does_not_have_read_as_zeros():
    b = Batch([(3, 64)], [40, 9, 20], [1, 2, 1], 2, 4, seed=11)
    b.tables[0, 5], b.tables[2, 4] = -1, b.pages
    b.tables[:, 2] = b.pages + 5                      # of the shared ones
    b.check()


@pytest.mark.parametrize("scale", [1e-6, 1.0, 30.0])
def test_scales(scale):
    """At large scales one weight outweighs the others; scores are then fp32 sums of 128 products of up to 2^4 with an error of 2^-17, times the scale."""
    b = Batch([(3, 64)], [40, 9, 20], [1, 2, 1], 2, 4, seed=12)
    b.q = (b.q * (1 if scale < 1 else 2.0 ** -5)).bfloat16()
    b.check(scale=scale)


def test_the_same_bits_every_time_and_on_another_stream():
    b = Batch([(8, 700), (8, 300)], [1 + i * 9 for i in range(16)], [1] * 16, 8, 4, seed=13)
    first = b.call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [b.call() for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, a) for a in again)


# ------------------------------------------------------------------ selection
def select(x, scores, k, ends=None, dtype=torch.float32, view=None):
    """x [S, beams, V], numpy; checks the kernel's answer against the definition on the values as the type holds them."""
    from kubeai_b200 import ops
    S, B, V = x.shape
    t = torch.tensor(x.reshape(S * B, V), dtype=torch.float64).to(dtype).cuda()
    if view:
        t = view(t)
    sc = torch.tensor(scores, dtype=torch.float32).cuda()
    got = ops.beam_select(t, sc, k, ends=None if ends is None else dev(ends))
    found, goes, gap = plain.selected(t.double().cpu().numpy().reshape(S, B, V), sc.double().cpu().numpy(), k, set(ends if ends is not None else ()))
    # what decides is exact to the sum's error: small terms of 2^-22 in fp32, and the inputs are chosen so that nothing lies closer
    assert gap > 1e-6, gap
    for want, (c, p, v) in ((found, (got.found_scores, got.found_parents, got.found_tokens)), (goes, (got.scores, got.parents, got.tokens))):
        n = len(want[0])
        assert c.shape == p.shape == v.shape == (S, n)
        assert p.tolist() == [[e[1] for e in row] for row in want]
        assert v.tolist() == [[e[2] for e in row] for row in want]
        w = np.array([[e[0] for e in row] for row in want])
        g = c.double().cpu().numpy()
        fine = np.isfinite(w)
        assert (g[~fine] == w[~fine]).all()
        assert (np.abs(g - w)[fine] <= 2.0 ** -24 * np.abs(w[fine]) + 2.0 ** -20).all()
    return got


def spread(S, B, rng):
    return -np.cumsum(rng.uniform(0.1, 2, (S, B)), 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,B,V,k", [(1, 1, 1, 1), (1, 1, 1, 4), (2, 3, 2, 9), (3, 4, 7, 8), (1, 4, 1000, 8), (5, 2, 999, 64), (2, 32, 333, 64), (1, 1, 5000, 64), (3, 5, 30011, 15), (1, 2, 128256, 4), (1, 3, 393216, 6)])
def test_candidates(dtype, S, B, V, k):
    rng = np.random.default_rng(V + k)
    select(rng.normal(0, 3, (S, B, V)), spread(S, B, rng), k, ends=[2, V // 2], dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,value", [(100, 0.0), (5000, -3.0), (128256, 1.5), (70001, -1e30)])
def test_rows_of_equal_logits_go_by_the_token(dtype, V, value):
    select(np.full((2, 2, V), value), np.array([[-1.0, -1.0], [-3.0, -2.0]]), 20, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_ties_than_the_list_holds(dtype):
    """Three larger values, then a thousand equal ones among smaller ones, spread over the row; -0 and 0 are one value."""
    rng = np.random.default_rng(1)
    x = rng.normal(-9, 1, (1, 2, 60000)).clip(-20, -1)
    for b in range(2):
        at = rng.permutation(60000)[:3003]
        x[0, b, at[:3000]] = np.where(rng.random(3000) < 0.5, -0.0, 0.0)
        x[0, b, at[3000:]] = [3.0, 2.0, 1.0]
    select(x, np.array([[-1.0, -1.3]]), 24, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_odd_logits_and_scores(dtype):
    rng = np.random.default_rng(2)
    x = rng.normal(0, 2, (6, 3, 700))
    x[0, :, ::2] = np.nan
    x[1, 0] = -np.inf                    # a beam that a grammar leaves nothing
    x[1, 1, 1:] = -np.inf
    x[2] = -np.inf                       # a request without candidates
    x[3, 0, [5, 9]] = np.inf             # infinities share the probability
    x[4, 1] = np.nan
    x[5, 2] = np.finfo(np.float32).min if dtype == torch.float32 else -3.3e38      # the type's lowest value is a value
    scores = spread(6, 3, rng)
    scores[4] = [-np.inf, -1.0, np.nan]  # nobody
    scores[5] = [-np.inf, -np.inf, -2.0]
    got = select(x, scores, 7, ends=[5], dtype=dtype)
    assert (got.parents[2] == -1).all() and (got.scores[4] == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 5), (7, 9)])
def test_rows_off_sixteen_bytes(dtype, offset, pad):
    def view(t):
        big = torch.full((t.shape[0], offset + t.shape[1] + pad), float("inf"), dtype=t.dtype, device=t.device)
        big[:, offset:offset + t.shape[1]] = t
        return big[:, offset:offset + t.shape[1]]
    rng = np.random.default_rng(3)
    for V in (1, 5, 1003, 40001):
        select(rng.normal(0, 3, (2, 3, V)), spread(2, 3, rng), 6, dtype=dtype, view=view)


def test_ends_and_the_first_step():
    rng = np.random.default_rng(4)
    x = rng.normal(0, 1, (2, 4, 500))
    x[:, :, [7, 11]] += 9                # the best ones all end
    select(x, spread(2, 4, rng), 8, ends=[7, 11])
    got = select(x, spread(2, 4, rng), 8, ends=list(range(500)))
    assert (got.parents == -1).all() and (got.found_parents >= 0).all()
    # behind the prompt the beams are alike, and only one counts
    x[:] = x[:, :1]
    s = np.full((2, 4), -np.inf)
    s[:, 0] = 0.0
    got = select(x, s, 8)
    assert (got.parents == 0).all()
    # or all count, and equal candidates go to the lower beam
    got = select(x, np.zeros((2, 4)), 8)
    assert got.found_parents[0].tolist() == [0, 1, 2, 3, 0, 1, 2, 3]


def test_close_candidates_keep_their_order():
    """Beams whose candidates lie 2^-20 apart: an fp32 sum of scores around -60 (steps of 2^-18) would tie them."""
    from kubeai_b200 import ops
    rng = np.random.default_rng(5)
    x = np.repeat(rng.normal(0, 3, (1, 1, 4000)), 4, 1)
    scores = np.float32(-60) + np.array([[0.0, 2.0, 1.0, 3.0]], dtype=np.float32) * np.float32(2.0 ** -18)
    x32 = x.astype(np.float32)
    x32[0, 1, :] -= np.float32(0)        # the same rows: the scores' steps decide
    got = ops.beam_select(torch.tensor(x32[0]).cuda(), torch.tensor(scores).cuda(), 8)
    assert got.found_parents.tolist()[0] == [3, 1, 2, 0, 3, 1, 2, 0]


# ------------------------------------------------------------------ reordering
def reorder(parents, ctx, kvh=2, layers=3, seed=0, width=None, text=True, room=None, apart=False, lens=None, tables=None):
    from kubeai_b200 import ops
    rng = np.random.default_rng(seed)
    parents = np.asarray(parents)
    S, B = parents.shape
    width = width or max(plain.pages(max(c, 0)) for c in ctx) + 1
    if tables is None:
        tables, at = np.zeros((S * B, width), dtype=np.int64), 0
        for s in range(S):
            for c in range(width):
                kinds = B if (c + 1) * PAGE > ctx[s] else min(B, 1 + (c * 5) % 4)
                tables[s * B:(s + 1) * B, c] = at + rng.permutation(np.arange(B) * kinds // B)
                at += kinds
        tables = rng.permutation(at)[tables]
    else:
        at = 40
    kv = torch.randn(layers, at, 2, kvh, PAGE, D, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()
    room = room or max(max(ctx), 1) + 3
    texts = rng.integers(0, 1000, (S * B, room)) if text else None
    lens = (rng.integers(0, room + 1, S * B) if lens is None else np.asarray(lens)) if text else None
    tokens, full = rng.integers(0, 1000, (S, B)), np.repeat(ctx, B)
    want = plain.reordered(parents.tolist(), tokens, full.tolist(), tables, kv.view(torch.int16).cpu().numpy(), texts=texts, text_lens=lens)
    t = wide(dev(tables)) if apart else dev(tables)
    out = wide(torch.full_like(dev(tables), -9)) if apart else None
    x = None if texts is None else wide(dev(texts)) if apart else dev(texts)
    was = t.clone()
    got = ops.beam_reorder(dev(parents), dev(tokens), dev(full), t, kv, texts=x, text_lens=None if lens is None else dev(lens), out=out)
    assert torch.equal(t, was)
    assert got.block_tables.tolist() == want["tables"].tolist()
    assert got.shared.tolist() == want["shared"] and got.released.tolist() == want["released"].tolist()
    assert np.array_equal(kv.view(torch.int16).cpu().numpy(), want["kv"])
    if text:
        assert got.texts.tolist() == want["texts"].tolist() and got.text_lens.tolist() == list(want["text_lens"])
    else:
        assert got.texts is None and got.text_lens is None
    return got


@pytest.mark.parametrize("ctx", [1, 15, 16, 17, 40, 100])
@pytest.mark.parametrize("parents", [[[0]], [[0, 1, 2, 3]], [[3, 2, 1, 0]], [[0, 0, 0, 0]], [[2, 2, 0, 2]], [[1, 0, 1, -1]], [[-1, 3, 9, 3]]])
def test_reordered_beams(parents, ctx):
    reorder(parents, [ctx], seed=ctx)


@pytest.mark.parametrize("B", [1, 2, 5, 31, 32])
def test_many_requests_and_beams(B):
    rng = np.random.default_rng(B)
    S = 9
    reorder(rng.integers(-1 if B > 1 else 0, B, (S, B)), rng.integers(0, 90, S).tolist(), seed=B, apart=True)


def test_requests_that_are_left_as_they_are():
    """No parent that is one, and lengths that the table does not hold, or that differ."""
    reorder([[-1, -1], [5, -3], [1, 0]], [20, 33, 40], width=3, seed=1)
    reorder([[1, 1], [1, 1]], [49, 20], width=3, seed=2)
    from kubeai_b200 import ops
    t = dev([[1, 2], [3, 4]])
    got = ops.beam_reorder(dev([[1, 1]]), dev([[0, 0]]), dev([20, 21]), t, None)
    assert torch.equal(got.block_tables, t) and got.shared.tolist() == [0] and (got.released == -1).all()
    got = ops.beam_reorder(dev([[1, 1]]), dev([[0, 0]]), dev([-5, -5]), t, None)
    assert torch.equal(got.block_tables, t) and got.shared.tolist() == [0]


def test_without_texts_cache_or_columns():
    from kubeai_b200 import ops
    reorder([[0, 0, 1], [2, 2, 2]], [37, 50], text=False)
    got = ops.beam_reorder(dev([[0, 0]]), dev([[0, 0]]), dev([20, 20]), dev([[1, 2], [1, 4]]), None)
    assert got.block_tables.tolist() == [[1, 2], [1, 4]]
    got = ops.beam_reorder(dev([[0, 0]]), dev([[0, 0]]), dev([0, 0]), dev(np.zeros((2, 0))), None)
    assert got.block_tables.shape == (2, 0) and got.shared.tolist() == [0]


def test_pages_that_the_cache_does_not_have_are_not_copied():
    t = np.array([[3, 9], [3, 44], [3, 11], [3, -1]])      # the cache has 40
    reorder([[0, 0, 1, 0]], [20], tables=t, width=2)
    reorder([[1, 1, 1, 3]], [20], tables=t, width=2)


def test_texts_without_room_stay():
    reorder([[1, 0], [0, 0]], [20, 30], lens=[5, 8, -1, 3], room=8, seed=6)


def test_layers_may_lie_apart():
    from kubeai_b200 import ops
    kv = torch.randn(6, 8, 2, 2, PAGE, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    was = kv.clone()
    ops.beam_reorder(dev([[1, 1]]), dev([[0, 0]]), dev([21, 21]), dev([[1, 2], [1, 4]]), kv[::2])
    assert torch.equal(kv[::2, 2, :, :, :5], was[::2, 4, :, :, :5]) and torch.equal(kv[::2, 2, :, :, 5:], was[::2, 2, :, :, 5:])
    kv[::2, 2] = was[::2, 2]
    assert torch.equal(kv, was)


# ------------------------------------------------------------------ calls of no size, and hints
def test_calls_of_no_size():
    from kubeai_b200 import ops
    kv = torch.zeros(2, 2, 1, PAGE, D, device="cuda").bfloat16()
    q = torch.ones(3, D, device="cuda").bfloat16()
    none, table = dev([]), torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    y = ops.paged_attn_shared(q, kv, table, dev([0]), none, dev([0]), none, 1, 1, 1)
    assert y.shape == (3, D) and not y.any()
    kept = torch.ones(3, D, device="cuda").bfloat16()
    ops.paged_attn_shared(q, kv, table, dev([0]), none, dev([0]), none, 1, 1, 1, out=kept)
    assert bool((kept == 1).all())
    assert ops.paged_attn_shared(q[:0], kv, table, dev([0]), none, dev([0]), none, 1, 1, 1).shape == (0, D)
    turn = ops.rotary()
    assert ops.norm_rope_kvwrite(torch.zeros(0, 3 * D, device="cuda").bfloat16(), none, none, kv, 1, 1, turn.freqs).shape == (0, D)
    best = ops.beam_select(torch.zeros(0, 9, device="cuda"), torch.zeros(0, 4, device="cuda"))
    assert best.parents.shape == (0, 4) and best.found_scores.shape == (0, 8)
    moved = ops.beam_reorder(torch.zeros(0, 4, dtype=torch.int32, device="cuda"), none, none, table, None)
    assert moved.block_tables.shape == (0, 4) and moved.shared.shape == (0,)
    torch.cuda.synchronize()


@pytest.mark.parametrize("max_ctx", [0, 1, 600, 1 << 30])
@pytest.mark.parametrize("max_rows", [3, 1000])
def test_hints_do_not_change_what_is_attended(max_ctx, max_rows):
    b = Batch([(40, 500), (3, 333)], [3 + 7 * s % 60 for s in range(43)], [1 + s % 3 for s in range(43)], 2, 4, seed=21)
    b.check(max_ctx=max_ctx, max_rows=max_rows)


def test_pages_behind_the_first_four_gigabytes():
    from kubeai_b200 import ops
    kvh, n = 8, 72000      # 2.36 * 10^9 values
    kv = torch.zeros(1, n, 2, kvh, PAGE, D, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(4)
    ends = [n - 1 - i for i in range(24)]
    kv[0, dev(ends, torch.long)] = torch.randn(24, 2, kvh, PAGE, D, generator=gen, device="cuda").bfloat16()
    # four beams behind three shared pages, each with its own fourth
    tables = [[ends[0], ends[1], ends[2], ends[3 + s]] for s in range(4)]
    q = torch.randn(4, kvh * 4 * D, generator=gen, device="cuda").bfloat16()
    small = kv[0, dev(ends, torch.long)]
    near = [[0, 1, 2, 3 + s] for s in range(4)]
    args = (dev([0, 1, 2, 3, 4]), dev([52, 53, 51, 55]), dev([0, 4]), dev([48]), 32, 8, 1)
    assert torch.equal(ops.paged_attn_shared(q, kv[0], dev(tables), *args), ops.paged_attn_shared(q, small, dev(near), *args))
    # rows into them
    qkv = torch.randn(2, (32 + 16) * D, generator=gen, device="cuda").bfloat16()
    ops.norm_rope_kvwrite(qkv, dev([3, 4]), dev([ends[10] * PAGE + 5, ends[11] * PAGE + 15]), kv[0], 32, 8, ops.rotary().freqs)
    assert torch.equal(kv[0, ends[10], 1, :, 5], qkv[0, 40 * D:].view(8, D)) and torch.equal(kv[0, ends[11], 1, :, 15], qkv[1, 40 * D:].view(8, D))
    # and from one to another
    moved = ops.beam_reorder(dev([[0, 0, 2, 3]]), dev([[1, 2, 3, 4]]), dev([53] * 4), dev(tables), kv)
    assert moved.block_tables.tolist() == tables
    assert torch.equal(kv[0, ends[4], :, :, :5], small[3, :, :, :5]) and torch.equal(kv[0, ends[4], :, :, 5:], small[4, :, :, 5:])


# ------------------------------------------------------------------ rotation of few heads, and far positions
@pytest.mark.parametrize("heads,kvh", [(0, 1), (1, 0), (2, 0), (0, 2), (1, 1)])
@pytest.mark.parametrize("dims,interleaved", [(128, False), (128, True), (72, False), (66, False), (96, True)])
@pytest.mark.parametrize("T", [3, 2050])
def test_rotation_of_one_or_two_heads(T, heads, kvh, dims, interleaved):
    """The first warps alone have heads, and all pairs' angles are wanted."""
    turned(T, heads, kvh, dims, interleaved, "one", 4000, seed=heads + dims)


@pytest.mark.parametrize("spare", [0, 2, 8, 100])
def test_a_row_alone_has_any_distance(spare):
    """A row alone of a wider buffer, and its queries in place as a view of their columns, as several rows may have them."""
    from kubeai_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(spare)
    big = torch.randn(2, 16 * D + 104, generator=gen, device="cuda").bfloat16()
    kv, f = torch.randn(5, 2, 2, PAGE, D, generator=gen, device="cuda").bfloat16(), ops.rotary().freqs
    want_kv = kv.clone()
    want = ops.norm_rope_kvwrite(big[:, :12 * D].contiguous(), dev([7, 9]), dev([3, 20]), want_kv, 8, 2, f)
    for rows in (1, 2):
        x, mine = big.clone(), kv.clone()
        view = x[:rows, :12 * D + spare]
        got = ops.norm_rope_kvwrite(view, dev([7, 9][:rows]), dev([3, 20][:rows]), mine, 8, 2, f, out=view[:, :8 * D])
        assert got.data_ptr() == x.data_ptr() and torch.equal(got, want[:rows]) and torch.equal(x[:, 8 * D:], big[:, 8 * D:]) and torch.equal(x[rows:], big[rows:])
        assert torch.equal(mine[0], want_kv[0]) and torch.equal(mine[1], (want_kv if rows == 2 else kv)[1])
        queries, out = x[:rows, :8 * D + spare], torch.zeros(2, 8 * D + 104, device="cuda").bfloat16()
        args = (want_kv, dev([[0], [1]][:rows]), dev([0, 1, 2][:rows + 1]), dev([3, 4][:rows]), dev([0]), dev([]), 8, 2, 1)
        y = ops.paged_attn_shared(queries, *args, out=out[:rows, :8 * D + spare])
        assert torch.equal(y[:, :8 * D], ops.paged_attn_shared(want[:rows].contiguous(), *args)) and not out[:, 8 * D:].any() and not out[rows:].any()


# ------------------------------------------------------------------ the logarithm of a row's sum
LOG_SUM, LOG_SUM_TIES = 2.0 ** -18, 2.0 ** -16
# Terms besides a part's largest ones are fp32.  A term's exponent t is rounded by |t| ln 2 2^-24 of the term, and terms of t < -19 are too small to matter: 2^-20; its exponential is off by 2^-22; log2 e in
# fp32 by 2^-22; a thread adds 32 terms one by one and those of three others: 2^-19 and 2^-23.  In all less than 2^-18.  Where more than 256 values of a part tie for the last place a thread adds 128 terms, whose
# differences from the largest are rounded too: 2^-17, 2^-19 and the others, less than 2^-16.


def shares(rows, dtype):
    """For rows of logits the score beside which the best candidate's own share is next to nothing, so that fp32 holds what is left of it: what the kernel says, and what it is."""
    from kubeai_b200 import ops
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    v = x.double().numpy()
    top = v.max(1)
    share = -np.log(np.exp(v - top[:, None]).sum(1))
    score = (-share).astype(np.float32)
    got = ops.beam_select(x.cuda(), torch.tensor(score).view(-1, 1).cuda(), 1)
    return got.found_scores[:, 0].double().cpu().numpy(), score.astype(np.float64) + share


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1100, 9999, 128256, 393216])
def test_the_log_of_a_flat_rows_sum(dtype, V):
    rng = np.random.default_rng(V)
    rows = [rng.normal(m, s, V) for m, s in ((0, 0.25), (0, 1), (0, 3), (40, 1), (-1000, 2), (3e5, 4))]
    rows += [np.where(np.arange(V) % 97 == 5, 0.0, -9.0 - rng.random(V)), np.linspace(-13, 0, V)]
    got, want = shares(np.stack(rows), dtype)
    assert (np.abs(got - want) <= (LOG_SUM if dtype == torch.float32 else LOG_SUM_TIES)).all(), np.abs(got - want)      # (bf16 values are few far from zero, and tie)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 300, 500, 9999, 128256])
def test_the_log_of_equal_values_sum(dtype, V):
    rows = np.full((4, V), -3.0)
    rows[1] = np.where(np.arange(V) % 2, 1.0, -0.5)
    rows[2, V // 2] = 8.0
    rows[3, : V // 2] = -15.0
    got, want = shares(rows, dtype)
    assert (np.abs(got - want) <= LOG_SUM_TIES).all(), np.abs(got - want)


@pytest.mark.parametrize("V", [5003, 128256])
def test_close_candidates_of_different_flat_rows_keep_their_order(V):
    """Their shares lie 2^-17 apart, twice what the logarithms are off by."""
    from kubeai_b200 import ops
    rng = np.random.default_rng(V)
    for _ in range(4):
        x = rng.normal(0, 1, (8, V)).astype(np.float32)
        v = x.astype(np.float64)
        share = -np.log(np.exp(v - v.max(1, keepdims=True)).sum(1))
        order = rng.permutation(8)
        score = (order * 2.125 * 2.0 ** -17 - share).astype(np.float32)
        c = score + share
        assert (np.diff(np.sort(c)) > 2.0 ** -17).all()
        got = ops.beam_select(torch.tensor(x).cuda(), torch.tensor(score).view(1, 8).cuda(), 8)
        want = np.argsort(-c)
        place = {int(p): i for i, p in reversed(list(enumerate(got.found_parents[0].tolist())))}
        assert sorted(place, key=place.get) == [int(p) for p in want][:len(place)]


# ------------------------------------------------------------------ angles with more digits than fp64 has
TURN = "0.15915494309189533576888376337251436203445964574045644874766734405889679763"      # of a radian: 1 / (2 pi)


@pytest.mark.parametrize("position", [1, 1000, 10 ** 6, 2 ** 24 + 1, 2 ** 30 - 1, 2 ** 31 - 1])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_angles_against_more_digits(position, base):
    """An angle of N turns: its frequency in turns has two roundings to fp64, N 2^-52; the position's product is exact but for 2^-65 of a turn a position; what is left of a turn goes through fp32, 2^-26,
    and a sine and cosine of 2 ulp, 2^-22, are multiplied and added with three roundings of 2^-24.  Values of a pair are chosen that nearly cancel, so that the one rounding to bf16 hides little."""
    from fractions import Fraction

    from kubeai_b200 import ops
    freqs = ops.rotary(128, base, device="cpu").freqs
    whole = [Fraction(float(f)) * position * Fraction(TURN) for f in freqs]
    angle = np.array([float((n - round(n)) * 2) * math.pi for n in whole])
    cos, sin = np.cos(angle), np.sin(angle)
    # of 128 first values each pair's own with the second one that cancels best
    a = 1 + np.arange(128) / 128
    b = torch.tensor(a[:, None] * cos / np.where(np.abs(sin) < 2.0 ** -30, 1, sin)).clamp(-2.0 ** 40, 2.0 ** 40).bfloat16().double().numpy()
    best = np.abs(a[:, None] * cos - b * sin).argmin(0)
    x = np.zeros((1, 128))
    x[0, :64], x[0, 64:] = a[best], b[best, np.arange(64)]
    q = ops.norm_rope_kvwrite(torch.tensor(x).bfloat16().cuda(), dev([position]), dev([-1]), torch.zeros(1, 2, 0, PAGE, D).bfloat16().cuda(), 1, 0, freqs.cuda())
    got = q.double().cpu().numpy()[0]
    first, second = x[0, :64], x[0, 64:]
    want, size = np.concatenate([first * cos - second * sin, second * cos + first * sin]), np.tile(np.abs(first) + np.abs(second), 2)
    off = 2 * math.pi * (np.array([float(n) for n in whole]) * 2.0 ** -52 + position * 2.0 ** -65 + 2.0 ** -26) + 2.0 ** -22 + 3 * 2.0 ** -24
    assert (np.abs(got - want) <= BF16 * np.abs(want) + np.tile(off, 2) * size).all(), (np.abs(got - want) - BF16 * np.abs(want)).max()
