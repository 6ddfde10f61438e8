"""Plain forms of the operations of a step whose requests share their beginnings, request by request in numpy: attention, norms and log-probabilities in 64 bits, tables and texts as they
are defined."""
import math

import numpy as np

PAGE, D = 16, 128


def pages(n):
    return -(-n // PAGE)


def rotated(x, w, eps, positions, freqs, gain, interleaved):
    """x [T, heads, 128] in 64 bits, w [128], [heads, 128] or None.  Returns the values and the magnitudes of the two products that each one is the sum of."""
    y = x * w / np.sqrt((x * x).mean(-1, keepdims=True) + eps) if w is not None else x.copy()
    n = len(freqs)
    a, b = (np.arange(n) * 2, np.arange(n) * 2 + 1) if interleaved else (np.arange(n), np.arange(n) + n)
    angle = np.asarray(positions, dtype=np.float64)[:, None, None] * freqs
    c, s = gain * np.cos(angle), gain * np.sin(angle)
    out, size = y.copy(), np.abs(y)
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    size[..., a] = size[..., b] = (np.abs(y[..., a]) + np.abs(y[..., b])) * abs(gain)
    return out, size


def attention(q, kv, tables, starts, ctx, scale=D ** -0.5):
    """q [T, heads, 128] and kv [pages, 2, kv_heads, 16, 128] in 64 bits: every request over its own table.  Returns the output and, of every value, the sum of weights times magnitudes that its
    rounding errors go by."""
    T, heads, _ = q.shape
    kvh = kv.shape[2]
    out, size = np.zeros((T, heads, D)), np.zeros((T, heads, D))
    for s, c in enumerate(ctx):
        a, n = starts[s], starts[s + 1] - starts[s]
        if n <= 0:
            continue
        names = np.asarray(tables[s][:pages(c + n)])
        inside = (names >= 0) & (names < len(kv))
        flat = np.where(inside[:, None, None, None, None], kv[np.where(inside, names, 0)], 0).transpose(1, 2, 0, 3, 4).reshape(2, kvh, -1, D)[:, :, :c + n]
        for h in range(heads):
            k, v = flat[:, h // (heads // kvh)]
            for i in range(n):
                with np.errstate(all="ignore"):
                    x = k[:c + i + 1] @ q[a + i, h] * scale
                    w = np.exp(x - x.max())
                    out[a + i, h] = w @ v[:c + i + 1] / w.sum()
                    size[a + i, h] = w @ np.abs(v[:c + i + 1]) / w.sum()
    return out, size


def selected(x, scores, k, ends=()):
    """x [S, beams, V] and scores [S, beams] in 64 bits.  Returns the candidates [S][k] and the beams that go on [S][beams] as (score, parent, token), and the smallest distance of two
    candidates of different beams that decided something."""
    S, B, V = x.shape
    found, goes, gap = [], [], math.inf
    for s in range(S):
        best = []
        for b in range(B):
            row = np.where(np.isnan(x[s, b]), -np.inf, x[s, b])
            top = row.max()
            if top == -np.inf or not scores[s, b] > -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                d = np.where(row == top, 0.0, row - top)
            log_sum = math.log(np.exp(d).sum())
            order = np.lexsort((np.arange(V), -row))[:k]
            best += [(scores[s, b] - log_sum + d[v], b, i, int(v)) for i, v in enumerate(order) if d[v] > -np.inf]
        best.sort(key=lambda e: (-e[0], e[1], e[2]))
        near = [a[0] - b[0] for a, b in zip(best[:k], best[1:k + 1]) if a[1] != b[1] and a[0] != b[0]]
        gap = min([gap] + near)
        best = [(c, b, v) for c, b, _, v in best[:k]]
        on = [f for f in best if f[2] not in ends][:B]
        found.append(best + [(-math.inf, -1, -1)] * (k - len(best)))
        goes.append(on + [(-math.inf, -1, -1)] * (B - len(on)))
    return found, goes, gap


def reordered(parents, tokens, ctx, tables, kv, num_pages=None, texts=None, text_lens=None):
    """What beam_reorder gives, with the cache [layers, pages, 2, heads, 16, 128] as it is afterwards.  parents [S][B]."""
    S, B = len(parents), len(parents[0])
    old, new = np.asarray(tables), np.array(tables)
    width = old.shape[1]
    released, shared = np.full_like(old, -1), []
    kv = None if kv is None else kv.copy()
    num_pages = kv.shape[1] if kv is not None else num_pages
    texts_out = None if texts is None else np.array(texts)
    lens_out = None if texts is None else list(text_lens)
    for s in range(S):
        rows = [s * B + b for b in range(B)]
        c = ctx[rows[0]]
        real = [p for p in parents[s] if 0 <= p < B]
        if not real or any(ctx[r] != c for r in rows) or c < 0 or pages(c) > width:
            shared.append(0)
            continue
        full, part = divmod(c, PAGE)
        follows = [p if 0 <= p < B else real[0] for p in parents[s]]
        spare = [b for b in range(B) if b not in follows]
        moves = []
        for i, p in enumerate(follows):
            new[rows[i], :full] = old[rows[p], :full]
            if part:
                heir = p if p not in follows[:i] else spare.pop(0)
                new[rows[i], full] = old[rows[heir], full]
                if heir != p:
                    moves.append((old[rows[p], full], old[rows[heir], full]))
            if texts is not None:
                texts_out[rows[i]], lens_out[rows[i]] = texts[rows[p]], text_lens[rows[p]]
                if 0 <= parents[s][i] < B and 0 <= lens_out[rows[i]] < texts_out.shape[1]:
                    texts_out[rows[i], lens_out[rows[i]]] = tokens[s][i]
                    lens_out[rows[i]] += 1
        if kv is not None:
            was = kv.copy() if moves else None
            for a, b in moves:
                if 0 <= a < num_pages and 0 <= b < num_pages:
                    kv[:, b, :, :, :part] = was[:, a, :, :, :part]
        for col in range(full):
            stays, seen = {int(p) for p in new[rows, col]}, set()
            for r in rows:
                page = int(old[r, col])
                if page not in stays and page not in seen:
                    released[r, col] = page
                seen.add(page)
        alike = [len({int(p) for p in new[rows, col]}) == 1 for col in range(full)] + [False]
        shared.append(alike.index(False) * PAGE)
    return dict(tables=new, shared=shared, released=released, kv=kv, texts=texts_out, text_lens=lens_out)
