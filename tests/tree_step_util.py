"""Plain forms of the operations on drafted trees, request by request in numpy: integers as they are defined, attention in 64 bits, logits in the 32-bit steps
that their definition names and in 64 bits."""
import numpy as np

PAGE, D = 16, 128


def pages(n):
    return -(-n // PAGE)


def random_tree(rng, n):
    """Parents of n rows, any row in front of each."""
    return [-1] + [int(rng.integers(0, i)) for i in range(1, n)] if n else []


def ancestors(parents):
    """Truth values [rows, rows]: row j leads to row i (a parent not in front of its child counts as none)."""
    n = len(parents)
    see = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            see[i] = see[p]
        see[i, i] = True
    return see


def pack(truth, words):
    """Truth values [rows, any] as int32 [rows, words]."""
    full = np.zeros((len(truth), 32 * words), dtype=np.uint8)
    full[:, :truth.shape[1]] = truth
    return np.packbits(full, axis=1, bitorder="little").view(np.int32).reshape(len(truth), words)


def maps(ctx, new, held, tables, free, cursor, rows, parents=None, words=0):
    """What step_maps gives, with the tables as they are afterwards."""
    tables, held, width = tables.copy(), list(held), tables.shape[1]
    out = dict(starts=[0], positions=[0] * rows, slots=[-1] * rows, seqs=[-1] * rows, masks=np.zeros((rows, 32 * words), dtype=bool), status=[])
    at, short = 0, False
    for s, (c, n) in enumerate(zip(ctx, new)):
        wanted, flag = max(n, 0), 0
        bad = c < 0 or n < 0 or held[s] < 0 or held[s] > width or c + n > width * PAGE or c > held[s] * PAGE or (words and n > 32 * words) or at + wanted > rows
        need = 0 if bad else max(0, pages(c + n) - held[s])
        if bad:
            flag = 2
        elif need and (short or cursor + need > len(free)):
            flag, short = 1, True
        else:
            tables[s, held[s]:held[s] + need] = free[cursor:cursor + need]
            held[s], cursor = held[s] + need, cursor + need
        for i in range(min(wanted, max(0, rows - at))):
            t = at + i
            out["seqs"][t] = s
            if flag:
                continue
            out["slots"][t] = int(tables[s, (c + i) // PAGE]) * PAGE + (c + i) % PAGE
            out["positions"][t] = c + i
            if words:
                out["masks"][t, :i + 1] = True
        if not flag and parents is not None:
            mine = list(parents[at:at + n])
            see = ancestors(mine)
            for i in range(n):
                out["positions"][at + i] = c + int(see[i].sum()) - 1
                if words:
                    out["masks"][at + i] = False
                    out["masks"][at + i, :n] = see[i]
            if any(p < -1 or p >= i for i, p in enumerate(mine)):
                flag |= 4
        at = min(at + wanted, rows)
        out["starts"].append(at)
        out["status"].append(flag)
    out["masks"] = pack(out["masks"], words) if words else None
    return out | dict(tables=tables, held=held, cursor=cursor)


def attention(q, kv, tables, starts, ctx, see, scale=D ** -0.5):
    """q [T, heads, 128] and kv [pages, 2, kv_heads, 16, 128] in float64; see[s]: truth values [rows, rows] of each request.  Returns the output and, of every value,
    the sum of weights times magnitudes that its rounding errors go by."""
    T, heads, _ = q.shape
    kvh = kv.shape[2]
    out, size = np.zeros((T, heads, D)), np.zeros((T, heads, D))
    for s, c in enumerate(ctx):
        a, n = starts[s], starts[s + 1] - starts[s]
        if not n:
            continue
        flat = kv[tables[s][:pages(c + n)]].transpose(1, 2, 0, 3, 4).reshape(2, kvh, -1, D)[:, :, :c + n]
        for h in range(heads):
            k, v = flat[:, h // (heads // kvh)]
            for i in range(n):
                keys = np.concatenate([np.arange(c), c + np.flatnonzero(see[s][i])]).astype(int)
                if not len(keys):
                    continue
                with np.errstate(all="ignore"):
                    x = k[keys] @ q[a + i, h] * scale
                    w = np.exp(x - x.max())
                    out[a + i, h] = w @ v[keys] / w.sum()
                    size[a + i, h] = w @ np.abs(v[keys]) / w.sum()
    return out, size


def constrained(x, rows_of, said, prompt, drafts, see, penalties, bias, allowed, exact=False):
    """x [T, V]; rows_of[s]: the rows of request s; said[s], prompt[s]: its tokens and how many of them are the prompt; drafts [T]; see[s] [rows, rows];
    penalties [S, 3]; bias[s]: [(token, value)], the last of a token counts; allowed [T, V].  In float32 steps, or with exact in float64."""
    f = np.float64 if exact else np.float32
    T, V = x.shape
    y, ids = x.astype(f), np.full(T, -1)
    for s, rows in enumerate(rows_of):
        rho, pi, phi = (f(p) for p in penalties[s]) if penalties is not None else (f(1), f(0), f(0))
        for i, r in enumerate(rows):
            everything, count = set(said[s]), {}
            mine = [drafts[rows[j]] for j in np.flatnonzero(see[s][i])] if drafts is not None else []
            for t in list(said[s][prompt[s]:]) + mine:
                count[t] = count.get(t, 0) + 1
            with np.errstate(all="ignore"):
                for t in everything | set(mine):
                    if 0 <= t < V:
                        v = y[r, t]
                        y[r, t] = v / rho if v > 0 else v * rho
                for t, c in count.items():
                    if 0 <= t < V:
                        y[r, t] = y[r, t] - phi * f(c)
                        y[r, t] = y[r, t] - pi
                for t, b in dict(bias[s]).items():
                    if 0 <= t < V:
                        y[r, t] = y[r, t] + f(b)
            y[r, ~allowed[r]] = -np.inf
            choice = np.where(np.isnan(y[r]), -np.inf, y[r])
            best = choice[allowed[r]].max() if allowed[r].any() else None
            ids[r] = int(np.flatnonzero(allowed[r] & (choice == best))[0]) if best is not None else -1
    return y, ids


def accepted(ids, drafts, parents, starts, ctx, tables, kv, max_path):
    """What tree_accept gives, with the cache [layers, pages, 2, heads, 16, 128] as it is afterwards."""
    kv, was = kv.copy(), kv
    paths, tokens, lens = [], [], []
    for s, c in enumerate(ctx):
        a, n = starts[s], starts[s + 1] - starts[s]
        path = [0] if n else []
        while path and len(path) < max_path:
            nxt = [i for i in range(path[-1] + 1, n) if parents[a + i] == path[-1] and ids[a + path[-1]] >= 0 and drafts[a + i] == ids[a + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        for k, i in enumerate(path):
            kv[:, tables[s][(c + k) // PAGE], :, :, (c + k) % PAGE] = was[:, tables[s][(c + i) // PAGE], :, :, (c + i) % PAGE]
        paths.append(path + [-1] * (max_path - len(path)))
        tokens.append([int(ids[a + i]) for i in path] + [-1] * (max_path - len(path)))
        lens.append(len(path))
    return dict(accepted=lens, path=paths, tokens=tokens, ctx_lens=[c + n for c, n in zip(ctx, lens)], kv=kv)
