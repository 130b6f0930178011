"""CPU restatement, in numpy, of the 4-bit cache and its operators: what the tests hold the GPU's results against.

mxfp4: 32 channels share 2^e, e the least integer in [-23, 13] with max |x| <= 6 * 2^e; a value is the nearest of 0, 0.5, 1,
1.5, 2, 3, 4, 6 times it, ties to the even code. A token of a head with a NaN or an infinity in its key or value is held as a
key of NaN and a value of 0. Arithmetic is float64 throughout.
"""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E_MIN, E_MAX = -23, 13


def exponents(x):
    """[..., 32] -> the exponent of each block"""
    most = np.abs(x.astype(np.float64)).max(-1)
    e = np.full(most.shape, E_MIN)
    for i in range(E_MIN, E_MAX):      # one more while it does not hold the largest
        e = np.where(most > 6.0 * 2.0 ** i, i + 1, e)
    return e


def codes(y):
    """values / 2^e -> 4-bit codes"""
    a = np.abs(y)
    d = np.abs(a[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    first = near.argmax(-1)
    last = 7 - near[..., ::-1].argmax(-1)
    c = np.where(first == last, first, np.where(first % 2 == 0, first, last))   # two as near: the even one
    return np.where(np.signbit(y), c + 8, c)


def quantise(x):
    """rows [..., D] -> (codes [..., D], exponents [..., D / 32]), no NaN handling"""
    b = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    e = exponents(b)
    return codes(b / 2.0 ** e[..., None]).reshape(x.shape), e


def values(c, e):
    v = np.where(c >= 8, -GRID[c & 7], GRID[c & 7]).reshape(*e.shape, 32)
    return (v * 2.0 ** e[..., None].astype(np.float64)).reshape(c.shape)


def held(k, v):
    """what the cache gives back for keys and values [..., D]"""
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    out = []
    for x, put in ((k, np.nan), (v, 0.0)):
        y = values(*quantise(np.where(bad[..., None], 0.0, x)))
        out.append(np.where(bad[..., None], put, y))
    return out


def offsets(D):
    """byte offsets in a run of 32 tokens: key codes [32, D], key exponents [32, D / 32], value codes, value exponents"""
    t, c = np.arange(32)[:, None], np.arange(D)[None]
    g, u, i = t % 16 // 4, t // 16, t % 16
    if D == 64:
        kc = ((c // 16) * 16 + i) * 16 + u * 8 + c % 16 // 2
    else:
        kc = (u * (D // 128) + c // 128) * 1024 + (c % 128 // 32 * 16 + i) * 16 + c % 32 // 2
    vc = 17 * D + c // 64 * 1024 + (g * 16 + c % 32 // 2) * 16 + c // 32 % 2 * 8 + u * 4 + i % 4
    b = np.arange(D // 32)[None]
    if D == 64:
        ke = 16 * D + (b * 16 + i) * 2 + u
    else:
        ke = 16 * D + (((b % 4) * 16 + i) * 2 + u) * (D // 128) + b // 4
    ve = 33 * D + (g * (D // 32) + b) * 8 + u * 4 + i % 4
    return kc, ke, vc, ve


class Cache:
    """A pool of pages on the host, byte for byte as the device holds it."""

    def __init__(self, n_pages, page, heads, dim, seed=None):
        self.n_pages, self.page, self.heads, self.dim = n_pages, page, heads, dim
        shape = (n_pages, heads, page // 32, 34 * dim)
        self.pool = np.zeros(shape, np.uint8) if seed is None else np.random.default_rng(seed).integers(0, 256, shape, np.uint8)
        self.at = offsets(dim)

    def write(self, pg, t, h, k, v):
        run = self.pool[pg, h, t // 32]
        t %= 32
        bad = not (np.isfinite(k).all() and np.isfinite(v).all())
        for x, code_at, exp_at, e_bad in ((k, self.at[0], self.at[1], 255), (v, self.at[2], self.at[3], E_MIN + 127)):
            c, e = quantise(np.where(bad, 0.0, x))
            run[code_at[t, 0::2]] = c[0::2] | c[1::2] << 4
            run[exp_at[t]] = e_bad if bad else e + 127

    def read(self, pg, t, h):
        run = self.pool[pg, h, t // 32]
        t %= 32
        out = []
        for code_at, exp_at in (self.at[:2], self.at[2:]):
            b = run[code_at[t]].astype(int)
            c = np.where(np.arange(self.dim) % 2 == 0, b & 15, b >> 4)
            e = run[exp_at[t]].astype(int)
            with np.errstate(over="ignore", invalid="ignore"):
                out.append(np.where(np.repeat(e, 32) == 255, np.nan, values(c, e - 127)))
        return out

    def tokens(self, table_row, n, h):
        """keys, values [n, D] and which tokens have a page"""
        k, v, ok = np.zeros((n, self.dim)), np.zeros((n, self.dim)), np.zeros(n, bool)
        for t in range(n):
            pg = table_row[t // self.page]
            if 0 <= pg < self.n_pages:
                k[t], v[t] = self.read(pg, t % self.page, h)
                ok[t] = True
        return k, v, ok


def attention(cache, table, length, q, rows=None, scale=None, window=0, sinks=0):
    """q [B, M, heads, D] -> [B, M, heads, D]"""
    B, M, Hq, D = q.shape
    G = Hq // cache.heads
    scale = scale or 1.0 / np.sqrt(D)
    out = np.zeros(q.shape)
    for b in range(B):
        n = int(np.clip(length[b], 0, table.shape[1] * cache.page))
        m = M if rows is None else int(np.clip(rows[b], 0, M))
        kv = [cache.tokens(table[b], n, h) for h in range(cache.heads)]
        t = np.arange(n)
        for i in range(m):
            p = n - m + i
            sees = t <= p
            if window:
                sees &= (t > p - window) | (t < sinks)
            for hq in range(Hq):
                k, v, ok = kv[hq // G]
                use = sees & ok
                if not use.any():
                    continue
                s = k[use] @ q[b, i, hq].astype(np.float64) * scale
                w = np.exp(s - np.nanmax(s)) if not np.isnan(s).all() else s
                out[b, i, hq] = w @ v[use] / w.sum()
    return out


def update(table, length, page, n_pages, Bo, src=None, keep=None, grow=None, grow_n=0, window=0, sinks=0):
    """-> (table, length, holders of each page, status, [(from, to)]): one sequence, one column at a time"""
    B, cols = table.shape
    length = np.clip(length, 0, cols * page)
    clean = lambda b, j: table[b, j] if 0 <= table[b, j] < n_pages else -1  # noqa: E731
    new, kept, grown = np.full((Bo, cols), -1), np.zeros(Bo, int), np.zeros(Bo, int)
    for b in range(Bo):
        s = b if src is None else int(src[b])
        if 0 <= s < B:
            kept[b] = length[s] if keep is None else min(max(int(keep[b]), 0), length[s])
            for j in range(-(-kept[b] // page)):
                if window and (j + 1) * page <= kept[b] - window + 1 and j * page >= sinks:
                    continue
                new[b, j] = clean(s, j)
        grown[b] = kept[b] + max(0, int(grow_n if grow is None else grow[b]))
    opens = [new[b, kept[b] // page] if grown[b] > kept[b] and kept[b] % page else None for b in range(Bo)]
    stuck = (grown > cols * page) | np.array([o == -1 for o in opens], bool)   # too long, or to go on in a page that is none
    wants = []
    for b in range(Bo):
        o = opens[b]
        copy = False
        if o is not None and o >= 0:
            holders = [x for x in range(Bo) if (new[x] == o).any()]
            held = int((new == o).sum())
            writers = [x for x in range(Bo) if opens[x] is not None and opens[x] == o]
            copy = held > 1 and not (len(writers) == held and writers[0] == b)
            assert holders
        if grown[b] > kept[b] and not stuck[b]:
            for j in range(kept[b] // page, -(-grown[b] // page)):
                fresh = j * page >= kept[b]
                if fresh or copy:
                    wants.append((b, j, o if copy and not fresh else None))
    free = [pg for pg in range(n_pages) if not (new == pg).any()]
    missing = max(0, len(wants) - len(free))
    if missing or stuck.any():
        old, oldlen = np.full((Bo, cols), -1), np.zeros(Bo, int)
        for b in range(min(B, Bo)):
            oldlen[b] = length[b]
            for j in range(-(-int(length[b]) // page)):
                old[b, j] = clean(b, j)
        return old, oldlen, None, [missing, len(free), 0, int(stuck.sum())], []
    moves = []
    for (b, j, o), pg in zip(wants, free):
        new[b, j] = pg
        if o is not None:
            moves.append((o, pg))
    holders = np.array([(new == pg).sum() for pg in range(n_pages)])
    return new, grown, holders, [0, len(free) - len(wants), len(moves), 0], moves


def compact(table, length, page, n_pages):
    """-> (table, status, [(from, to)])"""
    B, cols = table.shape
    out = np.full((B, cols), -1)
    for b in range(B):
        for j in range(-(-int(np.clip(length[b], 0, cols * page)) // page)):
            if 0 <= table[b, j] < n_pages:
                out[b, j] = table[b, j]
    live = sorted(set(out[out >= 0].tolist()))
    n = len(live)
    moves = list(zip([x for x in live if x >= n], [x for x in range(n) if x not in set(live)]))
    for a, b in moves:
        out[out == a] = b
    return out, [n, len(moves)], moves


def beam(logits, score, W, k, done=None, eos=-1):
    """-> (token, parent, score, done) [n][k] and, per search, the least gap between neighbours of its first k + 1 candidates"""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    rows, V = x.shape
    done = np.zeros(rows, bool) if done is None else np.asarray(done) != 0
    out, gaps = [[], [], [], []], []
    for g in range(rows // W):
        cand = []
        for w in range(W):
            r = g * W + w
            if done[r]:
                cand += [(score[r] if i == 0 and score[r] == score[r] else -np.inf, w, i, eos) for i in range(k)]
                continue
            with np.errstate(invalid="ignore"):
                m = x[r].max()
                lse = m + np.log(np.exp(x[r] - m).sum())
                order = np.argsort(-x[r], kind="stable")[:k]
                for i, t in enumerate(order):
                    s = float(score[r]) + (x[r, t] - lse)
                    cand.append((-np.inf if s != s else s, w, i, int(t)))
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        best = cand[:k]
        gaps.append(min([a[0] - b[0] for a, b in zip(cand[:k], cand[1:k + 1]) if a[0] > b[0]] + [np.inf]))
        for o, v in zip(out, ([c[3] for c in best], [g * W + c[1] for c in best], [c[0] for c in best],
                              [bool(done[g * W + c[1]]) or (eos >= 0 and c[3] == eos) for c in best])):
            o.append(v)
    return [np.array(o) for o in out], min(gaps + [np.inf])
