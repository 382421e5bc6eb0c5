"""The paged KV cache and its attentions in numpy, in 64 bits and loop by loop, and a cache on the device to compare
with: pools whose every unwritten value is NaN."""
import numpy as np

from lokal_amd import kernels as K

NO = K.NO_PAGE


def pages_for(n, page):
    return -(-n // page)


class Cache:
    """Host pools [layer][page][kv head][row][dim] and a table with shuffled pages, and their device copies."""

    def __init__(self, rng, lengths, *, kv=2, hd=64, page=16, f32=False, layers=1, spare=2, width=None, scale=1.0):
        self.kv, self.hd, self.page, self.f32, self.layers = kv, hd, page, f32, layers
        self.n = len(lengths)
        self.width = width or max(1, max(pages_for(n, page) for n in lengths))
        held = [pages_for(n, page) for n in lengths]
        self.n_pages = sum(held) + spare
        ids = list(rng.permutation(self.n_pages))
        self.table = np.full((self.n, self.width), NO, np.uint32)
        for s, h in enumerate(held):
            for x in range(h):
                self.table[s, x] = ids.pop()
        self.len = np.array(lengths, np.uint32)
        self.refs = np.zeros(self.n_pages, np.uint32)
        for i in self.table[self.table != NO]:
            self.refs[i] += 1
        t = np.float32 if f32 else np.float16
        shape = (layers, self.n_pages, kv, page, hd)
        self.k, self.v = np.full(shape, np.nan, t), np.full(shape, np.nan, t)
        for s, n in enumerate(lengths):
            for x in range(held[s]):
                rows = min(page, n - x * page)
                at = (slice(None), self.table[s, x], slice(None), slice(0, rows))
                self.k[at] = (rng.standard_normal((layers, kv, rows, hd)) * scale).astype(t)
                self.v[at] = rng.standard_normal((layers, kv, rows, hd)).astype(t)

    def up(self):
        self.dk, self.dv = K.DeviceArray.from_numpy(self.k), K.DeviceArray.from_numpy(self.v)
        self.dt, self.dl, self.dr = (K.DeviceArray.from_numpy(x) for x in (self.table, self.len, self.refs))
        self.pages = K.KvPages(self.dk, self.dv, K.F32 if self.f32 else K.F16, self.layers, self.n_pages, self.kv,
                               self.page, self.hd)
        self.seqs = K.PageTable(self.dt, self.dl, self.dr, self.n, self.width)
        return self

    def rows(self, pool, layer, s, n):
        """[kv][n][hd] of sequence s in 64 bits; NaN in holes."""
        out = np.full((self.kv, n, self.hd), np.nan)
        for x in range(n):
            pg = x // self.page
            i = self.table[s, pg] if pg < self.width else NO
            if i < self.n_pages:
                out[:, x] = pool[layer, i, :, x % self.page]
        return out

    def live(self, s, n):
        return np.array([x // self.page < self.width and self.table[s, x // self.page] < self.n_pages
                         for x in range(n)], bool)


def softmax_rows(q, k, v, sees):
    """Rows of q [r][hd] over k, v [n][hd] where sees [r][n]; zeros where nothing is seen.  Unseen values do not count."""
    out = np.zeros((len(q), v.shape[1] if v.ndim == 2 else 0))
    for i in range(len(q)):
        w = np.nonzero(sees[i])[0]
        if len(w) == 0:
            continue
        s = k[w] @ q[i] / np.sqrt(q.shape[1])
        if s.max() == -np.inf:
            continue
        p = np.exp(s - s.max())
        out[i] = p @ v[w] / p.sum()
    return out


def tree_rows(c, layer, q, ctx, nd, mask, heads, out, slots=None):
    """q, out [n][T][heads * hd]; mask [n][T][words] or None."""
    n, T = q.shape[:2]
    G = heads // c.kv
    out = out.astype(np.float64)
    for i in range(n):
        s = i if slots is None else int(slots[i])
        if s >= c.n:
            continue
        rows = min(int(nd[i]), T)
        cap = c.width * c.page
        x = min(int(ctx[i]), cap)
        total = min(x + rows, cap)
        k, v = c.rows(c.k, layer, s, total), c.rows(c.v, layer, s, total)
        live = c.live(s, total)
        for t in range(rows):
            sees = live.copy()
            for j in range(total - x):
                sees[x + j] &= bool(mask[i, t, j // 32] >> (j % 32) & 1) if mask is not None else j <= t
            for h in range(heads):
                qq = q[i, t, h * c.hd:(h + 1) * c.hd].astype(np.float64)
                out[i, t, h * c.hd:(h + 1) * c.hd] = softmax_rows(qq[None], k[h // G], v[h // G], sees[None])[0]
    return out


def bounds_of(c, layer, s, start, end, bounds):
    """bounds [page][kv][2][hd], changed in place."""
    end = min(end, c.width * c.page)
    if start >= end:
        return
    for pg in range(start // c.page, (end - 1) // c.page + 1):
        i = c.table[s, pg]
        if i >= c.n_pages:
            continue
        rows = c.k[layer, i, :, :min(c.page, end - pg * c.page)]
        bounds[i, :, 0], bounds[i, :, 1] = rows.min(1), rows.max(1)  # numpy's keep a NaN


def choose(c, s, q, ctx, bounds, heads, take, first, last):
    """[kv][take] page numbers."""
    G = heads // c.kv
    ctx = min(ctx, c.width * c.page)
    held = pages_for(ctx, c.page)
    out = np.full((c.kv, take), NO, np.uint32)
    for h in range(c.kv):
        if held <= take:
            out[h, :held] = range(held)
            continue
        score = np.empty(held)
        for x in range(held):
            i = c.table[s, x]
            if i >= c.n_pages:
                score[x] = -np.inf
                continue
            b = bounds[i, h].astype(np.float64)
            qq = q[h * G * c.hd:(h + 1) * G * c.hd].reshape(G, c.hd).astype(np.float64)
            score[x] = (qq * np.where(qq > 0, b[1], b[0])).sum(1).max() if np.isfinite(b).all() else np.nan
        keep = [x for x in range(held) if x < first or x >= held - last]
        # bounds that are not finite first, then by score, then the lowest page
        rest = sorted((x for x in range(held) if x not in keep),
                      key=lambda x: (not np.isnan(score[x]), 0 if np.isnan(score[x]) else -score[x], x))
        out[h, :take] = sorted(keep + rest[:take - len(keep)])
    return out


def sparse_rows(c, layer, s, q, ctx, taken, heads):
    G, out = heads // c.kv, np.zeros(len(q))
    ctx = min(ctx, c.width * c.page)
    k, v = c.rows(c.k, layer, s, ctx), c.rows(c.v, layer, s, ctx)
    live = c.live(s, ctx)
    for h in range(heads):
        sees = live & np.isin(np.arange(ctx) // c.page, taken[h // G])
        out[h * c.hd:(h + 1) * c.hd] = softmax_rows(q[None, h * c.hd:(h + 1) * c.hd].astype(np.float64), k[h // G],
                                                    v[h // G], sees[None])[0]
    return out


def attn_tol(hd, n, q, k):
    """How far an output may be from 64 bits, relative to the largest |v| that is seen.

    A score is a sum of hd products in f32 (q in two f16 parts is off by 2^-22 at most, 4 steps of 2^-24): off by
    (hd + 8) 2^-24 sum |q_d k_d| / sqrt(hd); its exponential is off by that, its own rounding and the exponent's, |s|
    2^-24 each; and a weight counts twice (above and below the line).  The sums over n positions round at most once a
    position and once a chunk or wave: n + 128 steps.  Weights in two f16 parts: 4 steps."""
    q, k = np.abs(q[np.isfinite(q)]), np.abs(k[np.isfinite(k)].astype(np.float64))
    s = float(hd * q.mean() * k.mean() * 4 / np.sqrt(hd)) if q.size and k.size else 0.0  # 4: no row's sum is as far off
    return 2.0 ** -24 * (2 * (hd + 8 + 2) * s + n + 128 + 8)


def ancestors(rng, T):
    """A random tree: bit rows of each token's ancestors and itself."""
    sees = np.eye(T, dtype=bool)
    for j in range(1, T):
        sees[j] |= sees[rng.integers(0, j)]
    return sees


def words(sees):
    T = sees.shape[-1]
    pad = np.zeros(sees.shape[:-1] + (pages_for(T, 32) * 32,), bool)
    pad[..., :T] = sees
    return np.ascontiguousarray(np.packbits(pad, axis=-1, bitorder="little")).view(np.uint32)


class Book:
    """fork / grow / trim on Python lists."""

    def __init__(self, c):
        self.page, self.width, self.n_pages = c.page, c.width, c.n_pages
        self.held = [[int(i) for i in row if i != NO] for row in c.table]
        self.len = [int(x) for x in c.len]
        self.refs = [int(x) for x in c.refs]

    def fork(self, src, dst):
        ok = []
        for i, (s, d) in enumerate(zip(src, dst)):
            good = s < len(self.len) and d < len(self.len) and d not in dst[:i] and s not in dst and self.len[d] == 0
            ok.append(int(good))
        for i, (s, d) in enumerate(zip(src, dst)):
            if ok[i]:
                self.held[d], self.len[d] = list(self.held[s]), self.len[s]
                for p in self.held[s]:
                    self.refs[p] += 1
        return ok

    def trim(self, slots, keep):
        for i, (s, n) in enumerate(zip(slots, keep)):
            if s >= len(self.len) or s in slots[:i]:
                continue
            n = min(n, self.len[s])
            for p in self.held[s][pages_for(n, self.page):]:
                self.refs[p] -= 1
            del self.held[s][pages_for(n, self.page):]
            self.len[s] = n

    def grow(self, slots, add):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        before = list(self.refs)
        ok, copied, at, short = [], [], 0, False
        for i, (s, more) in enumerate(zip(slots, add)):
            copied.append((NO, NO))
            if s >= len(self.len) or s in slots[:i] or pages_for(self.len[s] + more, self.page) > self.width:
                ok.append(0)
                continue
            n = self.len[s]
            copy = more > 0 and n % self.page != 0 and before[self.held[s][-1]] > 1
            need = pages_for(n + more, self.page) - pages_for(n, self.page) + copy
            short |= at + need > len(free)
            if need and short:
                ok.append(0)
                continue
            ok.append(1)
            new = free[at:at + need]
            at += need
            if copy:
                copied[-1] = (self.held[s][-1], new[0])
                self.refs[self.held[s].pop()] -= 1
            for p in new:
                self.refs[p] = 1
            self.held[s] += new
            self.len[s] += more
        return ok, copied

    def table(self):
        t = np.full((len(self.len), self.width), NO, np.uint32)
        for s, h in enumerate(self.held):
            t[s, :len(h)] = h
        return t
