"""Inputs and 64-bit references for the operators of a decoder's memory (paged key-value
cache, linear attention with a decay), shared by the CPU and GPU tests."""
import numpy as np

EPS = 2.0 ** -24        # half a step of float32 relative to the value


class Cache(object):
    """Pools whose places are NaN except for the slots the rows fill; the table's unused
    entries are numbers no pool has."""

    def __init__(self, seed, kv_heads, dim, page, lengths, max_pages=None, spare=2):
        r = np.random.default_rng(seed)
        self.page, self.lengths = page, np.array(lengths, np.int32)
        b = len(lengths)
        need = [-(-int(n) // page) for n in lengths]
        self.max_pages = max_pages or max(max(need), 1)
        own = [max(n, self.max_pages if max_pages else n) for n in need]
        total = sum(own) + spare
        order = r.permutation(total)
        self.table = np.full((b, self.max_pages), -7, np.int32)
        shape = (total, kv_heads, page, dim)
        self.k, self.v = np.full(shape, np.nan, np.float32), np.full(shape, np.nan, np.float32)
        at = 0
        for i, n in enumerate(lengths):
            self.table[i, :own[i]] = order[at:at + own[i]]
            at += own[i]
            for j in range(int(n)):
                for pool in (self.k, self.v):
                    pool[self.table[i, j // page], :, j % page] = r.standard_normal((kv_heads, dim))
        self.capacity = self.max_pages * page

    def rows(self, pool, b, n):
        """[n, kv_heads, dim] of row b's slots."""
        j = np.arange(n)
        return pool[self.table[b, j // self.page], :, j % self.page]


def attention(q, cache, lengths, scale=None, mask=None, weights=None):
    """(out, new weights, bound of |out|'s float32 error, bound of the weights') in 64 bits.

    The bound: a score is a sum of dim products, dim / 4 of them in a row and two more sums,
    a product with the scale and a sum with the mask: |ds| <= (dim / 4 + 6) EPS sum |q k scale|
    + EPS |s|.  p = e^(s - m) / l then is off by a factor of at most 1 + x with x = 2 max |ds|
    (the maximum's error is a score's) + (2 |s - m| + 8) EPS (the difference, the product with
    log2 e, a 2-ulp exponential and the factors that join partial sums) + depth EPS for each of
    the two sums; depth: a sum over n terms in any order is off by at most n EPS of the sum of
    magnitudes."""
    bsz, heads, _, dim = q.shape
    kv = cache.k.shape[1]
    group = heads // kv
    out = np.zeros((bsz, 1, heads, dim))
    off = np.zeros((bsz, 1, heads, dim))
    new = None if weights is None else np.zeros(weights.shape)
    woff = None if weights is None else np.zeros(weights.shape)
    for b in range(bsz):
        n = int(lengths[b])
        shown = np.arange(n) if mask is None else np.flatnonzero(mask[b, :n] != -np.inf)
        k = cache.rows(cache.k, b, n)[shown].astype(np.float64)
        v = cache.rows(cache.v, b, n)[shown].astype(np.float64)
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            qh = q[b, h, 0].astype(np.float64) * (1.0 if scale is None else float(np.float32(scale)))
            s = kh @ qh
            ds = (dim / 4 + 6) * EPS * (np.abs(kh) @ np.abs(qh))
            if mask is not None:
                s = s + mask[b, shown].astype(np.float64)
            ds = ds + EPS * np.abs(s)
            if len(shown):
                e = np.exp(s - s.max())
                p = e / e.sum()
                x = 2 * ds.max() + (2 * np.minimum(s.max() - s, 100) + 8) * EPS + 2 * len(shown) * EPS
                out[b, 0, h] = p @ vh
                off[b, 0, h] = (p * x) @ np.abs(vh) + EPS * np.abs(out[b, 0, h]) + 1e-37
                if weights is not None:
                    new[b, h // group, shown] += p
                    woff[b, h // group, shown] += p * (x + group * EPS) + 1e-37
        if weights is not None:
            new[b, :, :n] += weights[b, :, :n]
            woff[b, :, :n] += EPS * np.abs(new[b, :, :n])
    return out, new, off, woff


def evict(cache, weights, lengths, budget, recent, positions=None, total=None):
    """(weights, positions, lengths, kept, k pool, v pool) after an eviction, slot by slot."""
    bsz, heads, cap = weights.shape
    k, v = cache.k.copy(), cache.v.copy()
    ow, op = np.zeros(weights.shape, np.float32), np.full(weights.shape, -1, np.int32)
    kept = np.full((bsz, heads, budget), -1, np.int32)
    ol = np.minimum(lengths, budget).astype(np.int32)
    for b in range(bsz):
        n, m = int(lengths[b]), int(ol[b])
        seen = n if total is None else int(total[b])
        for h in range(heads):
            pos = [seen - (n - j) for j in range(n)]
            if positions is not None:
                pos = [int(positions[b, h, j]) if positions[b, h, j] >= 0 else pos[j] for j in range(n)]

            def rank(j):
                w = weights[b, h, j]
                if pos[j] >= seen - recent:
                    return (0, 0.0, j)
                if np.isnan(w):
                    return (1, 0.0, j)
                return (2, -float(w), j)
            keep = sorted(range(n), key=rank)[:m]
            late = sorted(j for j in keep if j >= m)
            free = [j for j in range(m) if j not in set(keep)]
            src = list(range(m))
            for to, frm in zip(free, late):
                src[to] = frm
            for to in range(m):
                frm = src[to]
                ow[b, h, to], op[b, h, to], kept[b, h, to] = weights[b, h, frm], pos[frm], frm
                if frm != to:
                    for old, pool in ((cache.k, k), (cache.v, v)):
                        pool[cache.table[b, to // cache.page], h, to % cache.page] = \
                            old[cache.table[b, frm // cache.page], h, frm % cache.page]
    return ow, op, ol, kept, k, v


def linear(q, k, v, log_decay, state=None, scale=None, lengths=None):
    """(out, state, bounds of their float32 errors) of the recurrence in 64 bits.

    The bound: a term of out_t or S_t that is j steps old carries the decay's error (e^x of an
    argument rounded once, 2 ulp, and either j products or one exponential of j times the
    logarithm: at most (3 j + 4 + |j log_decay|) EPS) and is one of at most t + dim_k terms of
    sums whose roundings are each EPS of what is summed; products taken in pieces of 11 bits
    (three tensor-core products) leave out 2^-22 of each.  A sum of magnitudes, decayed the
    same way, therefore bounds the error with the factor (5 t + dim_k + 48) EPS."""
    bsz, heads, seq, dk = q.shape
    dv = v.shape[3]
    g = np.exp(log_decay.astype(np.float64))[None, :, None, None]
    s = np.zeros((bsz, heads, dk, dv)) if state is None else state.astype(np.float64)
    a = np.abs(s)
    out, off = np.zeros((bsz, seq, heads, dv)), np.zeros((bsz, seq, heads, dv))
    soff = 24 * EPS * a
    sc = 1.0 if scale is None else float(np.float32(scale))
    n = np.full(bsz, seq) if lengths is None else np.asarray(lengths)
    for t in range(seq):
        live = (t < n)[:, None, None, None]
        kt, vt, qt = (x[:, :, t].astype(np.float64) for x in (k, v, q))
        s = np.where(live, g * s + kt[..., :, None] * vt[..., None, :], s)
        a = np.where(live, g * a + np.abs(kt)[..., :, None] * np.abs(vt)[..., None, :], a)
        factor = (5 * (t + 1) + dk + 48) * EPS
        soff = np.where(live, factor * a, soff)
        out[:, t] = np.where(live[..., 0], np.einsum("bhk,bhkv->bhv", qt, s) * sc, 0)
        off[:, t] = np.where(live[..., 0], np.einsum("bhk,bhkv->bhv", np.abs(qt), a) * abs(sc) * factor, 0)
    return out, s, off + 1e-37, soff + 1e-37
