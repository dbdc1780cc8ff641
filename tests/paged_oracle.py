"""Drafted tokens over a paged cache, plainly and in 64 bits: trees, keys and values into pages, their attention, the path that stays."""
import numpy as np

import long_context_oracle as lc


def entries(q_start, T, max_new):
    """(first row, tokens) of each entry: what does not fit the rows is no token"""
    out = []
    for i in range(len(q_start) - 1):
        a, b = int(q_start[i]), int(q_start[i + 1])
        out.append((a, 0 if a < 0 or a > T or b <= a else min(min(b, T) - a, max_new)))
    return out


def ancestors(parents):
    """[t] -> the token's number and those of its ancestors, from itself on"""
    out = []
    for t in range(len(parents)):
        way, u, before = [], t, t + 1
        while 0 <= u < before:
            way.append(u)
            before, u = u, int(parents[u])
        out.append(way)
    return out


def tree_mask(parents, q_start, pos0, max_new, words):
    """(mask rows as python integers or None where the row is no entry's, positions)"""
    T = len(parents)
    mask, pos = [None] * T, [None] * T
    for i, (a, m) in enumerate(entries(q_start, T, max_new)):
        for t, way in enumerate(ancestors(parents[a:a + m])):
            mask[a + t] = sum(1 << u for u in way if u < 64 * words)
            pos[a + t] = int(pos0[i]) + len(way) - 1
    return mask, pos


def mask_int(row):
    """int64 words of a row -> one python integer"""
    return sum((int(w) & (1 << 64) - 1) << (64 * i) for i, w in enumerate(row))


def tree_accept(tokens, parents, choice, q_start, max_new):
    paths, then = [], []
    for a, m in entries(q_start, len(tokens), max_new):
        path = [0] if m else []
        while path:
            c = path[-1]
            more = [u for u in range(c + 1, m) if parents[a + u] == c and tokens[a + u] == choice[a + c]]
            if not more:
                break
            path.append(more[0])
        paths.append(path)
        then.append(int(choice[a + path[-1]]) if path else -1)
    return paths, then


class Cache:
    """Pools [n_layer, n_pages, H, page, hd] and a table as numpy arrays."""

    def __init__(self, k, v, table):
        self.k, self.v, self.table = k, v, table
        self.n_pages, self.H, self.page, self.hd = k.shape[1:]
        self.n_seq, self.n_ctx = table.shape[0], table.shape[1] * self.page

    def place(self, sq, slot):
        """(page, row) of a slot, None where it is not there"""
        if not (0 <= sq < self.n_seq and 0 <= slot < self.n_ctx):
            return None
        p = int(self.table[sq, slot // self.page])
        return (p, slot % self.page) if 0 <= p < self.n_pages else None


def known(cache, sq, pos):
    return 0 <= sq < cache.n_seq and 0 <= pos < cache.n_ctx


def append(cache, layer, k, v, q_start, pos0, seq, max_new, pos, freqs, mscale, halves):
    """New pools in 64 bits (before their rounding), a mask of the rows that were written, and each key's sum of magnitudes of its pair (for its tolerance)."""
    T = k.shape[0]
    kn, vn = cache.k.astype(np.float64), cache.v.astype(np.float64)
    wrote = np.zeros(cache.k.shape[:4], bool)
    ents = entries(q_start, T, max_new)
    for i, (a, m) in enumerate(ents):
        sq = i if seq is None else int(seq[i])
        if not known(cache, sq, int(pos0[i])) or any((j if seq is None else int(seq[j])) == sq and known(cache, sq, int(pos0[j])) and ents[j][1] for j in range(i + 1, len(ents))):
            continue
        for t in range(m):
            at = cache.place(sq, int(pos0[i]) + t)
            if at is None:
                continue
            p = int(pos0[i]) + t if pos is None else int(pos[a + t])
            row = k[a + t:a + t + 1].astype(np.float64)
            if freqs is not None:
                row = lc.rope(row, np.array([p]), freqs, mscale, cache.hd, halves)
            kn[layer, at[0], :, at[1]] = row.reshape(cache.H, cache.hd)
            vn[layer, at[0], :, at[1]] = v[a + t].astype(np.float64).reshape(cache.H, cache.hd)
            wrote[layer, at[0], :, at[1]] = True
    return kn, vn, wrote


def sees(cache, sq, pos, m, t, bits):
    """slots that token t of an entry of m tokens sees; bits: its mask as an integer, None: those up to its own"""
    if not known(cache, sq, pos) or pos + t >= cache.n_ctx:
        return []
    slots = list(range(pos)) + [pos + u for u in range(m) if (u <= t if bits is None else bits >> u & 1)]
    return [j for j in slots if cache.place(sq, j) is not None]


def attention(cache, layer, q, n_head, q_start, pos0, seq, max_new, mask, scale, u_row, u_p):
    """(out, tolerance), both [T, n_head, hd] in 64 bits; rows of no entry are NaN.  u_row: half a step of the rows' type; u_p: of a probability."""
    T, hd, H = q.shape[0], cache.hd, cache.H
    group, u32 = n_head // H, 2.0 ** -24
    q = q.astype(np.float64).reshape(T, n_head, hd)
    out, tol = np.full((T, n_head, hd), np.nan), np.full((T, n_head, hd), np.nan)
    for i, (a, m) in enumerate(entries(q_start, T, max_new)):
        sq, pos = i if seq is None else int(seq[i]), int(pos0[i])
        for t in range(m):
            slots = sees(cache, sq, pos, m, t, None if mask is None else mask_int(mask[a + t]))
            out[a + t] = tol[a + t] = 0.0
            if not slots:
                continue
            at = np.array([cache.place(sq, j) for j in slots])
            n = len(slots)
            for h in range(H):
                kk, vv = (x[layer, at[:, 0], h, at[:, 1]].astype(np.float64) for x in (cache.k, cache.v))
                qq = q[a + t, h * group:(h + 1) * group]
                s = scale * qq @ kk.T
                e = abs(scale) * (np.abs(qq) @ np.abs(kk).T).max(1, keepdims=True)
                p = np.exp(s - s.max(1, keepdims=True))
                total = p.sum(1, keepdims=True)
                p /= total
                o = p @ vv
                weight = p @ np.abs(vv)
                e_s = e * (hd + 10) * u32
                out[a + t, h * group:(h + 1) * group] = o
                # (2^-33: half a step of what a probability is held to at least, beside a largest one of 1 over 2^7 or more)
                tol[a + t, h * group:(h + 1) * group] = weight * (2 * e_s + (2 * n + 16) * u32 + u_p) + 2.0 ** -32 * np.abs(vv).sum(0) / total + u_row * np.abs(o) + (2.0 ** -25 if u_row > u32 else 0)
    return out, tol


def keep(cache, path, n_path, pos0, seq):
    k, v = cache.k.copy(), cache.v.copy()
    n = len(n_path)
    for i in range(n):
        sq, pos, rows = i if seq is None else int(seq[i]), int(pos0[i]), min(int(n_path[i]), path.shape[1])
        if not known(cache, sq, pos) or any((j if seq is None else int(seq[j])) == sq and n_path[j] > 0 for j in range(i + 1, n)):
            continue
        before = -1
        for r in range(rows):
            at = int(path[i, r])
            if at <= before:
                break
            before = at
            a, b = cache.place(sq, pos + at), cache.place(sq, pos + r)
            if a is not None and b is not None:
                k[:, b[0], :, b[1]], v[:, b[0], :, b[1]] = cache.k[:, a[0], :, a[1]], cache.v[:, a[0], :, a[1]]
    return k, v
