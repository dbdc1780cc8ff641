"""The operators of a long context written down plainly, in 64 bits (codes and scales by their steps in FP32, which define them)."""
import numpy as np

ONE127 = np.float32(1.0) / np.float32(127.0)
TINY = np.finfo(np.float32).tiny


def rope(x, pos, freqs, mscale, hd, halves):
    """x [T, heads * hd], freqs [n_rot / 2] in 64 bits"""
    T, half = x.shape[0], len(freqs)
    y = x.astype(np.float64).reshape(T, -1, hd).copy()
    a = np.asarray(pos, np.float64)[:, None] * np.asarray(freqs, np.float64)[None, :]
    c, s = np.cos(a)[:, None] * mscale, np.sin(a)[:, None] * mscale
    i0, i1 = (np.arange(half), np.arange(half) + half) if halves else (np.arange(half) * 2, np.arange(half) * 2 + 1)
    x0, x1 = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    return y.reshape(T, -1)


class Cache:
    def __init__(self, n_seq, H, n_ctx, hd, block):
        self.codes = {n: np.zeros((n_seq, H, n_ctx, hd), np.int8) for n in "kv"}
        self.scale = {n: np.zeros((n_seq, H, n_ctx // block), np.float32) for n in "kv"}
        self.n_seq, self.H, self.n_ctx, self.hd, self.block = n_seq, H, n_ctx, hd, block

    def entries(self, q_start, pos0, seq, T, max_new):
        """(entry, first row, tokens, first slot, sequence or -1)"""
        for i in range(len(pos0)):
            first, n = int(q_start[i]), min(int(q_start[i + 1]) - int(q_start[i]), max_new)
            n = max(0, min(n, T - first)) if 0 <= first <= T else 0
            sq, p = (i if seq is None else int(seq[i])), int(pos0[i])
            yield i, first, n, p, (sq if 0 <= sq < self.n_seq and 0 <= p < self.n_ctx else -1)

    def last(self, q_start, pos0, seq, T, max_new):
        """... of those that have tokens and a sequence, and of entries that name one sequence the last one"""
        e = [x for x in self.entries(q_start, pos0, seq, T, max_new) if x[2] > 0 and x[4] >= 0]
        return [x for j, x in enumerate(e) if x[4] not in [y[4] for y in e[j + 1:]]]

    def store(self, k, v, q_start, pos0, seq=None, max_new=1 << 30):
        B = self.block
        for name, x in (("k", k), ("v", v)):
            x = x.astype(np.float32).reshape(x.shape[0], self.H, self.hd)
            for _, first, n, p, sq in self.last(q_start, pos0, seq, x.shape[0], max_new):
                end = min(p + n, self.n_ctx)
                for b in range(p // B, (end - 1) // B + 1):
                    lo, hi = max(p, b * B), min(end, (b + 1) * B)
                    new = x[first + lo - p:first + hi - p]
                    for h in range(self.H):
                        y = new[:, h]
                        fin = np.abs(y[np.isfinite(y)])
                        old = self.scale[name][sq, h, b] if lo > b * B else np.float32(0)
                        s = max((fin.max() if fin.size else np.float32(0)) * ONE127, old)
                        s = np.float32(s) if s >= TINY else np.float32(0)
                        inv = np.float32(1) / s if s > 0 else np.float32(0)
                        with np.errstate(invalid="ignore", over="ignore"):
                            z = y * inv
                        z = np.rint(np.clip(np.where(np.isnan(z), 0, z), -127, 127))
                        if lo > b * B and s > old:
                            had = self.codes[name][sq, h, b * B:lo]
                            self.codes[name][sq, h, b * B:lo] = np.rint(had.astype(np.float32) * (old / s))
                        self.codes[name][sq, h, lo:hi] = z
                        self.scale[name][sq, h, b] = s

    def values(self, name, sq, h, n):
        return self.codes[name][sq, h, :n].astype(np.float64) * np.repeat(self.scale[name][sq, h].astype(np.float64), self.block)[:n, None]

    def attention(self, q, n_head, scale, q_start, pos0, seq=None, max_new=1 << 30, w_in=None, w_out=None, out=None):
        """(out; at each element sum p |v|; at each row and head scale * max_j sum_d |q_d k_jd|, and the slots it sees times the largest value that their
        blocks hold)"""
        T, group = q.shape[0], n_head // self.H
        q = q.astype(np.float64).reshape(T, n_head, self.hd)
        out = np.zeros_like(q) if out is None else out.astype(np.float64).reshape(q.shape).copy()
        size, terms, most = np.zeros_like(q), np.zeros((T, n_head)), np.zeros((T, n_head))
        live = {x[0] for x in self.last(q_start, pos0, seq, T, max_new)}
        for i, first, n, p, sq in self.entries(q_start, pos0, seq, T, max_new):
            out[first:first + n] = 0.0
            if sq < 0 or n == 0:
                continue
            end = min(p + n, self.n_ctx)
            for h in range(self.H):
                k, v = self.values("k", sq, h, end), self.values("v", sq, h, end)
                total = np.zeros(end)
                for t in range(end - p):
                    seen = p + t + 1
                    for g in range(group):
                        x = q[first + t, h * group + g]
                        s = scale * (k[:seen] @ x)
                        e = np.exp(s - s.max())
                        e /= e.sum()
                        out[first + t, h * group + g] = e @ v[:seen]
                        size[first + t, h * group + g] = e @ np.abs(v[:seen])
                        terms[first + t, h * group + g] = abs(scale) * (np.abs(k[:seen]) @ np.abs(x)).max()
                        most[first + t, h * group + g] = seen * 127.0 * self.scale["v"][sq, h, :(seen - 1) // self.block + 1].max()
                        total[:seen] += e
                if w_out is not None and i in live:
                    w_out[sq, h, :end] = total
                    if w_in is not None:
                        w_out[sq, h, :p] += w_in[sq, h, :p]
        return out.reshape(T, -1), size.reshape(T, -1), terms, most

    def evict(self, w, lens, keep, n_sink, n_recent, seq=None, w_out=None):
        B = self.block
        kept = np.full((len(lens), self.H, keep), -1, np.int32)
        which = list(range(len(lens))) if seq is None else [int(s) for s in seq]
        for i, n in enumerate(lens):
            sq, n = which[i], max(0, min(int(n), self.n_ctx))
            if sq in which[i + 1:] or not 0 <= sq < self.n_seq:
                continue
            for h in range(self.H):
                m = min(n, keep)
                kept[i, h, :m] = np.arange(m)
                if n > keep:
                    rank = np.where(np.isnan(w[sq, h, :n]), np.inf, w[sq, h, :n].astype(np.float64))
                    order = sorted(range(n), key=lambda j: (0 if j < n_sink or j >= n - n_recent else 1, 0 if np.isnan(w[sq, h, j]) else 1, -rank[j], j))
                    best = np.zeros(n, bool)
                    best[order[:keep]] = True
                    kept[i, h, np.flatnonzero(~best[:keep])] = keep + np.flatnonzero(best[keep:])
                if w_out is not None:
                    w_out[sq, h, :m] = w[sq, h, kept[i, h, :m]]
                for name in "kv":
                    codes, scale = self.codes[name][sq, h], self.scale[name][sq, h]
                    was, was_scale = codes.copy(), scale.copy()
                    for b in range(keep // B):
                        src = kept[i, h, b * B:(b + 1) * B]
                        if not (src >= keep).any():
                            continue
                        of = was_scale[src // B]                          # (a block that takes rows in is full)
                        scale[b] = of.max()
                        with np.errstate(invalid="ignore", divide="ignore"):
                            ratio = np.where(of == scale[b], np.float32(1), of / scale[b]).astype(np.float32)
                        codes[b * B:(b + 1) * B] = np.rint(was[src].astype(np.float32) * ratio[:, None])
        return kept
