"""Plain implementations of the operators of a batched step, in 64 bits (numpy) or, for the pages,
as one step after another: what the device's results are held to."""
import numpy as np


def norm_rows(x, add, w, eps):
    """(s, q, d) bit for bit: fp32 with the sum of squares in order, then the 32-block quantiser."""
    f = np.float32
    s = x if add is None else (x + add).astype(f)
    sq = (s * s).astype(f)
    ss = np.zeros(len(s), f)
    for i in range(s.shape[1]):
        ss = (ss + sq[:, i]).astype(f)
    scale = (f(1) / np.sqrt((ss / f(s.shape[1])).astype(f) + f(eps)).astype(f)).astype(f)
    v = ((s * scale[:, None]).astype(f) * w[None]).astype(f)
    b = v.reshape(len(s), -1, 32)
    d = (np.abs(b).max(2) / f(127)).astype(f)
    inv = np.where(d != 0, f(1) / np.where(d != 0, d, f(1)), f(0)).astype(f)
    q = np.rint((b * inv[..., None]).astype(f)).astype(np.int8).reshape(s.shape)
    return s, q, d


class Pages:
    """The tables of a paged cache, and its data as k[layer, page, position, head, :]."""

    def __init__(self, table, n_len, ref, k, v, page):
        self.table, self.len, self.ref = table.copy(), n_len.copy(), ref.copy()
        self.k, self.v, self.page, self.refused = k.copy(), v.copy(), page, 0

    def ok(self, slot):
        return 0 <= slot < len(self.len)

    def free_pages(self):
        return [p for p in range(len(self.ref)) if self.ref[p] == 0]

    def grow(self, slots, add):
        fresh, short, seen = self.free_pages(), False, set()
        for s in slots:
            bad = not self.ok(s) or s in seen
            seen.add(s)
            if not bad:
                have, need = -(-self.len[s] // self.page), -(-(self.len[s] + add) // self.page)
                bad = need > self.table.shape[1]
                if not bad and need > have:
                    short = short or need - have > len(fresh)
                    bad = short
            if bad:
                self.refused += 1
                continue
            for j in range(have, need):
                self.table[s, j] = p = fresh.pop(0)
                self.ref[p] = 1
            self.len[s] += add

    def fork(self, src, dst):
        fresh, seen, n0, t0 = self.free_pages(), set(), self.len.copy(), self.table.copy()
        for a, b in zip(src, dst):
            bad = not self.ok(a) or not self.ok(b) or b in seen or n0[b] != 0
            seen.add(b)
            if not bad:
                whole, rest = divmod(int(n0[a]), self.page)
                bad = rest > 0 and not fresh
            if bad:
                self.refused += 1
                continue
            for j in range(whole):
                self.table[b, j] = t0[a, j]
                self.ref[t0[a, j]] += 1
            if rest:
                self.table[b, whole] = p = fresh.pop(0)
                self.ref[p] = 1
                for x in (self.k, self.v):
                    x[:, p, :rest] = x[:, t0[a, whole], :rest]
            self.len[b] = n0[a]

    def free(self, slots):
        for s in slots:
            if not self.ok(s):
                self.refused += 1
                continue
            for j in range(-(-int(self.len[s]) // self.page)):
                self.ref[self.table[s, j]] -= 1
            self.len[s] = 0

    def compact(self):
        live = int((self.ref > 0).sum())
        holes = [p for p in range(live) if self.ref[p] == 0]
        moved = {}
        for p in range(live, len(self.ref)):
            if self.ref[p]:
                d = holes.pop(0)
                moved[p] = d
                self.ref[d], self.ref[p] = self.ref[p], 0
                self.k[:, d], self.v[:, d] = self.k[:, p], self.v[:, p]
        for s, n in enumerate(self.len):
            for j in range(-(-int(n) // self.page)):
                self.table[s, j] = moved.get(int(self.table[s, j]), self.table[s, j])
        return live


def rope(x, cs):
    """x [..., hd] turned by cs [..., hd] (cos, sin pairs), 64 bits."""
    p, c = x.astype(np.float64).reshape(*x.shape[:-1], -1, 2), cs.astype(np.float64).reshape(*cs.shape[:-1], -1, 2)
    return np.stack((p[..., 0] * c[..., 0] - p[..., 1] * c[..., 1],
                     p[..., 0] * c[..., 1] + p[..., 1] * c[..., 0]), -1).reshape(x.shape)


def attention(q, keys, values, n_len, n_tok, scale):
    """One sequence: q [n_tok, heads, hd], keys and values [at least n_len, kv, hd], 64 bits."""
    heads, kv = q.shape[1], keys.shape[1]
    out = np.zeros(q.shape)
    for t in range(n_tok):
        seen = n_len - n_tok + t + 1
        if seen <= 0:
            continue
        for h in range(heads):
            k, v = keys[:seen, h // (heads // kv)], values[:seen, h // (heads // kv)]
            x = k @ q[t, h] * scale
            w = np.exp(x - x.max())
            out[t, h] = w @ v / w.sum()
    return out


def adapters(q, d, which, base, a, b, rank, scale):
    """base + scale B (A x) row by row, 64 bits."""
    x = q.astype(np.float64) * np.repeat(d.astype(np.float64), 32, 1)
    y = base.astype(np.float64).copy()
    for r, s in enumerate(which):
        if 0 <= s < len(rank):
            n = max(0, min(int(rank[s]), a.shape[1]))
            y[r] += float(scale[s]) * (b[s][:, :n].astype(np.float64) @ (a[s][:n].astype(np.float64) @ x[r]))
    return y
