"""Plain restatements (numpy, float64; lists for the tables) of the paged key-value cache
operators: attention over pages, the append of new tokens, and the page bookkeeping."""
import numpy as np


def gather(pages, table, n, hk):
    """The first n tokens of key head hk of a sequence: pages [P, Hkv, page, hd] -> [n, hd]."""
    page = pages.shape[2]
    out = np.zeros((n, pages.shape[3]))
    for j in range(-(-n // page)):
        m = min(page, n - j * page)
        out[j * page:j * page + m] = pages[table[j], hk, :m]
    return out


def attention(q, k_pages, v_pages, table, seq_lens, cu, *, window=0, k_sink=None, gate=None, scale=None):
    """(o, lse, spread, ds): o and lse of every packed row; spread = sum_k p_k |v_k| (what a relative
    error of the weights moves o by), ds = the largest sum |q_i k_i| * scale of a row's visible keys
    (what a relative error of the products moves a logit by)."""
    T, H, hd = q.shape
    Hkv = k_pages.shape[1]
    scale = 1.0 / np.sqrt(hd) if scale is None else scale
    o, spread = np.zeros((T, H, hd)), np.zeros((T, H, hd))
    lse, ds = np.full((T, H), -np.inf), np.zeros((T, H))
    for s in range(len(seq_lens)):
        n, total = cu[s + 1] - cu[s], int(seq_lens[s])
        for h in range(H):
            hk = h // (H // Hkv)
            lo = max(0, total - n - window + 1) if window else 0    # earlier keys are not looked at
            K, V = (np.zeros((total, hd)) for _ in range(2))
            if total > lo:
                K[lo:] = gather_tail(k_pages, table[s], lo, total, hk)
                V[lo:] = gather_tail(v_pages, table[s], lo, total, hk)
            for i in range(n):
                p = total - n + i
                if p < 0 and k_sink is None:
                    continue
                first = max(0, p - window + 1) if window else 0
                Kv, Vv = K[first:max(p + 1, 0)], V[first:max(p + 1, 0)]
                qi = q[cu[s] + i, h]
                logit = Kv @ qi * scale
                size = np.abs(Kv) @ np.abs(qi) * abs(scale)
                z, zs = np.array([]), np.array([])
                if k_sink is not None:
                    z = np.array([qi @ k_sink[h] * scale])
                    zs = np.array([np.abs(qi) @ np.abs(k_sink[h]) * abs(scale)])
                everything = np.concatenate([logit, z])
                if everything.size == 0:
                    continue
                top = everything.max()
                w = np.exp(logit - top)
                den = np.exp(everything - top).sum()
                r = cu[s] + i
                lse[r, h] = top + np.log(den)
                ds[r, h] = np.concatenate([size, zs]).max()
                g = 1.0 if gate is None else 1.0 / (1.0 + np.exp(-gate[r, h]))
                o[r, h] = g * (w @ Vv) / den
                spread[r, h] = g * (w @ np.abs(Vv)) / den
    return o, lse, spread, ds


def gather_tail(pages, table, lo, total, hk):
    page = pages.shape[2]
    idx = np.arange(lo, total)
    return pages[np.asarray(table)[idx // page], hk, idx % page]


def append(qkvg, k_pages, v_pages, table, seq_lens, cu, *, n_heads, q_weight=None, k_weight=None, eps=1e-6, cos=None,
           sin=None):
    """(q, k pages, v pages, size): size bounds |a| + |b| of the rotated pairs of q and of k."""
    T = qkvg.shape[0]
    _, Hkv, page, hd = k_pages.shape
    H = n_heads
    k_pages, v_pages = k_pages.copy(), v_pages.copy()
    q, qs, ks = np.zeros((T, H, hd)), np.zeros((T, H, hd)), np.zeros(k_pages.shape)
    for s in range(len(seq_lens)):
        n = cu[s + 1] - cu[s]
        for i in range(n):
            p, t = int(seq_lens[s]) - n + i, cu[s] + i
            if p < 0:
                continue
            row = qkvg[t, :(H + 2 * Hkv) * hd].reshape(-1, hd).copy()
            size = np.abs(row)
            for h in range(H + Hkv):
                if q_weight is not None:
                    w = q_weight if h < H else k_weight
                    row[h] = row[h] / np.sqrt(np.mean(row[h] ** 2) + eps) * (1.0 + w)
                size[h] = np.abs(row[h])
                if cos is not None:
                    rot, half = cos.shape[1], hd // 2
                    a, b = row[h, :rot].copy(), row[h, half:half + rot].copy()
                    row[h, :rot] = a * cos[p] - b * sin[p]
                    row[h, half:half + rot] = b * cos[p] + a * sin[p]
                    size[h, :rot] = size[h, half:half + rot] = np.abs(a) + np.abs(b)
            q[t], qs[t] = row[:H], size[:H]
            pg, at = table[s][p // page], p % page
            k_pages[pg, :, at], v_pages[pg, :, at] = row[H:H + Hkv], row[H + Hkv:]
            ks[pg, :, at] = size[H:H + Hkv]
    return q, k_pages, v_pages, (qs, ks)


class Cache:
    """The bookkeeping on lists.  kv: numpy [L, 2, P, Hkv, page, hd] (changed in place)."""

    def __init__(self, kv, max_seqs, max_pages):
        self.kv, self.page = kv, kv.shape[4]
        self.table = [[-1] * max_pages for _ in range(max_seqs)]
        self.lens = [0] * max_seqs
        self.ref = [0] * kv.shape[2]
        self.refused = 0

    def _take(self, k, free):
        pages = free[:k]
        del free[:k]
        return pages

    def extend(self, slots, tokens):
        free = [p for p, r in enumerate(self.ref) if r == 0]
        seen, full = set(), False
        for s, t in zip(slots, tokens):
            if not 0 <= s < len(self.lens) or t < 0 or s in seen:
                self.refused += 1
                continue
            seen.add(s)
            old = -(-self.lens[s] // self.page)
            need = -(-(self.lens[s] + t) // self.page) - old
            if self.lens[s] + t > len(self.table[s]) * self.page:
                self.refused += 1
                continue
            if need and (full or need > len(free)):
                full = True
                self.refused += 1
                continue
            for j, p in enumerate(self._take(need, free)):
                self.table[s][old + j] = p
                self.ref[p] = 1
            self.lens[s] += t

    def fork(self, src, dst):
        table, lens = [list(r) for r in self.table], list(self.lens)
        free = [p for p, r in enumerate(self.ref) if r == 0]
        seen, full = set(), False
        data = self.kv.copy()
        for s, d in zip(src, dst):
            if not (0 <= s < len(lens) and 0 <= d < len(lens)):
                self.refused += 1
                if 0 <= d < len(lens):
                    seen.add(d)
                continue
            if d in seen:
                self.refused += 1
                continue
            seen.add(d)
            if s == d:
                continue
            whole, tail = divmod(lens[s], self.page)
            if tail and (full or not free):
                full = True
                self.refused += 1
                continue
            row = table[s][:whole]
            if tail:
                (p,) = self._take(1, free)
                self.kv[:, :, p, :, :tail] = data[:, :, table[s][whole], :, :tail]
                row.append(p)
            for p in row:
                self.ref[p] += 1
            for p in table[d]:
                if p >= 0:
                    self.ref[p] -= 1
            self.table[d] = row + [-1] * (len(table[d]) - len(row))
            self.lens[d] = lens[s]

    def free(self, slots):
        for s in slots:
            if not 0 <= s < len(self.lens):
                self.refused += 1
                continue
            for p in self.table[s]:
                if p >= 0:
                    self.ref[p] -= 1
            self.table[s] = [-1] * len(self.table[s])
            self.lens[s] = 0

    def compact(self):
        used = [p for p, r in enumerate(self.ref) if r]
        U = len(used)
        name = {}
        holes = [p for p in range(U) if not self.ref[p]]
        for a, b in zip([p for p in used if p >= U], holes):
            self.kv[:, :, b] = self.kv[:, :, a]
            self.ref[b], self.ref[a] = self.ref[a], 0
            name[a] = b
        self.table = [[name.get(p, p) for p in row] for row in self.table]

    def copy_pages(self, src, dst):
        P = len(self.ref)
        sources = {s for s in src if 0 <= s < P}
        data, seen = self.kv.copy(), set()
        for s, d in zip(src, dst):
            if 0 <= s < P and s == d:
                seen.add(d)
                continue
            first = d not in seen
            if 0 <= d < P:
                seen.add(d)
            if not (0 <= s < P and 0 <= d < P) or not first or d in sources:
                self.refused += 1
                continue
            self.kv[:, :, d] = data[:, :, s]

    def meta(self):
        return [p for row in self.table for p in row] + self.lens + self.ref
