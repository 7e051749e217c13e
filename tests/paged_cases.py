"""Paged caches on the host and the paged operators in float64: the tests' oracle.

Written from the definitions in ``include/xq_attn.h``; a tolerance counts roundings of at most
half a step each (f16 2^-11, bf16 2^-8, f32 2^-24 of a value) and is formed per element."""
import numpy as np

import oracle
from xqattn import workloads as wl


def bf16(x):
    """float32 -> the float32 values of its bf16 rounding (to even)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


class Cache:
    """K and V pools in host bytes: pages of [page_rows][heads][record] or head-major, with `pad`
    bytes between the pieces; table and rows."""

    def __init__(self, rng, kv_type, D, Hkv, P, rows, extra, cols=None, spare=2, head_major=False, pad=0, shuffle=True):
        self.kv_type, self.D, self.Hkv, self.P = kv_type, D, Hkv, P
        self.rec = wl.record_bytes(kv_type, D)
        need = [-(-(r + e) // P) for r, e in zip(rows, extra)]
        self.cols = cols or max(1, max(need))
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages) if shuffle else np.arange(self.n_pages)
        self.table = np.full((len(rows), self.cols), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.rows = np.array(rows, np.int32)
        if head_major:
            self.row = self.rec + pad
            self.head = P * self.row + 2 * pad
            self.page = Hkv * self.head
        else:
            self.head = self.rec + pad
            self.row = Hkv * self.head + 2 * pad
            self.page = P * self.row
        self.k = self._plane(rng)
        self.v = self._plane(rng)

    def _plane(self, rng):
        x = rng.standard_normal((self.n_pages, self.P, self.Hkv, self.D)).astype(np.float32)
        raw = oracle.quantize(self.kv_type, x).reshape(self.n_pages, self.P, self.Hkv, self.rec)
        buf = np.full(self.n_pages * self.page, 0xAB, np.uint8)
        self.view(buf)[...] = raw
        return buf

    def view(self, buf):
        """The plane's records, [n_pages, P, Hkv, rec], over its bytes."""
        return np.lib.stride_tricks.as_strided(buf, (self.n_pages, self.P, self.Hkv, self.rec), (self.page, self.row, self.head, 1))

    def place(self, b, r):
        return int(self.table[b, r // self.P]), r % self.P

    def values(self, buf, b, n):
        """float64 [n, Hkv, D]: rows 0..n-1 of sequence b; NaN rows where there is no page."""
        out = np.full((n, self.Hkv, self.D), np.nan)
        view = self.view(buf)
        for r in range(n):
            if r // self.P < self.cols:
                p, i = self.place(b, r)
                if 0 <= p < self.n_pages:
                    out[r] = oracle.dequant(self.kv_type, np.ascontiguousarray(view[p, i]).reshape(-1), self.Hkv * self.D).reshape(self.Hkv, self.D)
        return out

    def has(self, b, n):
        """Which of rows 0..n-1 have a page."""
        return np.array([r // self.P < self.cols and 0 <= self.table[b, r // self.P] < self.n_pages for r in range(n)], bool)

    def device(self, torch):
        import xqattn
        dk, dv = (torch.from_numpy(x.copy()).cuda() for x in (self.k, self.v))
        ne, nb = (self.D, self.P, self.Hkv, self.n_pages), (wl.TYPE_SIZE[self.kv_type], self.row, self.head, self.page)
        return xqattn.KvPages(xqattn.DevTensor(self.kv_type, ne, nb, dk), xqattn.DevTensor(self.kv_type, ne, nb, dv),
                              torch.from_numpy(self.table.copy()).cuda(), torch.from_numpy(self.rows.copy()).cuda())


def ancestors(parents):
    """bool [T, T]: which tokens each token sees."""
    T = len(parents)
    seen = np.zeros((T, T), bool)
    for i in range(T):
        j = i
        while j >= 0:
            seen[i, j] = True
            p = int(parents[j])
            j = p if 0 <= p < j else -1
    return seen


def random_parents(rng, T):
    return np.array([-1] + [rng.integers(-1, i) for i in range(1, T)], np.int32)


def tree_f64(q, cache, parents, n_tok, scale, narrow):
    """q float [B, T, H, D] -> (out, lse, tol_out, tol_lse) in float64; padding tokens stay NaN.

    `narrow`: BF16 q. The kernel's roundings: scores, each product's operands (f32 q as hi + lo:
    2^-21; q8_0/q4_0 K as one f16 where narrow: 2^-11), D + 8 f32 operations; a weight's
    exponent argument 2^-22 of the score; the weight as f16 (narrow: 2^-11 of it and, below the f16
    normal range, 2^-25 of the 1/16 of the largest) or hi + lo (2^-21); values alike; one f32
    operation per row in the sums; the output's rounding."""
    B, T, H, D = q.shape
    G = H // cache.Hkv
    quant = cache.kv_type in (wl.Q8_0, wl.Q4_0)
    out, lse = np.full((B, T, H, D), np.nan), np.full((B, T, H), np.nan)
    tol, tol_lse = np.zeros((B, T, H, D)), np.zeros((B, T, H))
    op = 2.0**-11 if narrow and quant else 2.0**-21
    wt = 2.0**-11 if narrow else 2.0**-21
    for b in range(B):
        n0, t = max(0, int(cache.rows[b])), int(n_tok[b])
        n = n0 + t
        K, V, has = cache.values(cache.k, b, n), cache.values(cache.v, b, n), cache.has(b, n)
        tree = ancestors(parents[b])
        for i in range(t):
            rows = np.array([r for r in range(n) if has[r] and (r < n0 or tree[i, r - n0])], int)
            for h in range(H):
                if not len(rows):
                    out[b, i, h], lse[b, i, h] = 0.0, -np.inf
                    continue
                k, v = K[rows, h // G], V[rows, h // G]
                x = q[b, i, h].astype(np.float64)
                s = (k @ x) * scale
                m = s.max()
                w = np.exp(s - m)
                z = w.sum()
                out[b, i, h] = (w / z) @ v
                lse[b, i, h] = m + np.log(z)
                big = (np.abs(k) @ np.abs(x)).max() * abs(scale)
                ds = big * (op + (D + 8) * 2.0**-24) + np.abs(s).max() * 2.0**-22
                vmax = np.abs(v).max(0)
                tol[b, i, h] = vmax * (2 * ds + 2.0**-20 + wt + op + len(rows) * (2.0**-24 + 2.0**-25 / z / (1 if narrow else 1024)))
                tol[b, i, h] += 2.0**-24 if not narrow else 2.0**-8 * (np.abs(out[b, i, h]) + tol[b, i, h])
                tol_lse[b, i, h] = ds + 2.0**-20 + len(rows) * 2.0**-24 + abs(lse[b, i, h]) * 2.0**-22
    return out, lse, tol, tol_lse


def rope_f64(x, w, pos, n_rot, base, mode, eps, scale=1.0, ff=None, attn=1.0):
    """x [..., heads, D] of tokens at pos [...] -> float64."""
    x = x.astype(np.float64)
    D = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    half = n_rot // 2
    i = np.arange(half)
    t = pos.astype(np.float64)[..., None, None] * scale * float(base) ** (-2.0 * i / max(1, n_rot))
    if ff is not None:
        t = t / ff.astype(np.float64)
    c, s = np.cos(t) * attn, np.sin(t) * attn
    y = x.copy()
    a, b = (slice(0, half), slice(half, n_rot)) if mode == 0 else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


class Pages:
    """The page operations on host tables, one sequence and one page after another."""

    def __init__(self, table, rows, refs, P):
        self.table, self.rows, self.refs, self.P = table.copy(), rows.copy(), refs.copy(), P

    def take(self):
        free = np.flatnonzero(self.refs == 0)
        if not len(free):
            return -1
        self.refs[free[0]] = 1
        return int(free[0])

    def reserve(self, want):
        got = np.zeros(len(want), np.int32)
        cols = self.table.shape[1]
        for b, w in enumerate(want):
            for c in range(min(cols, -(-max(0, int(w)) // self.P))):
                if self.table[b, c] == -1:
                    self.table[b, c] = self.take()
            held = 0
            while held < cols and 0 <= self.table[b, held] < len(self.refs):
                held += 1
            got[b] = held * self.P
        return got

    def fork(self, parents, children):
        """done, and (source page, page, rows) copies."""
        done, copies = np.zeros(len(parents), np.int32), []
        n_seq, cols = self.table.shape
        rows0 = self.rows.copy()
        for i, (p, c) in enumerate(zip(parents, children)):
            if not (0 <= p < n_seq and 0 <= c < n_seq) or c in children[:i] or c in parents:
                continue
            held = int(rows0[p])
            if self.rows[c] != 0 or self.table[c, 0] != -1 or held < 0 or held > cols * self.P:
                continue
            full, part = divmod(held, self.P)
            page = -1
            if part:
                src = int(self.table[p, full])
                if not 0 <= src < len(self.refs):
                    continue
                page = self.take()
                if page < 0:
                    continue
                copies.append((src, page, part))
                self.table[c, full] = page
            for x in range(full):
                q = int(self.table[p, x])
                self.table[c, x] = q
                if 0 <= q < len(self.refs):
                    self.refs[q] += 1
            self.rows[c] = held
            done[i] = 1
        return done, copies

    def release(self, seqs):
        for b in seqs:
            if 0 <= b < len(self.table):
                for c in range(self.table.shape[1]):
                    q = int(self.table[b, c])
                    if 0 <= q < len(self.refs):
                        self.refs[q] -= 1
                    self.table[b, c] = -1
                self.rows[b] = 0
