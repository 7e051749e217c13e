"""The chunk operators in float64, eviction and verification one step after another: the tests' oracle.

Written from the definitions in ``include/xq_attn.h``; tolerances count roundings of at most half a
step each (f16 2^-11, bf16 2^-8, f32 2^-24 of a value) and are formed per element."""
import dataclasses
import math

import numpy as np

from xqattn import workloads as wl


@dataclasses.dataclass
class Params:
    scale: float
    window: int = 0
    cap: float = 0.0
    bias: float = 0.0

    def struct(self):
        import xqattn
        return xqattn.chunk_params(self.scale, self.window, self.cap, self.bias)


def slopes(H, bias):
    n = 1 << int(math.log2(H))
    return np.array([2.0 ** (-bias / n * (h + 1)) if h < n else 2.0 ** (-bias / 2 / n * (2 * (h - n) + 1)) for h in range(H)]) if bias else np.zeros(H)


def seen(rows, t, n, window, first, prefix):
    """bool [t, n]: the rows that each token sees."""
    at = rows + np.arange(t)[:, None]
    hi = at + 1 if prefix is None else np.maximum(at + 1, min(int(prefix), rows + t))
    lo = np.zeros_like(at) if not window else at + 1 - window
    if first is not None:
        lo = np.maximum(lo, np.asarray(first)[:t, None])
    r = np.arange(n)
    return (r >= lo) & (r < hi)


def scores(x, k, par, slope, at, op):
    """float64 scores [t, n] of queries x [t, D] and keys k [n, D], and how far the kernels' may be off.

    The products' operands (`op` of each), D + 8 f32 operations, f32 arithmetic on the score; a capped
    score's tanh: 2^-20 of it (the exponential 1 step and the rounding of its argument, a difference from
    1 that loses up to 2 bits, a reciprocal 1 step); a bias: its slope to 8 steps."""
    with np.errstate(all="ignore"):
        s = x @ k.T * par.scale
        ds = (np.abs(x) @ np.abs(k).T) * abs(par.scale) * (op + (k.shape[1] + 8) * 2.0**-24)
        if par.cap:
            s = par.cap * np.tanh(s / par.cap)
            ds = ds + np.abs(s) * 2.0**-20
        if par.bias:
            far = np.arange(k.shape[0])[None, :] - at[:, None]
            s = s + slope * far
            ds = ds + np.abs(slope * far) * 2.0**-20
        return s, ds + np.abs(s) * 2.0**-22


def chunk_f64(q, cache, n_tok, par, narrow, first=None, prefix=None):
    """q float [B, T, H, D] -> (out, lse, tol_out, tol_lse) in float64; padding tokens stay NaN. The kernel's
    roundings beside the scores': q8_0 / q4_0 values beside BF16 q as one f16 (2^-11), else hi + lo (2^-21); the
    weight as f16 (2^-11, below f16's normal range 2^-25 of a 1/16 of the largest) or hi + lo; one f32
    operation per row in the sums; the output's rounding."""
    B, T, H, D = q.shape
    G = H // cache.Hkv
    quant = cache.kv_type in (wl.Q8_0, wl.Q4_0)
    out, lse = np.full((B, T, H, D), np.nan), np.full((B, T, H), np.nan)
    tol, tol_lse = np.zeros((B, T, H, D)), np.zeros((B, T, H))
    op = 2.0**-11 if narrow and quant else 2.0**-21
    wt = 2.0**-11 if narrow else 2.0**-21
    slope = slopes(H, par.bias)
    for b in range(B):
        r, t = max(0, int(cache.rows[b])), int(n_tok[b])
        n = r + t
        K, V = cache.values(cache.k, b, n), cache.values(cache.v, b, n)
        see = seen(r, t, n, par.window, None if first is None else first[b], None if prefix is None else prefix[b]) & cache.has(b, n)
        for h in range(H):
            k, v = K[:, h // G], V[:, h // G]
            s, ds = scores(q[b, :t, h].astype(np.float64), k, par, slope[h], r + np.arange(t), op)
            for i in range(t):
                m = see[i]
                if not m.any():
                    out[b, i, h], lse[b, i, h] = 0.0, -np.inf
                    continue
                with np.errstate(all="ignore"):
                    top = s[i, m].max()
                    w = np.exp(s[i, m] - top)
                    z = w.sum()
                    out[b, i, h] = (w / z) @ v[m]
                    lse[b, i, h] = top + np.log(z)
                    d, vmax, c = ds[i, m].max(), np.abs(v[m]).max(0), m.sum()
                    tol[b, i, h] = vmax * (2 * d + 2.0**-20 + wt + op + c * (2.0**-24 + 2.0**-25 / z / (1 if narrow else 1024)))
                    tol[b, i, h] += 2.0**-24 if not narrow else 2.0**-8 * (np.abs(out[b, i, h]) + tol[b, i, h])
                    tol_lse[b, i, h] = d + 2.0**-20 + c * 2.0**-24 + abs(lse[b, i, h]) * 2.0**-22
    return out, lse, tol, tol_lse


def weights_f64(q, cache, n_tok, par, lse, scores_in, cols, decay, fresh, first=None, prefix=None):
    """float64 scores_out [B, cols] and its tolerance; NaN where nothing is written. Operands of 22 bits and
    more whatever q is; a weight's exponential 2^-22 and its argument's rounding; one f32 operation per
    token and head, and per part and lane of the sum."""
    B, T, H, D = q.shape
    G = H // cache.Hkv
    out, tol = np.full((B, cols), np.nan), np.zeros((B, cols))
    slope = slopes(H, par.bias)
    for b in range(B):
        r, t = max(0, int(cache.rows[b])), int(n_tok[b])
        n = r + t
        m = min(n, cols)
        old = np.zeros(m) if scores_in is None else scores_in[b, :m].astype(np.float64) * np.float64(np.float32(decay))
        if fresh:
            old[r:] = 0.0
        out[b, :m] = old
        tol[b, :m] = np.abs(old) * 2.0**-23
        if not t:
            continue
        K = cache.values(cache.k, b, n)
        see = seen(r, t, n, par.window, None if first is None else first[b], None if prefix is None else prefix[b]) & cache.has(b, n)
        for h in range(H):
            s, ds = scores(q[b, :t, h].astype(np.float64), K[:, h // G], par, slope[h], r + np.arange(t), 2.0**-21)
            l = lse[b, :t, h].astype(np.float64)[:, None]
            use = see & (l > -np.inf)
            with np.errstate(all="ignore"):
                w = np.where(use, np.exp(s - l), 0.0)
                e = np.where(use, w * (ds + np.abs(l) * 2.0**-22 + 2.0**-21 + (t * H + 40) * 2.0**-24), 0.0)
            out[b, :m] += w.sum(0)[:m]
            tol[b, :m] += e.sum(0)[:m] + 2.0**-126 * t
    return out, tol


def evict(table, rows, refs, keep, first_rows, last_rows, scores_in, positions, P, n_pages):
    """What an eviction does, sequence after sequence: (table, refs, rows_out, moves, order) where moves are (sequence,
    row from, row to) and order[b] lists, for each row held after it, the row that it was."""
    table, refs_out = table.copy(), None if refs is None else refs.copy()
    rows_out, moves, order = rows.copy(), [], []
    cols = scores_in.shape[1]
    for b, n in enumerate(rows):
        n, k = int(n), max(0, int(keep[b]))
        ok = 0 <= n <= min(cols, table.shape[1] * P)
        order.append(list(range(n)) if ok else [])
        if not ok or n <= k:
            continue
        pos = [int(p) for p in (positions[b, :n] if positions is not None else range(n))]
        newest = max(pos)
        val = [-math.inf if s != s else float(s) for s in scores_in[b, :n]]
        nan = [s != s for s in scores_in[b, :n]]
        rank = sorted(range(n), key=lambda r: (not (pos[r] < first_rows or newest - pos[r] < last_rows), nan[r], -val[r], r))
        stays = set(rank[:k])
        hole = [r for r in range(k) if r not in stays]
        tail = [r for r in range(k, n) if r in stays]
        assert len(hole) == len(tail)
        at = lambda r: int(table[b, r // P])  # noqa: E731
        if any(not 0 <= at(r) < n_pages for r in hole + tail) or (refs is not None and any(refs[at(r)] > 1 for r in hole)):
            continue
        now = list(range(k))
        for f, h in zip(tail, hole):
            now[h] = f
            moves.append((b, (at(f), f % P), (at(h), h % P)))
        order[b], rows_out[b] = now, k
        if refs is not None:
            for c in range(-(-k // P), table.shape[1]):
                if 0 <= table[b, c] < n_pages:
                    refs_out[table[b, c]] -= 1
                table[b, c] = -1
    return table, refs_out, rows_out, moves, order


def verify(logits, tokens, parents, n_tok, temperature, uniform, draft=None):
    """The walk, one token after another, in float64: (path, n_path, next, logp). `parents` None: a chain."""
    B, T, V = logits.shape
    path, n_path, nxt, logp = np.full((B, T), -1, np.int32), np.zeros(B, np.int32), np.full(B, -1, np.int32), np.zeros((B, T + 1))
    for b in range(B):
        n = int(n_tok[b])
        heat = 0.0 if uniform is None else 1.0 if temperature is None else float(temperature[b])
        greedy = not heat > 0.0
        up = [c - 1 if parents is None else int(parents[b, c]) for c in range(T)]

        def dist(i):
            x = logits[b, i].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            with np.errstate(all="ignore"):
                top = x.max()
                w = np.where(x == top, 1.0, np.exp((x - top) / (1.0 if greedy else heat)))
                return (w if top > -np.inf else np.zeros(V)), np.where(x == top, 0.0, (x - top) / (1.0 if greedy else heat)), top

        for c in range(1, n):
            if 0 <= up[c] < c:
                w, lx, top = dist(up[c])
                ok = 0 <= tokens[b, c] < V and top > -np.inf
                logp[b, c] = lx[tokens[b, c]] - np.log(w.sum()) if ok else -np.inf
        if n == 0:
            continue
        at, walk = 0, [0]
        while True:
            w, lx, top = dist(at)
            p = w / w.sum() if top > -np.inf else w
            kids = [c for c in range(1, n) if up[c] == at]
            left, stood = p.copy(), None
            for c in kids:
                x = int(tokens[b, c])
                inside = 0 <= x < V
                if greedy:
                    good = inside and top > -np.inf and x == int(np.argmax(np.where(np.isnan(logits[b, at]), -np.inf, logits[b, at])))
                elif draft is not None:
                    good = inside and float(uniform[b, c]) * float(draft[b, at, x]) < p[x]
                else:
                    good = inside and float(uniform[b, c]) * left.sum() < left[x]
                if good:
                    stood = c
                    break
                if inside:
                    left[x] = 0.0
            if stood is None:
                break
            at = stood
            walk.append(at)
        path[b, :len(walk)], n_path[b] = walk, len(walk)
        if not top > -np.inf:
            logp[b, T] = -np.inf
            continue
        if greedy:
            nxt[b] = int(np.argmax(np.where(np.isnan(logits[b, at]), -np.inf, logits[b, at])))
        else:
            if draft is not None:
                left = np.maximum(p - draft[b, at].astype(np.float64), 0.0) if kids else p
            if not left.sum() > 0.0:
                left = p
            run = np.cumsum(left)
            nxt[b] = min(int((run <= float(uniform[b, T]) * run[-1]).sum()), int(np.flatnonzero(left > 0).max()))
        logp[b, T] = lx[nxt[b]] - np.log(w.sum())
    return path, n_path, nxt, logp
