"""Pages of the cache copied, compacted, reserved, forked and released, against the same done
one after another on the host; and one speculative step through all of the paged operators."""
import numpy as np
import pytest

import xqattn
from conftest import case_note
from paged_cases import Cache, Pages, bf16, random_parents, rope_f64, tree_f64
from test_gpu_fa_tree import dst4, rows4
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

TYPES = {"f16": wl.F16, "q8_0": wl.Q8_0, "q4_0": wl.Q4_0, "e5m2": wl.E5M2}


def i32(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def pool_set(torch, rng, layouts, P, n_pages):
    """Pools of random bytes: (kv type, D, heads, head major, pad) each."""
    host, dev = [], []
    for kt, D, Hkv, major, pad in layouts:
        c = Cache(rng, TYPES[kt], D, Hkv, P, [P * n_pages], [0], spare=0, head_major=major, pad=pad, shuffle=False)
        c.k = rng.integers(0, 256, c.k.size, dtype=np.uint8)
        host.append(c)
        dev.append(xqattn.DevTensor(c.kv_type, (D, P, Hkv, n_pages), (wl.TYPE_SIZE[c.kv_type], c.row, c.head, c.page), torch.from_numpy(c.k.copy()).cuda()))
    return host, dev


LAYOUTS = [("f16", 128, 8, False, 0), ("q8_0", 256, 4, False, 0), ("q4_0", 128, 3, True, 0), ("e5m2", 64, 1, False, 0),
           ("q4_0", 32, 1, False, 2), ("q8_0", 64, 5, True, 6), ("f16", 96, 2, False, 10)]


@pytest.mark.parametrize("P,n_pages,n", [(16, 9, 4), (1, 30, 13), (7, 5, 1), (64, 80, 40)])
def test_copy(torch_gpu, P, n_pages, n):
    torch = torch_gpu
    rng = np.random.default_rng(P)
    host, dev = pool_set(torch, rng, LAYOUTS, P, n_pages)
    ids = rng.permutation(n_pages)[:2 * n]
    src, dst = ids[:n].copy(), ids[n:].copy()
    src = np.concatenate([src, [n_pages, 0, -1, 2]])
    dst = np.concatenate([dst, [1, -1, 3, 2**31 - 1]])
    case_note(f"copy P {P} pages {n_pages} pairs {n}")
    xqattn.kv_pages_copy(dev, i32(torch, src), i32(torch, dst))
    torch.cuda.synchronize()
    for c, d in zip(host, dev):
        v = c.view(c.k)
        for s, t in zip(src[:n], dst[:n]):
            v[t] = v[s]
        assert np.array_equal(d.t.cpu().numpy(), c.k)


def test_copy_many_pools(torch_gpu):
    """More pools than one launch takes."""
    torch = torch_gpu
    rng = np.random.default_rng(3)
    host, dev = pool_set(torch, rng, [LAYOUTS[i % 7] for i in range(95)], 4, 6)
    xqattn.kv_pages_copy(dev, i32(torch, [0, 5]), i32(torch, [3, 1]))
    torch.cuda.synchronize()
    for c, d in zip(host, dev):
        v = c.view(c.k)
        v[3], v[1] = v[0].copy(), v[5].copy()
        assert np.array_equal(d.t.cpu().numpy(), c.k)


@pytest.mark.parametrize("P", [1, 5, 16, 64])
@pytest.mark.parametrize("seed", range(4))
def test_compact(torch_gpu, P, seed):
    """Paths of any length (past a wave's 64 rows, empty, full), entries below their place skipped,
    rows in pages that are none skipped."""
    torch = torch_gpu
    rng = np.random.default_rng(10 * P + seed)
    B, T = 5, (6, 25, 64, 150)[seed]
    rows = rng.integers(0, 90, B)
    need = [-(-(int(r) + T) // P) for r in rows]
    n_pages = sum(need) + 1
    table = np.full((B, max(need)), -1, np.int32)
    ids = rng.permutation(n_pages)
    for b in range(B):
        table[b, :need[b]] = ids[sum(need[:b]):sum(need[:b + 1])]
    lens = [0, T, min(5, T), int(rng.integers(1, T)), T // 2]
    path = np.zeros((B, T), np.int32)
    for b, n in enumerate(lens):
        path[b, :n] = np.sort(rng.choice(T, n, replace=False))
        path[b, n:] = 10**6
    if seed == 1:
        path[4, 3] = 1  # below its place
        table[2, int(rows[2]) // P] = n_pages
    n_path = np.array(lens, np.int32)
    if seed == 2:
        n_path[0], n_path[1] = -3, 10**9
    host, dev = pool_set(torch, rng, LAYOUTS, P, n_pages)
    out = i32(torch, np.zeros(B))
    case_note(f"compact P {P} seed {seed} rows {rows} paths {lens}")
    xqattn.kv_pages_compact(dev, i32(torch, table), i32(torch, rows), i32(torch, path), i32(torch, n_path), out)
    torch.cuda.synchronize()
    n_path = np.clip(n_path, 0, T)
    assert np.array_equal(out.cpu().numpy(), rows + n_path)
    for c, d in zip(host, dev):
        v = c.view(c.k)
        for b in range(B):
            for j in range(n_path[b]):
                e = int(path[b, j])
                s, t = int(rows[b]) + e, int(rows[b]) + j
                if e > j and s // P < table.shape[1] and all(0 <= table[b, r // P] < n_pages for r in (s, t)):
                    v[table[b, t // P], t % P] = v[table[b, s // P], s % P]
        assert np.array_equal(d.t.cpu().numpy(), c.k)


def state(torch, m):
    return [i32(torch, x) for x in (m.table, m.rows, m.refs)]


def same(m, dev):
    for x, d in zip((m.table, m.rows, m.refs), dev):
        assert np.array_equal(x, d.cpu().numpy())


@pytest.mark.parametrize("seed,n_seq,cols,n_pages,P", [(0, 3, 4, 10, 16), (1, 70, 9, 200, 5), (2, 20, 130, 1500, 1), (3, 1, 1, 1, 64), (4, 1500, 3, 5000, 8)])
def test_reserve_fork_release_in_turn(torch_gpu, seed, n_seq, cols, n_pages, P):
    """Random turns of the three, pages running out among them, ids out of range and named twice."""
    torch = torch_gpu
    rng = np.random.default_rng(seed)
    m = Pages(np.full((n_seq, cols), -1, np.int32), np.zeros(n_seq, np.int32), np.zeros(n_pages, np.int32), P)
    host, dev = pool_set(torch, rng, LAYOUTS[:3], P, n_pages)
    t, r, f = state(torch, m)
    for turn in range(6):
        case_note(f"pages seed {seed} turn {turn}: {int((m.refs == 0).sum())} free")
        want = np.where(rng.random(n_seq) < 0.5, rng.integers(-1, cols * P + 2 * P, n_seq), m.rows).astype(np.int32)
        if turn == 1:
            want[:] = 2**31 - 1
        got = i32(torch, np.zeros(n_seq))
        xqattn.kv_pages_reserve(t, f, P, i32(torch, want), got)
        torch.cuda.synchronize()
        hg = m.reserve(want)
        assert np.array_equal(got.cpu().numpy(), hg)
        same(m, (t, r, f))
        m.rows = np.minimum(rng.integers(0, cols * P + 1, n_seq), hg).astype(np.int32)
        r.copy_(i32(torch, m.rows))
        seqs = rng.integers(-2, n_seq + 2, max(1, n_seq // 2))
        xqattn.kv_pages_release(t, r, f, i32(torch, seqs))
        torch.cuda.synchronize()
        m.release(dict.fromkeys(seqs.tolist()))
        same(m, (t, r, f))
        n = min(1024, max(1, n_seq))
        parents, children = rng.integers(-1, n_seq + 1, n), rng.integers(-1, n_seq + 1, n)
        if turn % 2:  # parents and children apart, most of them good
            parents, children = rng.integers(0, max(1, n_seq // 2), n), rng.integers(n_seq // 2, n_seq, n)
        done = i32(torch, np.full(n, 9))
        xqattn.kv_pages_fork(dev, t, r, f, i32(torch, parents), i32(torch, children), done)
        torch.cuda.synchronize()
        hd, copies = m.fork(parents.tolist(), children.tolist())
        assert np.array_equal(done.cpu().numpy(), hd)
        same(m, (t, r, f))
        for c, d in zip(host, dev):
            v = c.view(c.k)
            for s, p, rows in copies:
                v[p, :rows] = v[s, :rows]
            assert np.array_equal(d.t.cpu().numpy(), c.k)


def test_pages_in_a_graph(torch_gpu):
    """Release, fork and compact captured once, replayed on tables changed in between."""
    torch = torch_gpu
    rng = np.random.default_rng(5)
    P, n_seq, cols, n_pages = 8, 6, 4, 40
    host, dev = pool_set(torch, rng, LAYOUTS[:2], P, n_pages)
    m = Pages(np.full((n_seq, cols), -1, np.int32), np.zeros(n_seq, np.int32), np.zeros(n_pages, np.int32), P)
    m.reserve(np.array([30, 17, 8, 0, 0, 0]))
    m.rows[:3] = [25, 17, 8]
    t, r, f = state(torch, m)
    kids, folk, done, out = i32(torch, [3, 4, 5]), i32(torch, [0, 1, 2]), i32(torch, [0] * 3), i32(torch, [0] * n_seq)
    path, n_path = i32(torch, [[1, 3]] * n_seq), i32(torch, [2, 0, 0, 0, 0, 0])
    ws = torch.empty(4096, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        xqattn.kv_pages_release(t, r, f, kids)
        xqattn.kv_pages_fork(dev, t, r, f, folk, kids, done, workspace=ws)
        xqattn.kv_pages_compact(dev, t, r, path, n_path, out)
    for turn in range(4):
        order = rng.permutation(3)
        folk.copy_(i32(torch, order))
        rows0 = int(rng.integers(17, 28))
        m.rows[0] = rows0
        r.copy_(i32(torch, m.rows))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        m.release([3, 4, 5])
        _, copies = m.fork(order.tolist(), [3, 4, 5])
        same(m, (t, r, f))
        for c, d in zip(host, dev):
            v = c.view(c.k)
            for s, p, rows in copies:
                v[p, :rows] = v[s, :rows]
            for j, e in enumerate([1, 3]):
                s, q = rows0 + e, rows0 + j
                v[m.table[0, q // P], q % P] = v[m.table[0, s // P], s % P]
            assert np.array_equal(d.t.cpu().numpy(), c.k), turn


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
def test_a_speculative_step(torch_gpu, kt, narrow):
    """Reserve, norm and turn a tree's tokens into the cache, attend, keep the accepted path, fork,
    and decode one token of both holders: the outputs are the float64 attention over what the cache
    holds, and the kept rows are the path's."""
    torch = torch_gpu
    rng = np.random.default_rng(77)
    D, H, Hkv, P, B, T = 128, 16, 4, 16, 3, 10
    held = [37, 5, 64]
    c = Cache(rng, TYPES[kt], D, Hkv, P, held + [0], [0] * 4, cols=8, spare=12)
    used = c.table.copy()
    refs = np.zeros(c.n_pages, np.int32)
    refs[used[used >= 0]] = 1
    dev = c.device(torch)
    t, r, f = dev.table, dev.rows, i32(torch, refs)
    got = i32(torch, [0] * 4)
    xqattn.kv_pages_reserve(t, f, P, i32(torch, [x + T for x in held] + [0]), got)
    torch.cuda.synchronize()
    assert all(g >= h + T for g, h in zip(got.cpu().tolist(), held))
    c.table = t.cpu().numpy()
    dt, typ = (torch.bfloat16, wl.BF16) if narrow else (torch.float32, wl.F32)
    three = xqattn.KvPages(dev.k, dev.v, t[:3].contiguous(), r[:3].contiguous())
    q, k, v = (rng.standard_normal((B, T, h, D)).astype(np.float32) for h in (H, Hkv, Hkv))
    q, k, v = bf16(q), bf16(k), bf16(v)
    parents = np.stack([random_parents(rng, T) for _ in range(B)])
    depth = np.zeros((B, T), np.int32)
    for b in range(B):
        for i in range(T):
            depth[b, i] = 0 if parents[b, i] < 0 else depth[b, parents[b, i]] + 1
    pos = np.array(held)[:, None] + depth
    w = [(1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
    put = lambda x, d=None: torch.from_numpy(np.ascontiguousarray(x)).cuda().to(d) if d else torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    tq, tk, tv = (put(x, dt) for x in (q, k, v))
    turned, out = torch.zeros_like(tq), torch.zeros_like(tq)
    lse = torch.zeros((B, T, H), device="cuda")
    tp = put(parents)
    xqattn.qk_norm_rope(rows4(torch, tq, typ), rows4(torch, tk, typ), rows4(torch, tv, typ), put(pos.astype(np.int32)),
                        xqattn.rope_params(D, 1e4), rows4(torch, turned, typ), three, q_weight=put(w[0]), k_weight=put(w[1]))
    xqattn.fa_tree(rows4(torch, turned, typ), three, dst4(torch, out, typ), D**-0.5, parents=tp, lse=lse)
    torch.cuda.synchronize()
    qt = turned.float().cpu().numpy()
    want_q = rope_f64(q, w[0], pos, D, 1e4, 0, 1e-6)
    assert np.all(np.abs(qt - want_q) <= 2.0**-18 * 16 + (2.0**-8 * np.abs(want_q) if narrow else 0))
    c.k, c.v = dev.k.t.cpu().numpy(), dev.v.t.cpu().numpy()
    c.table, c.rows = c.table[:3], np.array(held, np.int32)
    w_out, w_lse, tol, tol_lse = tree_f64(qt, c, parents, [T] * B, D**-0.5, narrow)
    assert np.all(np.abs(out.float().cpu().numpy() - w_out) <= tol)
    assert np.all(np.abs(lse.cpu().numpy() - w_lse) <= tol_lse)
    # the deepest path is accepted
    paths = []
    for b in range(B):
        i, p = int(depth[b].argmax()), []
        while i >= 0:
            p.append(i)
            i = int(parents[b, i])
        paths.append(p[::-1])
    n = max(map(len, paths))
    path = np.array([p + [0] * (n - len(p)) for p in paths], np.int32)
    new = i32(torch, [0] * 3)
    xqattn.kv_pages_compact([dev.k, dev.v], three.table, three.rows, put(path), i32(torch, [len(p) for p in paths]), new)
    r[:3] = new
    kept = [c.values(x, b, held[b] + T) for x in (c.k, c.v) for b in range(B)]
    # a fourth sequence forks from the first; both decode one token
    done = i32(torch, [0])
    xqattn.kv_pages_fork([dev.k, dev.v], t, r, f, i32(torch, [0]), i32(torch, [3]), done)
    xqattn.kv_pages_reserve(t, f, P, r + 1, got)
    torch.cuda.synchronize()
    assert done.item() == 1
    c.table, c.rows = t.cpu().numpy(), r.cpu().numpy()
    assert np.array_equal(c.rows, [held[b] + len(paths[b]) for b in range(3)] + [held[0] + len(paths[0])])
    c.k, c.v = dev.k.t.cpu().numpy(), dev.v.t.cpu().numpy()
    for x, plane in enumerate((c.k, c.v)):
        for b, src in ((0, 0), (1, 1), (2, 2), (3, 0)):
            rows = list(range(held[src])) + [held[src] + i for i in paths[src]]
            assert np.array_equal(c.values(plane, b, int(c.rows[b])), kept[3 * x + src][rows])
    assert c.table[3, int(c.rows[3]) // P] != c.table[0, int(c.rows[0]) // P]
    q1 = bf16(rng.standard_normal((4, 1, H, D)).astype(np.float32))
    k1, v1 = (bf16(rng.standard_normal((4, 1, Hkv, D)).astype(np.float32)) for _ in range(2))
    a, o1 = put(q1, dt), torch.zeros((4, 1, H, D), dtype=dt, device="cuda")
    xqattn.qk_norm_rope(rows4(torch, a, typ), rows4(torch, put(k1, dt), typ), rows4(torch, put(v1, dt), typ), r.clone(), xqattn.rope_params(D, 1e4),
                        rows4(torch, a, typ), dev, q_weight=put(w[0]), k_weight=put(w[1]))
    xqattn.fa_tree(rows4(torch, a, typ), dev, dst4(torch, o1, typ), D**-0.5)
    torch.cuda.synchronize()
    c.k, c.v = dev.k.t.cpu().numpy(), dev.v.t.cpu().numpy()
    w_out, _, tol, _ = tree_f64(a.float().cpu().numpy(), c, np.full((4, 1), -1, np.int32), [1] * 4, D**-0.5, narrow)
    assert np.all(np.abs(o1.float().cpu().numpy() - w_out) <= tol)
