"""Eviction of the rows of least weight: every array and every pool's bytes against the oracle."""
import numpy as np
import pytest

import xqattn
from chunk_cases import evict
from conftest import case_note
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

TYPES = {"f16": wl.F16, "q8_0": wl.Q8_0, "q4_0": wl.Q4_0, "e5m2": wl.E5M2, "bf16": wl.BF16, "f32": wl.F32}


class World:
    """Pools of random bytes (padding included), a shuffled table, references, weights, positions."""

    def __init__(self, seed, kind, D, Hkv, P, rows, n_pools=2, cols=None, spare=3, head_major=False, pad=0, width=None):
        rng = self.rng = np.random.default_rng(seed)
        self.kt, self.P, self.rec, self.Hkv, self.D = TYPES[kind], P, wl.record_bytes(TYPES[kind], D), Hkv, D
        self.rows = np.array(rows, np.int32)
        need = [-(-max(0, r) // P) for r in rows]
        self.cols, self.n_pages = cols or max(1, max(need)), sum(need) + spare
        ids = rng.permutation(self.n_pages)
        self.table, at = np.full((len(rows), self.cols), -1, np.int32), 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.refs = np.zeros(self.n_pages, np.int32)
        self.refs[self.table[self.table >= 0]] = 1
        if head_major:
            self.row = self.rec + pad
            self.head = P * self.row
            self.page = Hkv * self.head + 2 * pad
        else:
            self.head = self.rec
            self.row = Hkv * self.rec + pad
            self.page = P * self.row + 2 * pad
        self.pools = [rng.integers(0, 256, self.n_pages * self.page, dtype=np.uint8) for _ in range(n_pools)]
        self.width = width or max(1, max(rows) + 2)
        self.scores = rng.random((len(rows), self.width)).astype(np.float32)
        self.positions = None

    def view(self, buf):
        return np.lib.stride_tricks.as_strided(buf, (self.n_pages, self.P, self.Hkv, self.rec), (self.page, self.row, self.head, 1))

    def run(self, torch, keep, first=0, last=0, refs=True, inplace=False, stream=None, note=""):
        case_note(f"kv_pages_evict {note}")
        dev = lambda x: None if x is None else torch.from_numpy(x.copy()).cuda()  # noqa: E731
        pools, table, rows, tr = [dev(p) for p in self.pools], dev(self.table), dev(self.rows), dev(self.refs) if refs else None
        ts, tp = dev(self.scores), dev(self.positions)
        so, po = (ts, tp) if inplace else (torch.full_like(ts, -3.0), torch.full(ts.shape, -3, dtype=torch.int32, device="cuda"))
        ro, tk = torch.zeros_like(rows), dev(np.asarray(keep, np.int32))
        ne, nb = (self.D, self.P, self.Hkv, self.n_pages), (wl.TYPE_SIZE[self.kt], self.row, self.head, self.page)
        torch.cuda.synchronize()
        xqattn.kv_pages_evict([xqattn.DevTensor(self.kt, ne, nb, p) for p in pools], table, rows, tr, tk, ts, ro, first, last, tp, so, po, stream=stream)
        torch.cuda.synchronize()
        want_t, want_r, want_rows, moves, order = evict(self.table, self.rows, self.refs if refs else None, keep, first, last, self.scores,
                                                        self.positions, self.P, self.n_pages)
        assert np.array_equal(ro.cpu().numpy(), want_rows) and np.array_equal(table.cpu().numpy(), want_t)
        assert not refs or np.array_equal(tr.cpu().numpy(), want_r)
        assert np.array_equal(rows.cpu().numpy(), self.rows)
        for got, old in zip(pools, self.pools):
            new = old.copy()
            for _, (fp, fi), (tp_, ti) in moves:
                self.view(new)[tp_, ti] = self.view(old)[fp, fi]
            assert np.array_equal(got.cpu().numpy(), new), "a pool's bytes differ"
        gs, gp = so.cpu().numpy(), None if po is None else po.cpu().numpy()
        for b, now in enumerate(order):
            n = len(now)
            assert np.array_equal(gs[b, :n].view(np.uint32), self.scores[b, now].view(np.uint32))
            assert np.array_equal(gs[b, n:], self.scores[b, n:] if inplace else np.full(self.width - n, -3.0), equal_nan=True)
            if gp is not None:
                assert np.array_equal(gp[b, :n], self.positions[b, now] if self.positions is not None else now)
        return moves


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("head_major", [False, True])
def test_types_and_strides(torch_gpu, kind, head_major):
    w = World(1, kind, 128 if kind != "f32" else 64, 3, 16, [100, 33, 64], head_major=head_major, pad=4 if kind in ("f32", "bf16") else 2)
    assert w.run(torch_gpu, [40, 32, 63], note=f"{kind} head_major={head_major}")


@pytest.mark.parametrize("rows,keep", [([1], [0]), ([1], [1]), ([0], [0]), ([0, 5, 5, 5], [3, 5, 6, -4]), ([2, 3], [1, 1]), ([1000, 17, 300], [999, 16, 150]),
                                       ([5000], [4000]), ([1025, 1024, 1023], [1024, 1, 512])])
@pytest.mark.parametrize("P", [1, 7, 16, 64])
def test_sizes(torch_gpu, rows, keep, P):
    World(2, "e5m2", 32, 1, P, rows).run(torch_gpu, keep, note=f"{rows} {keep} page {P}")


def test_ties_zeros_infinities_and_nan(torch_gpu):
    """Equal weights go by index, NaN the least, -0 is 0, and so at every place of the budget."""
    w = World(3, "q8_0", 64, 2, 16, [300] * 6)
    w.scores[0] = 0.0
    w.scores[1, ::2] = -0.0
    w.scores[1, 1::2] = 0.0
    w.scores[2] = w.rng.integers(0, 3, w.width)
    w.scores[3] = w.rng.choice(np.array([np.nan, np.inf, -np.inf, 1.0, -1.0, 0.0, 1e-42], np.float32), w.width)
    w.scores[4] = np.float32(np.nan)
    w.scores[5] = -w.scores[5]
    for keep in (1, 50, 299):
        w.run(torch_gpu, [keep] * 6, note=f"ties, keep {keep}")
    for k in range(40, 60):
        w.run(torch_gpu, [k] * 6, first=3, last=5, note=f"ties, keep {k}, protected")


def test_protected_rows_and_moved_positions(torch_gpu):
    w = World(4, "q4_0", 128, 2, 16, [200, 200, 200])
    w.scores[:, :8] = 0.0
    w.scores[:, 190:200] = 0.0
    w.run(torch_gpu, [60, 12, 5], first=4, last=9, note="protected, and more protected than the budget")
    w.positions = np.stack([w.rng.permutation(w.width) for _ in range(3)]).astype(np.int32)
    w.run(torch_gpu, [60, 12, 5], first=4, last=9, note="protected by positions")
    w.positions[0, :200] = 0x7fffffff - np.arange(200)
    w.positions[1, :200] = -0x80000000 + np.arange(200)
    w.positions[2, ::2] = -0x80000000
    w.positions[2, 1::2] = 0x7fffffff
    w.run(torch_gpu, [60, 12, 5], first=4, last=0x7fffffff, note="positions at the ends of 32 bits")


def test_shared_and_missing_pages_leave_a_sequence(torch_gpu):
    w = World(5, "f16", 64, 2, 16, [100, 100, 100, 100], spare=0)
    # 0 and 1 share their first page; 2's page of tails is none; 3 is fine
    old = w.table[1, 0]
    w.table[1, 0] = w.table[0, 0]
    w.refs[w.table[0, 0]], w.refs[old] = 2, 0
    w.table[2, 5] = -1
    w.scores[:, :8] = 0.0
    w.scores[2, 80:96] = 2.0
    assert {m[0] for m in w.run(torch_gpu, [50] * 4, note="shared")} == {3}
    # without references no page is shared (the caller says so), and a page that is none still leaves its sequence
    w.table[1, 0] = old
    assert {m[0] for m in w.run(torch_gpu, [50] * 4, refs=False, note="without references")} == {0, 1, 3}
    # a shared page of which no row is written does no harm, and loses one holder where it is given back
    w = World(6, "f16", 64, 2, 16, [100, 100], spare=0)
    w.table[1, 6], w.refs[w.table[0, 6]], w.refs[w.table[1, 6]] = w.table[0, 6], 2, 0
    assert {m[0] for m in w.run(torch_gpu, [50] * 2, note="shared tail")} == {0, 1}


def test_rows_beyond_table_or_columns_leave_a_sequence(torch_gpu):
    w = World(7, "f16", 64, 2, 16, [64, 60, 64], width=62)
    w.rows[:] = [65, 60, -3]
    assert {m[0] for m in w.run(torch_gpu, [30] * 3, note="rows beyond")} == {1}


@pytest.mark.parametrize("n,k", [(40000, 39990), (33000, 5)])
def test_more_rows_than_lds_holds(torch_gpu, n, k):
    w = World(12, "e5m2", 32, 1, 64, [n, 100])
    w.positions = np.stack([w.rng.permutation(w.width) for _ in range(2)]).astype(np.int32)
    w.run(torch_gpu, [k, 50], first=4, last=100, note=f"{n} rows to {k}")


def test_in_place_again_and_again(torch_gpu):
    """A cache held at its budget: a new row each step, weights and positions moved in place."""
    w = World(8, "q8_0", 128, 2, 16, [41, 50], spare=4)
    w.positions = np.tile(np.arange(w.width, dtype=np.int32), (2, 1))
    for step in range(6):
        w.run(torch_gpu, [40, 45], first=2, last=3, inplace=True, note=f"in place, step {step}")
        _, _, rows, moves, order = evict(w.table, w.rows, None, [40, 45], 2, 3, w.scores, w.positions, w.P, w.n_pages)
        for b, now in enumerate(order):
            w.scores[b, :len(now)], w.positions[b, :len(now)] = w.scores[b, now], w.positions[b, now]
            w.scores[b, len(now)], w.positions[b, len(now)] = w.rng.random(), 100 + step
            w.rows[b] = len(now) + 1


def test_many_pools_and_many_sequences(torch_gpu):
    World(9, "e5m2", 32, 1, 4, [30, 9], n_pools=83).run(torch_gpu, [11, 8], note="83 pools")
    rng = np.random.default_rng(1)
    rows = [int(x) for x in rng.integers(0, 40, 300)]
    World(10, "e5m2", 32, 1, 4, rows).run(torch_gpu, [int(x) for x in rng.integers(0, 30, 300)], note="300 sequences")


def test_replays_on_another_stream(torch_gpu):
    torch = torch_gpu
    w = World(11, "q8_0", 64, 2, 16, [90, 70], spare=0)
    pools = [torch.from_numpy(p.copy()).cuda() for p in w.pools]
    start = [p.clone() for p in pools]
    table, rows, refs = (torch.from_numpy(x.copy()).cuda() for x in (w.table, w.rows, w.refs))
    scores, so, ro = torch.from_numpy(w.scores).cuda(), torch.zeros(w.scores.shape, device="cuda"), torch.zeros_like(rows)
    keep = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    desc = [xqattn.DevTensor(w.kt, (w.D, w.P, w.Hkv, w.n_pages), (wl.TYPE_SIZE[w.kt], w.row, w.head, w.page), p) for p in pools]
    case_note("kv_pages_evict capture")
    ws = xqattn.kv_pages_evict(desc, table, rows, refs, keep, scores, ro, 0, 0, None, so)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xqattn.kv_pages_evict(desc, table, rows, refs, keep, scores, ro, 0, 0, None, so, workspace=ws)
    side = torch.cuda.Stream()
    for n in ([90, 70], [90, 41], [12, 70]):
        for k in ([40, 40], [5, 64]):
            results = []
            for how in ("replay", "eager"):
                for p, s in zip(pools, start):
                    p.copy_(s)
                table.copy_(torch.from_numpy(w.table)), refs.copy_(torch.from_numpy(w.refs))
                rows.copy_(torch.tensor(n, dtype=torch.int32)), keep.copy_(torch.tensor(k, dtype=torch.int32))
                so.fill_(-1.0)
                torch.cuda.synchronize()
                if how == "replay":
                    graph.replay()
                else:
                    xqattn.kv_pages_evict(desc, table, rows, refs, keep, scores, ro, 0, 0, None, so, stream=side)
                torch.cuda.synchronize()
                results.append([x.clone() for x in (*pools, table, refs, ro, so)])
            assert all(torch.equal(a, b) for a, b in zip(*results))
