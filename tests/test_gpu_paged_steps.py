"""Several speculative steps of a server over the paged cache, one after another: reserve, norms and
rotation into the cache, attention, the accepted path kept, and the new row counts taken over for the
next step. Eager and as one captured graph that is replayed for every step."""
import numpy as np
import pytest

import xqattn
from conftest import case_note
from paged_cases import Cache, random_parents, tree_f64
from test_gpu_fa_tree import TYPES, check, dst4, rows4
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

D, H, HKV, P, B, T, LAYERS = 128, 8, 4, 16, 3, 7, 2
HELD = [30, 1, 64]


class Server:
    """The state of a server's layers on the device, and one step over it."""

    def __init__(self, torch, kt, seed):
        self.torch = torch
        self.caches = [Cache(np.random.default_rng(seed + n), TYPES[kt], D, HKV, P, HELD, [0] * B, cols=12, spare=20) for n in range(LAYERS)]
        for c in self.caches[1:]:
            c.table = self.caches[0].table.copy()  # one table serves all layers
        kv = [c.device(torch) for c in self.caches]
        self.table, self.rows = kv[0].table, kv[0].rows
        self.kv = [xqattn.KvPages(x.k, x.v, self.table, self.rows) for x in kv]
        refs = np.zeros(self.caches[0].n_pages, np.int32)
        refs[self.caches[0].table[self.caches[0].table >= 0]] = 1
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.refs = torch.from_numpy(refs).cuda()
        self.want, self.got, self.new_rows, self.n_path = (i32(B) for _ in range(4))
        self.positions, self.parents, self.path = i32(B, T), i32(B, T), i32(B, T)
        f32 = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        self.q, self.out = ([f32(B, T, H, D) for _ in range(LAYERS)] for _ in range(2))
        self.k, self.v = ([f32(B, T, HKV, D) for _ in range(LAYERS)] for _ in range(2))
        self.turned = [f32(B, T, H, D) for _ in range(LAYERS)]
        self.w = torch.ones(D, device="cuda")
        args = rows4(torch, self.turned[0], wl.F32), self.kv[0], dst4(torch, self.out[0], wl.F32)
        self.w0 = torch.zeros(4096, dtype=torch.uint8, device="cuda")
        self.w1 = torch.zeros(xqattn.fa_tree_workspace(*args) + 256, dtype=torch.uint8, device="cuda")

    def inputs(self, step):
        """Another step's tokens, trees and accepted paths, of the step alone."""
        rng = np.random.default_rng(500 + step)
        put = lambda dst, x: dst.copy_(self.torch.from_numpy(np.ascontiguousarray(x)))  # noqa: E731
        for n in range(LAYERS):
            for dst, h in ((self.q[n], H), (self.k[n], HKV), (self.v[n], HKV)):
                put(dst, rng.standard_normal((B, T, h, D)).astype(np.float32))
        self.host_parents = np.stack([random_parents(rng, T) for _ in range(B)])
        paths, depth = np.zeros((B, T), np.int32), np.zeros((B, T), np.int32)
        n_path = np.zeros(B, np.int32)
        for b in range(B):
            for i in range(T):
                depth[b, i] = 0 if self.host_parents[b, i] < 0 else depth[b, self.host_parents[b, i]] + 1
            i, p = int(depth[b].argmax()), []
            while i >= 0:
                p.append(i)
                i = int(self.host_parents[b, i])
            n_path[b] = len(p)
            paths[b, :len(p)] = p[::-1]
        put(self.positions, self.rows.cpu().numpy()[:, None] + depth)
        put(self.parents, self.host_parents)
        put(self.path, paths)
        put(self.n_path, n_path)

    def attend(self):
        torch = self.torch
        torch.add(self.rows, T, out=self.want)
        xqattn.kv_pages_reserve(self.table, self.refs, P, self.want, self.got, workspace=self.w0)
        for n in range(LAYERS):
            xqattn.qk_norm_rope(*(rows4(torch, x[n], wl.F32) for x in (self.q, self.k, self.v)), self.positions, xqattn.rope_params(D, 1e4),
                                rows4(torch, self.turned[n], wl.F32), self.kv[n], q_weight=self.w, k_weight=self.w)
            xqattn.fa_tree(rows4(torch, self.turned[n], wl.F32), self.kv[n], dst4(torch, self.out[n], wl.F32), D**-0.5, parents=self.parents,
                           workspace=self.w1)

    def accept(self):
        xqattn.kv_pages_compact([p for x in self.kv for p in (x.k, x.v)], self.table, self.rows, self.path, self.n_path, self.new_rows)
        self.rows.copy_(self.new_rows)

    def state(self):
        return [x.cpu().numpy() for x in (self.table, self.rows, self.refs, self.got, *self.out, *(p.t for y in self.kv for p in (y.k, y.v)))]


@pytest.mark.parametrize("kt", list(TYPES))
def test_steps_one_after_another(torch_gpu, kt):
    torch = torch_gpu
    eager, captured = Server(torch, kt, 3), Server(torch, kt, 3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.attend()
        captured.accept()
    held = np.array(HELD)
    for step in range(4):
        case_note(f"step {step} {kt} rows {held}")
        for s in (eager, captured):
            s.inputs(step)
        eager.attend()
        torch.cuda.synchronize()
        assert np.array_equal(eager.rows.cpu().numpy(), held) and np.all(eager.got.cpu().numpy() >= held + T)
        for n, c in enumerate(eager.caches):
            c.table, c.rows = eager.table.cpu().numpy(), held.astype(np.int32)
            c.k, c.v = eager.kv[n].k.t.cpu().numpy(), eager.kv[n].v.t.cpu().numpy()
            check(eager.out[n].cpu().numpy(), None, tree_f64(eager.turned[n].cpu().numpy(), c, eager.host_parents, [T] * B, D**-0.5, False))
        path, n_path = eager.path.cpu().numpy(), eager.n_path.cpu().numpy()
        kept = [[c.values(x, b, int(held[b]) + T)[np.r_[:held[b], held[b] + path[b, :n_path[b]]]] for b in range(B)]
                for c in eager.caches for x in (c.k, c.v)]
        eager.accept()
        torch.cuda.synchronize()
        held = held + n_path
        planes = [p.t.cpu().numpy() for x in eager.kv for p in (x.k, x.v)]
        for x, (plane, rows) in enumerate(zip(planes, kept)):
            for b in range(B):  # the next step starts from the accepted rows
                assert np.array_equal(eager.caches[x // 2].values(plane, b, int(held[b])), rows[b])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), captured.state()):
            assert np.array_equal(a, b), step
    assert np.array_equal(eager.rows.cpu().numpy(), held) and np.all(held > np.array(HELD) + 3)
