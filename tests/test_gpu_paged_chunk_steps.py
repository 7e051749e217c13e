"""A server's loop through all of the paged operators: a chunk of a prompt read and its rows' weights taken, the cache
cut to its budget, then drafted tokens attended, verified and accepted; several rounds, eager and replayed from one graph."""
import numpy as np
import pytest

import xqattn
from chunk_cases import Params, chunk_f64, evict, verify, weights_f64
from conftest import case_note
from paged_cases import Cache, random_parents
from test_gpu_fa_tree import dst4, rows4
from test_gpu_verify_tokens import rows3
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

TYPES = {"f16": wl.F16, "q8_0": wl.Q8_0}
B, T, C, H, HKV, D, P, COLS, LAYERS, V, WIDTH = 3, 6, 40, 8, 4, 128, 16, 10, 2, 700, 160
KEEP, SINKS, LAST = 48, 2, 10


class Server:
    def __init__(self, torch, kt, seed):
        self.torch, rng = torch, np.random.default_rng(seed)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        f32 = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        self.caches = [Cache(rng, kt, D, HKV, P, [0] * B, [0] * B, cols=COLS, spare=B * COLS) for _ in range(LAYERS)]
        self.table, self.rows, self.refs = torch.full((B, COLS), -1, dtype=torch.int32, device="cuda"), i32(B), i32(B * COLS)
        self.kv = [xqattn.KvPages(x.k, x.v, self.table, self.rows) for x in (c.device(torch) for c in self.caches)]
        self.want, self.got, self.n_tok, self.new_rows, self.keep = (i32(B) for _ in range(5))
        self.keep.fill_(KEEP)
        self.scores, self.pos, self.cpos, self.tpos = f32(B, WIDTH), i32(B, WIDTH), i32(B, C), i32(B, T)
        self.qc, self.tc, self.oc = ([f32(B, C, H, D) for _ in range(LAYERS)] for _ in range(3))
        self.kc, self.vc = ([f32(B, C, HKV, D) for _ in range(LAYERS)] for _ in range(2))
        self.qt, self.tt, self.ot = ([f32(B, T, H, D) for _ in range(LAYERS)] for _ in range(3))
        self.kt, self.vt = ([f32(B, T, HKV, D) for _ in range(LAYERS)] for _ in range(2))
        self.lse = [f32(B, C, H) for _ in range(LAYERS)]
        self.logits, self.heat, self.u = f32(B, T, V), f32(B), f32(B, T + 1)
        self.parents, self.tokens, self.path, self.n_path, self.next = i32(B, T), i32(B, T), i32(B, T), i32(B), i32(B)
        self.logp = f32(B, T + 1)
        self.par = xqattn.chunk_params(D**-0.5, 0, 30.0)
        chunk = rows4(torch, self.tc[0], wl.F32), self.kv[0], dst4(torch, self.oc[0], wl.F32)
        tree = rows4(torch, self.tt[0], wl.F32), self.kv[0], dst4(torch, self.ot[0], wl.F32)
        # one workspace for all: the calls follow each other on one stream
        self.ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
        need = max(xqattn.fa_chunk_workspace(*chunk), xqattn.kv_weights_workspace(*chunk[:2]), xqattn.fa_tree_workspace(*tree),
                   xqattn.verify_tokens_workspace(rows3(torch, self.logits, wl.F32)))
        if need + 256 > self.ws.numel():
            self.ws = torch.zeros(need + 256, dtype=torch.uint8, device="cuda")

    def put(self, dst, x):
        dst.copy_(self.torch.from_numpy(np.ascontiguousarray(x)))

    def chunk_inputs(self, step):
        rng = np.random.default_rng(900 + step)
        for n in range(LAYERS):
            for dst, h in ((self.qc[n], H), (self.kc[n], HKV), (self.vc[n], HKV)):
                self.put(dst, rng.standard_normal((B, C, h, D)).astype(np.float32))
        n_tok = rng.integers(1, C + 1, B).astype(np.int32)
        n_tok[step % B] = C
        self.put(self.n_tok, n_tok)
        newest = 1000 * step + np.arange(C)
        self.put(self.cpos, np.tile(newest, (B, 1)).astype(np.int32))
        held, pos = self.rows.cpu().numpy(), self.pos.cpu().numpy()
        for b in range(B):
            pos[b, held[b]:held[b] + n_tok[b]] = newest[:n_tok[b]]
        self.put(self.pos, pos)
        return n_tok

    def read(self):
        torch = self.torch
        torch.add(self.rows, self.n_tok, out=self.want)
        xqattn.kv_pages_reserve(self.table, self.refs, P, self.want, self.got, workspace=self.ws)
        for n in range(LAYERS):
            xqattn.qk_norm_rope(*(rows4(torch, x[n], wl.F32) for x in (self.qc, self.kc, self.vc)), self.cpos, xqattn.rope_params(D, 1e4),
                                rows4(torch, self.tc[n], wl.F32), self.kv[n], n_tok=self.n_tok)
            q = rows4(torch, self.tc[n], wl.F32)
            xqattn.fa_chunk(q, self.kv[n], dst4(torch, self.oc[n], wl.F32), self.par, n_tok=self.n_tok, lse=self.lse[n], workspace=self.ws)
            xqattn.kv_weights(q, self.kv[n], self.par, self.lse[n], self.scores, self.scores, n_tok=self.n_tok,
                              decay=0.9 if n == 0 else 1.0, fresh=n == 0, workspace=self.ws)
        self.rows.copy_(self.want)

    def cut(self):
        xqattn.kv_pages_evict([p for x in self.kv for p in (x.k, x.v)], self.table, self.rows, self.refs, self.keep, self.scores, self.new_rows,
                              SINKS, LAST, self.pos, self.scores, self.pos, workspace=self.ws)
        self.rows.copy_(self.new_rows)

    def draft_inputs(self, step):
        rng = np.random.default_rng(700 + step)
        for n in range(LAYERS):
            for dst, h in ((self.qt[n], H), (self.kt[n], HKV), (self.vt[n], HKV)):
                self.put(dst, rng.standard_normal((B, T, h, D)).astype(np.float32))
        parents = np.stack([random_parents(rng, T) for _ in range(B)])
        parents[:, 1:] = np.maximum(parents[:, 1:], 0)
        logits = (rng.standard_normal((B, T, V)) * 3).astype(np.float32)
        tokens = rng.integers(0, V, (B, T)).astype(np.int32)
        for b in range(B):
            for c in range(1, T):
                tokens[b, c] = np.argsort(-logits[b, parents[b, c]], kind="stable")[(parents[b, :c] == parents[b, c]).sum()]
        for dst, x in ((self.parents, parents), (self.logits, logits), (self.tokens, tokens), (self.u, rng.random((B, T + 1)).astype(np.float32)),
                       (self.heat, np.array([0.0, 0.5, 0.9], np.float32)), (self.tpos, np.full((B, T), 1000 * step + C, np.int32))):
            self.put(dst, x)
        return parents, logits, tokens

    def speculate(self):
        torch = self.torch
        torch.add(self.rows, T, out=self.want)
        xqattn.kv_pages_reserve(self.table, self.refs, P, self.want, self.got, workspace=self.ws)
        for n in range(LAYERS):
            xqattn.qk_norm_rope(*(rows4(torch, x[n], wl.F32) for x in (self.qt, self.kt, self.vt)), self.tpos, xqattn.rope_params(D, 1e4),
                                rows4(torch, self.tt[n], wl.F32), self.kv[n])
            xqattn.fa_tree(rows4(torch, self.tt[n], wl.F32), self.kv[n], dst4(torch, self.ot[n], wl.F32), D**-0.5, parents=self.parents,
                           workspace=self.ws)
        xqattn.verify_tokens(rows3(torch, self.logits, wl.F32), self.tokens, self.path, self.n_path, self.next, self.u, None, self.parents,
                             None, self.heat, self.logp, workspace=self.ws)
        xqattn.kv_pages_compact([p for x in self.kv for p in (x.k, x.v)], self.table, self.rows, self.path, self.n_path, self.new_rows)
        self.rows.copy_(self.new_rows)

    def host(self, n, rows):
        c = self.caches[n]
        c.table, c.rows = self.table.cpu().numpy(), np.array(rows, np.int32)
        c.k, c.v = self.kv[n].k.t.cpu().numpy(), self.kv[n].v.t.cpu().numpy()
        return c

    def state(self):
        return [x.cpu().numpy() for x in (self.table, self.rows, self.refs, self.got, self.scores, self.pos, self.path, self.n_path, self.next, self.logp,
                                          *self.oc, *self.lse, *self.ot, *(p.t for y in self.kv for p in (y.k, y.v)))]


@pytest.mark.parametrize("kt", list(TYPES))
def test_rounds_one_after_another(torch_gpu, kt):
    torch = torch_gpu
    eager, captured = Server(torch, TYPES[kt], 4), Server(torch, TYPES[kt], 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.read()
        captured.cut()
        captured.speculate()
    par, cuts, stood = Params(D**-0.5, 0, 30.0), 0, 0
    for step in range(5):
        held = eager.rows.cpu().numpy()
        case_note(f"round {step} {kt} rows {held}")
        n_tok = [s.chunk_inputs(step) for s in (eager, captured)][0]
        parents, logits, tokens = [s.draft_inputs(step) for s in (eager, captured)][0]
        before = eager.scores.cpu().numpy()
        eager.read()
        torch.cuda.synchronize()
        expect, tol = None, 0.0
        for n in range(LAYERS):
            c, q = eager.host(n, held), eager.tc[n].cpu().numpy()
            out, lse, t_out, t_lse = chunk_f64(q, c, n_tok, par, False)
            live = ~np.isnan(lse[..., 0])
            assert np.all(np.abs(eager.oc[n].cpu().numpy()[live] - out[live]) <= t_out[live])
            got = eager.lse[n].cpu().numpy()
            assert np.all(np.abs(got[live] - lse[live]) <= t_lse[live])
            w, t = weights_f64(q, c, n_tok, par, got, before if expect is None else expect, WIDTH, 0.9 if n == 0 else 1.0, n == 0)
            expect, tol = np.where(np.isnan(w), before, w).astype(np.float32), tol + t + np.abs(np.nan_to_num(w)) * 2.0**-23
        scores = eager.scores.cpu().numpy()
        assert np.all(np.abs(scores - expect) <= tol)
        held = held + n_tok
        planes = [(eager.host(n, held).k.copy(), eager.host(n, held).v.copy()) for n in range(LAYERS)]
        kept_rows = [[c.values(x, b, int(held[b])) for b in range(B)] for n, c in enumerate(eager.caches) for x in planes[n]]
        table, refs, rows, moves, order = evict(eager.table.cpu().numpy(), held, eager.refs.cpu().numpy(), [KEEP] * B, SINKS, LAST, scores,
                                                eager.pos.cpu().numpy(), P, B * COLS)
        eager.cut()
        torch.cuda.synchronize()
        cuts += len(moves)
        assert np.array_equal(eager.table.cpu().numpy(), table) and np.array_equal(eager.refs.cpu().numpy(), refs)
        assert np.array_equal(eager.rows.cpu().numpy(), rows)
        for n, c in enumerate(eager.host(n, rows) for n in range(LAYERS)):
            for x, plane in enumerate((c.k, c.v)):
                for b in range(B):
                    assert np.array_equal(c.values(plane, b, int(rows[b])), kept_rows[2 * n + x][b][order[b]])
        eager.speculate()
        torch.cuda.synchronize()
        path, n_path, nxt, _ = verify(logits, tokens, parents, [T] * B, eager.heat.cpu().numpy(), eager.u.cpu().numpy())
        assert np.array_equal(eager.path.cpu().numpy(), path) and np.array_equal(eager.n_path.cpu().numpy(), n_path)
        assert np.array_equal(eager.next.cpu().numpy(), nxt) and np.array_equal(eager.rows.cpu().numpy(), rows + n_path)
        stood += int((n_path - 1).sum())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), captured.state()):
            assert np.array_equal(a, b, equal_nan=True), step
        for s in (eager, captured):  # the accepted tokens' rows start without weight, at the step's position
            sc, pos = s.scores.cpu().numpy(), s.pos.cpu().numpy()
            for b in range(B):
                sc[b, rows[b]:rows[b] + n_path[b]], pos[b, rows[b]:rows[b] + n_path[b]] = 0.0, 1000 * step + C
            s.put(s.scores, sc), s.put(s.pos, pos)
    assert cuts and stood
