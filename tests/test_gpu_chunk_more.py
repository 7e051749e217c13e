"""Calls of the paged chunk operators beside the ordinary ones: few tokens under masks, more sequences than a wave
has lanes, two calls at one time, graphs that share a workspace."""
import numpy as np
import pytest

import xqattn
from chunk_cases import Params, chunk_f64, weights_f64
from conftest import case_note
from test_gpu_fa_chunk import MASKS, on_gpu, setup
from test_gpu_fa_tree import TYPES, check, dst4, rows4
from test_gpu_kv_weights import check as check_weights, lse_of, on_gpu as weights_on_gpu
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu


# 4, 28 and 60 pairs of a KV head (each form for few pairs), dealt over three sequences' rows
@pytest.mark.parametrize("kind,D,H,Hkv,narrow", [("f16", 128, 16, 4, True), ("q8_0", 256, 24, 6, False), ("e5m2", 128, 8, 2, True), ("q4_0", 256, 4, 1, False)])
@pytest.mark.parametrize("T", [1, 7, 15])
@pytest.mark.parametrize("mask", MASKS, ids=lambda m: "w%d_cap%g_bias%g%s%s" % (m[0], m[1], m[2], "_docs" * m[3], "_prefix" * m[4]))
def test_few_tokens_under_masks(torch_gpu, mask, T, kind, D, H, Hkv, narrow):
    window, cap, bias, docs, pre = mask
    case_note(f"few tokens {T} masks {mask} {kind} {D} {H}/{Hkv}")
    rows, n_tok = [0, 100, 733], [T, max(T - 2, 0), T]
    rng, c, q, n_tok = setup(50 + T, TYPES[kind], D, H, Hkv, 16, rows, T, n_tok, narrow)
    first = np.stack([np.sort(rng.integers(-3, r + T, T)) for r in rows]) if docs else None
    if docs:
        first[1, :] = 1 << 20  # a whole sequence that sees nothing
    prefix = [40, 50, 1 << 30] if pre else None
    par = Params(D**-0.5, window, cap, bias)
    check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow, first, prefix), chunk_f64(q, c, n_tok, par, narrow, first, prefix))


@pytest.mark.parametrize("T,window", [(1, 0), (2, 70), (9, 0)])
def test_more_sequences_than_lanes(torch_gpu, T, window):
    B = 131
    rng = np.random.default_rng(T)
    rows = rng.integers(0, 40, B)
    rows[[0, 63, 64, 65, 127, 128, 130]] = [900, 0, 700, 64, 63, 1, 500]
    n_tok = rng.integers(0, T + 1, B)
    n_tok[[0, 64, 130]] = T
    case_note(f"{B} sequences T {T} window {window}")
    rng, c, q, n_tok = setup(T, wl.F16, 128, 8, 2, 16, list(rows), T, list(n_tok), True)
    par = Params(128**-0.5, window)
    out, lse = on_gpu(torch_gpu, q, c, par, n_tok, True)
    check(out, lse, chunk_f64(q, c, n_tok, par, True))
    scores = np.abs(rng.standard_normal((B, 1000))).astype(np.float32)
    l = lse_of(q, c, n_tok, par, True)
    got = weights_on_gpu(torch_gpu, q, c, par, n_tok, True, l, scores, 1000, decay=0.5)
    check_weights(got, weights_f64(q, c, n_tok, par, l, scores, 1000, 0.5, True))


def _call(torch, seed, kind, rows, T, D=128, H=16, Hkv=4):
    """A chunk's buffers and a function that launches it (and its weights) with a workspace."""
    rng, c, q, n_tok = setup(seed, TYPES[kind], D, H, Hkv, 16, rows, T, None, True)
    dev, tq = c.device(torch), torch.from_numpy(q).cuda().to(torch.bfloat16)
    out = torch.zeros(len(rows), T, H, D, dtype=torch.bfloat16, device="cuda")
    lse, scores = torch.zeros(len(rows), T, H, device="cuda"), torch.zeros(len(rows), 1200, device="cuda")
    par = Params(D**-0.5).struct()
    qt, ot = rows4(torch, tq, wl.BF16), dst4(torch, out, wl.BF16)

    def run(ws, stream=None):
        xqattn.fa_chunk(qt, dev, ot, par, lse=lse, workspace=ws, stream=stream)
        xqattn.kv_weights(qt, dev, par, lse, None, scores, workspace=ws, stream=stream)

    need = max(xqattn.fa_chunk_workspace(qt, dev, ot), xqattn.kv_weights_workspace(qt, dev)) + 256
    return run, need, (out, lse, scores), (q, c, n_tok, Params(D**-0.5))


def _results(torch, call):
    torch.cuda.synchronize()
    return [x.float().cpu().numpy() for x in call[2]]


def test_two_calls_at_one_time(torch_gpu):
    torch = torch_gpu
    a, b = _call(torch, 1, "q8_0", [900, 17, 500], 3), _call(torch, 2, "f16", [1000, 3], 40)
    ws = [torch.zeros(x[1], dtype=torch.uint8, device="cuda") for x in (a, b)]
    alone = []
    for x, w in zip((a, b), ws):
        x[0](w)
        alone.append(_results(torch, x))
        for y in x[2]:
            y.zero_()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    case_note("two chunk calls on two streams")
    for _ in range(20):
        for x, w, s in zip((a, b), ws, streams):
            x[0](w, s)
    for x, y in zip((a, b), alone):
        assert all(np.array_equal(p, r) for p, r in zip(_results(torch, x), y))
        q, c, n_tok, par = x[3]
        check(y[0], y[1], chunk_f64(q, c, n_tok, par, True))


def test_graphs_that_share_a_workspace(torch_gpu):
    torch = torch_gpu
    a, b = _call(torch, 3, "e5m2", [700, 1, 64], 2), _call(torch, 4, "q4_0", [300], 33)
    ws = torch.zeros(max(a[1], b[1]), dtype=torch.uint8, device="cuda")
    alone = []
    for x in (a, b):
        x[0](ws)
        alone.append(_results(torch, x))
    graphs = []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x[0](ws)
        graphs.append(g)
    case_note("two graphs, one workspace")
    for order in ((0, 1), (1, 0), (0, 0), (1, 1), (0, 1)):
        for x in (a, b):
            for y in x[2]:
                y.zero_()
        ws.fill_(255)  # what the other call left, and worse, has no part
        for i in order:
            graphs[i].replay()
        for i in set(order):
            got = _results(torch, (a, b)[i])
            assert all(np.array_equal(p, r) for p, r in zip(got, alone[i]))
