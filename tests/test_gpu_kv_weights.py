"""Accumulated attention weights of cached rows, against float64 (chunk_cases.weights_f64)."""
import numpy as np
import pytest

import xqattn
from chunk_cases import Params, chunk_f64, weights_f64
from conftest import case_note
from test_gpu_fa_chunk import i32, setup
from test_gpu_fa_tree import TYPES, dst4, rows4
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu


def on_gpu(torch, q, cache, par, n_tok, narrow, lse, scores, cols, decay=1.0, fresh=True, first=None, prefix=None, inplace=False, stream=None):
    dt, typ = (torch.bfloat16, wl.BF16) if narrow else (torch.float32, wl.F32)
    tq, tl = torch.from_numpy(q).cuda().to(dt), torch.from_numpy(lse.astype(np.float32)).cuda()
    ts = None if scores is None else torch.from_numpy(scores).cuda()
    out = ts if inplace else torch.full((q.shape[0], cols), -7.0, device="cuda")
    masks = [i32(torch, x) for x in (first, prefix, n_tok)]
    torch.cuda.synchronize()
    xqattn.kv_weights(rows4(torch, tq, typ), cache.device(torch), par.struct(), tl, ts, out, *masks, decay=decay, fresh=fresh, stream=stream)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check(got, want, untouched=-7.0):
    out, tol = want
    live = ~np.isnan(out)
    assert np.all(got[~live] == untouched), "columns behind the rows were written"
    err = np.abs(got[live] - out[live])
    assert np.all(err <= tol[live]), f"off by {err.max():.3e}, allowed {tol[live][err > tol[live]].min():.3e}"


def lse_of(q, c, n_tok, par, narrow, first=None, prefix=None):
    """What the chunk operator gives, to f32."""
    return np.nan_to_num(chunk_f64(q, c, n_tok, par, narrow, first, prefix)[1], nan=0.0).astype(np.float32)


SHAPES = [
    # D, H, Hkv, page rows, rows, T, tokens
    (128, 2, 2, 16, [0], 1, None),
    (256, 24, 4, 16, [377], 1, None),
    (128, 16, 8, 16, [0, 1, 127, 128, 129], 3, [3, 1, 2, 3, 0]),
    (128, 32, 8, 48, [260, 5], 33, None),
    (256, 24, 4, 5, [31, 130], 20, [20, 9]),
    (128, 32, 1, 1, [70], 2, None),
    (128, 8, 2, 64, [1000], 150, None),
]


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[0]}h{s[1]}kv{s[2]}p{s[3]}t{s[5]}")
def test_weights(torch_gpu, shape, kind, narrow):
    D, H, Hkv, P, rows, T, n_tok = shape
    case_note(f"kv_weights {kind} narrow={narrow} {shape}")
    rng, c, q, n_tok = setup(50 + T, TYPES[kind], D, H, Hkv, P, rows, T, n_tok, narrow, head_major=T % 2 == 0, pad=2 * (T % 3))
    par = Params(D**-0.5)
    lse = lse_of(q, c, n_tok, par, narrow)
    cols = max(r + t for r, t in zip(rows, n_tok)) + 3
    scores = rng.random((len(rows), cols)).astype(np.float32)
    want = weights_f64(q, c, n_tok, par, lse, scores, cols, 0.75, True)
    check(on_gpu(torch_gpu, q, c, par, n_tok, narrow, lse, scores, cols, 0.75), want)


@pytest.mark.parametrize("kind,D,H,Hkv", [("f16", 128, 16, 4), ("q8_0", 256, 24, 4), ("q4_0", 128, 6, 2), ("e5m2", 256, 4, 4)])
@pytest.mark.parametrize("window,cap,bias,docs,pre", [(1, 0.0, 0.0, False, False), (64, 30.0, 0.0, False, True), (0, 1.5, 8.0, True, False)])
def test_masks_caps_and_biases(torch_gpu, kind, D, H, Hkv, window, cap, bias, docs, pre):
    case_note(f"kv_weights masks {kind} {window} {cap} {bias} {docs} {pre}")
    T, rows, n_tok = 40, [0, 100, 333], [40, 37, 5]
    rng, c, q, n_tok = setup(6, TYPES[kind], D, H, Hkv, 16, rows, T, n_tok)
    first = None
    if docs:
        first = np.stack([np.sort(rng.integers(-3, r + T, T)) for r in rows])
        first[:, ::7] = 1 << 20
    prefix = [30, 120, 1 << 30] if pre else None
    par = Params(D**-0.5, window, cap, bias)
    lse = lse_of(q, c, n_tok, par, False, first, prefix)
    assert not docs or np.isneginf(lse).any()
    cols = max(rows) + T
    want = weights_f64(q, c, n_tok, par, lse, None, cols, 1.0, True, first, prefix)
    check(on_gpu(torch_gpu, q, c, par, n_tok, False, lse, None, cols, 1.0, True, first, prefix), want)


def test_layers_add_up_in_place_and_columns_end_early(torch_gpu):
    """The first layer decays and starts the new rows, the others add; fewer columns than rows."""
    rng, c, q, n_tok = setup(7, wl.F16, 128, 8, 2, 16, [90, 40], 6)
    par = Params(0.1)
    lse = lse_of(q, c, n_tok, par, False)
    cols = 93
    scores = rng.random((2, cols)).astype(np.float32)
    case_note("kv_weights layers in place")
    a = on_gpu(torch_gpu, q, c, par, n_tok, False, lse, scores, cols, 0.5, True, inplace=True)
    w1, t1 = weights_f64(q, c, n_tok, par, lse, scores, cols, 0.5, True)
    live = ~np.isnan(w1)
    assert np.all(np.abs(a - w1)[live] <= t1[live]) and np.array_equal(a[~live], scores[~live])
    b = on_gpu(torch_gpu, q, c, par, n_tok, False, lse, a.copy(), cols, 1.0, False, inplace=True)
    w2, t2 = weights_f64(q, c, n_tok, par, lse, a, cols, 1.0, False)
    assert np.all(np.abs(b - w2)[live] <= t2[live]) and np.array_equal(b[~live], scores[~live])


def test_weights_of_a_token_are_one_and_nan_stays_where_it_is_seen(torch_gpu):
    """Without bad values a row's weights sum to heads x tokens; a NaN key reaches exactly its row."""
    rng, c, q, n_tok = setup(9, wl.F16, 128, 8, 4, 16, [200], 10)
    par = Params(0.1, 60)
    lse = lse_of(q, c, n_tok, par, False)
    case_note("kv_weights sums, NaN")
    got = on_gpu(torch_gpu, q, c, par, n_tok, False, lse, None, 210)
    assert abs(got.sum() - 8 * 10) <= 80 * 2.0**-14
    assert np.all(got[0, :141] == 0.0)  # (token 0 sees 141.., the window's rows)
    for row in (100, 205):
        p, x = c.place(0, row)
        c.view(c.k)[p, x, 1][6:8] = np.array([0x7e00], np.uint16).view(np.uint8)
    bad = on_gpu(torch_gpu, q, c, par, n_tok, False, lse, None, 210)
    keep = np.arange(210) != 205
    assert np.isnan(bad[0, 205]) and np.array_equal(bad[0, keep], got[0, keep])


def test_last_tokens_alone(torch_gpu):
    """A view of a chunk's last tokens with rows moved up gives what these alone give."""
    torch = torch_gpu
    rng, c, q, n_tok = setup(10, wl.Q8_0, 256, 24, 4, 16, [300], 50, None, True)
    par = Params(256**-0.5)
    lse = lse_of(q, c, n_tok, par, True)
    c.rows[:] = [300 + 34]
    tail = np.ascontiguousarray(q[:, 34:])
    case_note("kv_weights last tokens")
    want = weights_f64(tail, c, [16], par, lse[:, 34:], None, 350, 1.0, True)
    tq = torch.from_numpy(q).cuda().bfloat16()[:, 34:]
    out = torch.full((1, 350), -7.0, device="cuda")
    xqattn.kv_weights(rows4(torch, tq, wl.BF16), c.device(torch), par.struct(), torch.from_numpy(lse[:, 34:].copy()).cuda(), None, out)
    torch.cuda.synchronize()
    check(out.cpu().numpy(), want)


def test_replays_and_streams(torch_gpu):
    torch = torch_gpu
    rng, c, q, n_tok = setup(32, wl.Q4_0, 128, 16, 4, 16, [400, 90], 20, None, False, cols=40, spare=60)
    dev = c.device(torch)
    dev.table.copy_(torch.from_numpy(rng.permutation(c.n_pages)[:80].reshape(2, 40).astype(np.int32)))
    tq, lse = torch.from_numpy(q).cuda(), torch.full((2, 20, 16), 3.0, device="cuda")
    tn, scores, out = i32(torch, [20, 20]), torch.rand((2, 640), device="cuda"), torch.zeros((2, 640), device="cuda")
    args = (rows4(torch, tq, wl.F32), dev, Params(0.1).struct(), lse, scores, out)
    case_note("kv_weights capture")
    ws = xqattn.kv_weights(*args, n_tok=tn, decay=0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xqattn.kv_weights(*args, n_tok=tn, decay=0.5, workspace=ws)
    side = torch.cuda.Stream()
    for rows, toks in (([400, 90], [20, 20]), ([3, 560], [1, 19]), ([0, 0], [20, 0])):
        dev.rows.copy_(torch.tensor(rows, dtype=torch.int32)), tn.copy_(torch.tensor(toks, dtype=torch.int32))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(9.0)
        torch.cuda.synchronize()
        xqattn.kv_weights(*args, n_tok=tn, decay=0.5, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got, out)
