"""Attention of a chunk of new tokens over the paged cache, against float64 (chunk_cases.chunk_f64)."""
import numpy as np
import pytest

import oracle
import xqattn
from chunk_cases import Params, chunk_f64
from conftest import case_note
from paged_cases import Cache, bf16
from test_gpu_fa_tree import TYPES, check, dst4, on_gpu as tree_on_gpu, rows4
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu


def i32(torch, x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def on_gpu(torch, q, cache, par, n_tok, narrow, first=None, prefix=None, dev=None, lse=True, fill=7.0, stream=None):
    B, T, H, D = q.shape
    dt, typ = (torch.bfloat16, wl.BF16) if narrow else (torch.float32, wl.F32)
    tq = torch.from_numpy(q).cuda().to(dt)
    out = torch.full((B, T, H, D), fill, dtype=dt, device="cuda")
    tl = torch.full((B, T, H), fill, device="cuda") if lse else None
    dev = dev or cache.device(torch)
    masks = [i32(torch, x) for x in (first, prefix, n_tok)]
    torch.cuda.synchronize()
    xqattn.fa_chunk(rows4(torch, tq, typ), dev, dst4(torch, out, typ), par.struct(), *masks, lse=tl, stream=stream)
    torch.cuda.synchronize()
    return out.float().cpu().numpy(), None if tl is None else tl.cpu().numpy()


def setup(seed, kt, D, H, Hkv, P, rows, T, n_tok=None, narrow=False, **more):
    rng = np.random.default_rng(seed)
    n_tok = [T] * len(rows) if n_tok is None else n_tok
    c = Cache(rng, kt, D, Hkv, P, rows, n_tok, **more)
    q = rng.standard_normal((len(rows), T, H, D)).astype(np.float32)
    return rng, c, bf16(q) if narrow else q, n_tok


SHAPES = [
    # D, H, Hkv, page rows, rows of each sequence, T, tokens of each sequence
    (128, 2, 2, 16, [0], 1, None),                       # one token, nothing cached
    (256, 24, 4, 16, [500], 17, None),
    (128, 16, 8, 16, [0, 1, 15, 63, 64], 3, [3, 1, 2, 3, 0]),
    (128, 32, 8, 48, [63, 64, 65], 70, [70, 1, 69]),
    (256, 24, 4, 5, [31, 130], 40, [40, 9]),             # pages that end inside every tile
    (128, 8, 1, 64, [300], 129, None),
    (128, 32, 1, 1, [70], 2, None),                      # group 32, one row per page
    (128, 16, 8, 32, [0, 700], 260, [260, 131]),
    (256, 4, 4, 100, [257], 130, None),
    (128, 12, 4, 32, [1300], 7, None),                   # a group that does not divide a tile
]


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[0]}h{s[1]}kv{s[2]}p{s[3]}t{s[5]}")
def test_chunk(torch_gpu, shape, kind, narrow):
    D, H, Hkv, P, rows, T, n_tok = shape
    case_note(f"fa_chunk {kind} narrow={narrow} {shape}")
    rng, c, q, n_tok = setup(11 + T, TYPES[kind], D, H, Hkv, P, rows, T, n_tok, narrow, head_major=T % 2 == 1, pad=2 * (T % 3))
    par = Params(D**-0.5)
    check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow), chunk_f64(q, c, n_tok, par, narrow))


MASKS = [
    # window, cap, bias, documents, prefix
    (1, 0.0, 0.0, False, False),                         # a token sees itself alone
    (50, 0.0, 0.0, False, False),
    (64, 30.0, 0.0, False, False),
    (0, 1.5, 8.0, False, False),
    (0, 0.0, 0.0, True, False),
    (0, 50.0, 0.0, False, True),
    (100, 2.0, 8.0, True, True),
]


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind,D,H,Hkv", [("f16", 128, 16, 4), ("q8_0", 256, 24, 4), ("q4_0", 128, 6, 2), ("e5m2", 256, 4, 4)])
@pytest.mark.parametrize("mask", MASKS, ids=lambda m: "w%d_cap%g_bias%g%s%s" % (m[0], m[1], m[2], "_docs" * m[3], "_prefix" * m[4]))
def test_masks_caps_and_biases(torch_gpu, mask, kind, D, H, Hkv, narrow):
    window, cap, bias, docs, pre = mask
    case_note(f"fa_chunk masks {mask} {kind} {D} {H}/{Hkv} narrow={narrow}")
    T, rows, n_tok = 90, [0, 100, 333], [90, 77, 5]
    rng, c, q, n_tok = setup(5, TYPES[kind], D, H, Hkv, 16, rows, T, n_tok, narrow)
    # documents: rising first rows, and tokens that see nothing (a first row behind their own)
    first = None
    if docs:
        first = np.stack([np.sort(rng.integers(-3, r + T, T)) for r in rows])
        first[:, ::7] = 1 << 20
        first[:, 3] = 0
    prefix = [40, 150, 1 << 30] if pre else None
    par = Params(D**-0.5, window, cap, bias)
    check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow, first, prefix), chunk_f64(q, c, n_tok, par, narrow, first, prefix))


def test_negative_zero_and_extreme_scales(torch_gpu):
    for scale in (0.0, -0.1, 2.0**-130, 3.0):
        case_note(f"fa_chunk scale {scale}")
        rng, c, q, n_tok = setup(3, wl.F16, 128, 8, 4, 16, [70], 20)
        par = Params(scale)
        check(*on_gpu(torch_gpu, q, c, par, n_tok, False), chunk_f64(q, c, n_tok, par, False))


def test_bad_pages_are_not_seen(torch_gpu):
    rng, c, q, n_tok = setup(8, wl.Q8_0, 128, 8, 4, 16, [200, 90], 30)
    c.table[0, 2], c.table[0, 5], c.table[1, 0] = -1, c.n_pages, 1 << 30
    case_note("fa_chunk bad pages")
    par = Params(0.1)
    check(*on_gpu(torch_gpu, q, c, par, n_tok, False), chunk_f64(q, c, n_tok, par, False))


def test_rows_past_the_table_are_not_seen(torch_gpu):
    """rows and tokens beyond the table's columns, and counts below 0 and above n_q."""
    rng, c, q, n_tok = setup(9, wl.F16, 128, 8, 4, 16, [56, 0], 8, cols=4)
    c.rows[:] = [60, -5]
    case_note("fa_chunk rows past the table")
    par = Params(0.1)
    got, lse = on_gpu(torch_gpu, q, c, par, [100, -3], False)
    c.rows[:] = [60, 0]
    check(got, lse, chunk_f64(q, c, [8, 0], par, False))


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_what_is_not_seen_has_no_part(torch_gpu, kind, narrow):
    """NaN and Inf in rows that some tokens see and others do not: exactly those that see them get them."""
    kt, D, T, r = TYPES[kind], 128, 70, 30
    rng, c, q, n_tok = setup(4, kt, D, 4, 2, 16, [r], T, None, narrow)
    vals = c.values(c.v, 0, r + T)
    bad = [3, 35, 50, 99]
    for i, row in enumerate(bad):
        p, x = c.place(0, row)
        rec = c.view(c.v)[p, x, i % 2]
        if kt == wl.F16:
            rec[10:12] = np.array([0x7c00, 0x7e00, 0xfc00, 0x7c00][i], np.uint16).reshape(1).view(np.uint8)
        elif kt == wl.E5M2:
            rec[5] = [0x7c, 0x7e, 0xfc, 0x7c][i]
        else:
            rec[0:2] = np.array([0x7c00, 0x7e00, 0xfc00, 0x7c00][i], np.uint16).reshape(1).view(np.uint8)
    window = 20
    case_note(f"fa_chunk non-finite {kind} narrow={narrow}")
    par = Params(D**-0.5, window)
    got, lse = on_gpu(torch_gpu, q, c, par, n_tok, narrow)
    out, wl_, tol, tol_lse = chunk_f64(q, c, n_tok, par, narrow)
    hit = ~np.isfinite(out[0])
    assert hit.any() and not hit.all()
    assert np.array_equal(np.isfinite(got[0]), ~hit), "non-finite values reach other tokens, heads or elements"
    assert np.all(np.abs(got[0] - out[0])[~hit] <= tol[0][~hit])
    assert np.all(np.abs(lse - wl_) <= tol_lse)


def test_one_token_and_chain_equal_the_tree(torch_gpu):
    """Without masks a chunk is the tree operator's chain."""
    for T in (1, 5, 64):
        case_note(f"fa_chunk against fa_tree, {T} tokens")
        rng, c, q, n_tok = setup(T, wl.F16, 128, 16, 8, 16, [333, 20], T)
        a, la = on_gpu(torch_gpu, q, c, Params(0.09), n_tok, False)
        b, lb = tree_on_gpu(torch_gpu, q, c, None, n_tok, 0.09, False)
        _, _, tol, tol_lse = chunk_f64(q, c, n_tok, Params(0.09), False)
        assert np.all(np.abs(a - b) <= 2 * tol) and np.all(np.abs(la - lb) <= 2 * tol_lse)


def test_a_chunk_in_pieces_is_the_chunk(torch_gpu):
    """Tokens of a prompt given in pieces, rows moved up, see the same rows."""
    torch = torch_gpu
    rng, c, q, n_tok = setup(2, wl.Q8_0, 256, 8, 4, 16, [10], 300, None, True)
    par = Params(256**-0.5, 77)
    case_note("fa_chunk in pieces")
    want = chunk_f64(q, c, n_tok, par, True)
    at = 0
    for n in (1, 128, 64, 107):
        c.rows[:] = [10 + at]
        got, lse = on_gpu(torch, np.ascontiguousarray(q[:, at:at + n]), c, par, [n], True)
        check(got, lse, [x[:, at:at + n] for x in want])
        at += n


def test_strided_rows_other_stream_and_padding(torch_gpu):
    """q inside a fused projection, dst inside a wider one, on a stream of its own; what lies beside stays."""
    torch = torch_gpu
    rng, c, q, n_tok = setup(21, wl.F16, 128, 8, 4, 16, [100, 5], 37, [37, 20], True)
    B, T, H, D = q.shape
    wide = torch.full((B, T, 3 * H * D), 3.0, dtype=torch.bfloat16, device="cuda")
    tq = wide[..., H * D:2 * H * D].unflatten(-1, (H, D))
    tq.copy_(torch.from_numpy(q))
    out = torch.full((B, T, H, D + 8), 5.0, dtype=torch.bfloat16, device="cuda")
    dev = c.device(torch)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    case_note("fa_chunk strided, other stream")
    par = Params(D**-0.5)
    lse = torch.full((B, T, H), 7.0, device="cuda")
    xqattn.fa_chunk(rows4(torch, tq, wl.BF16), dev, dst4(torch, out[..., :D], wl.BF16), par.struct(), n_tok=i32(torch, n_tok), lse=lse, stream=stream)
    torch.cuda.synchronize()
    got = out.float().cpu().numpy()
    assert np.all(got[..., D:] == 5.0) and torch.all(wide[..., :H * D] == 3.0) and torch.all(wide[..., 2 * H * D:] == 3.0)
    want = chunk_f64(q, c, n_tok, par, True)
    live = ~np.isnan(want[1][..., 0])
    assert np.all(got[~live] == 5.0) and np.all(lse.cpu().numpy()[~live] == 7.0)
    assert np.all(np.abs(got[live][..., :D] - want[0][live]) <= want[2][live])


def test_replays_follow_rows_and_tokens(torch_gpu):
    """A captured call, replayed with other rows, token counts and pages, gives the eager call's bits."""
    torch = torch_gpu
    rng, c, q, n_tok = setup(31, wl.E5M2, 128, 16, 4, 16, [400, 90], 50, None, False, cols=40, spare=60)
    dev = c.device(torch)
    dev.table.copy_(torch.from_numpy(rng.permutation(c.n_pages)[:80].reshape(2, 40).astype(np.int32)))
    B, T, H, D = q.shape
    tq, out = torch.from_numpy(q).cuda(), torch.zeros((B, T, H, D), device="cuda")
    lse, tn = torch.zeros((B, T, H), device="cuda"), i32(torch, [50, 50])
    first = torch.zeros((B, T), dtype=torch.int32, device="cuda")
    par = Params(D**-0.5, cap=20.0).struct()
    args = (rows4(torch, tq, wl.F32), dev, dst4(torch, out, wl.F32), par)
    case_note("fa_chunk capture")
    ws = xqattn.fa_chunk(*args, first=first, n_tok=tn, lse=lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xqattn.fa_chunk(*args, first=first, n_tok=tn, lse=lse, workspace=ws)
    for rows, toks, f in (([400, 90], [50, 50], 0), ([3, 560], [1, 49], 0), ([0, 0], [50, 0], 20), ([200, 590], [50, 50], 150)):
        dev.rows.copy_(torch.tensor(rows, dtype=torch.int32)), tn.copy_(torch.tensor(toks, dtype=torch.int32))
        first.fill_(f)
        out.fill_(9.0), lse.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got, gl = out.clone(), lse.clone()
        out.fill_(9.0), lse.fill_(9.0)
        xqattn.fa_chunk(*args, first=first, n_tok=tn, lse=lse, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(gl, lse)


def test_long_cache_offsets_past_32_bits(torch_gpu):
    """Pools of more than 2^32 bytes: the last pages' rows are the ones that are read."""
    torch = torch_gpu
    D, Hkv, P, n_pages = 256, 4, 64, 34000  # 64 * 4 * 512 bytes a page: 4.46e9
    k, v = (torch.zeros((n_pages, P, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ids = [33999, 5, 33000]
    g = torch.Generator("cuda").manual_seed(1)
    for p in ids:
        k[p], v[p] = (torch.randn((P, Hkv, D), generator=g, device="cuda").half() for _ in range(2))
    cache = xqattn.KvPages(xqattn.pool_tensor(k, wl.F16, D, P, Hkv, n_pages), xqattn.pool_tensor(v, wl.F16, D, P, Hkv, n_pages),
                           i32(torch, [ids]), i32(torch, [150]))
    q = torch.randn((1, 9, 8, D), generator=g, device="cuda")
    out = torch.zeros_like(q)
    case_note("fa_chunk long cache")
    xqattn.fa_chunk(rows4(torch, q, wl.F32), cache, dst4(torch, out, wl.F32), xqattn.chunk_params(D**-0.5))
    torch.cuda.synchronize()
    kk, vv = (x[ids].reshape(-1, Hkv, D)[:159].double().cpu() for x in (k, v))
    s = torch.stack([q[0, :, h].double().cpu() @ kk[:, h // 2].T for h in range(8)]) * D**-0.5
    s.masked_fill_(torch.arange(159) > 150 + torch.arange(9)[:, None], -float("inf"))
    want = torch.stack([torch.softmax(s[h], -1) @ vv[:, h // 2] for h in range(8)], 1)
    # (159 rows' sums of 2^-24 each, scores of 256 products at 2^-24 of up to 16, operands of 22 bits)
    assert (out[0].double().cpu() - want).abs().max() <= 2.0**-14 * vv.abs().max()
