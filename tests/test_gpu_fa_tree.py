"""Attention of drafted tokens over the paged cache, against float64 (paged_cases.tree_f64)."""
import numpy as np
import pytest

import oracle
import xqattn
from conftest import case_note
from paged_cases import Cache, bf16, random_parents, tree_f64
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

TYPES = {"f16": wl.F16, "q8_0": wl.Q8_0, "q4_0": wl.Q4_0, "e5m2": wl.E5M2}


def rows4(torch, x, typ):
    """[B, T, H, D] device tensor -> ggml [D, T, H, B] (q) descriptor."""
    es = x.element_size()
    return xqattn.DevTensor(typ, (x.shape[3], x.shape[1], x.shape[2], x.shape[0]), (es, x.stride(1) * es, x.stride(2) * es, x.stride(0) * es), x)


def dst4(torch, x, typ):
    es = x.element_size()
    return xqattn.DevTensor(typ, (x.shape[3], x.shape[2], x.shape[1], x.shape[0]), (es, x.stride(2) * es, x.stride(1) * es, x.stride(0) * es), x)


def on_gpu(torch, q, cache, parents, n_tok, scale, narrow, dev=None, lse=True, fill=7.0, stream=None):
    B, T, H, D = q.shape
    dt, typ = (torch.bfloat16, wl.BF16) if narrow else (torch.float32, wl.F32)
    tq = torch.from_numpy(q).cuda().to(dt)
    out = torch.full((B, T, H, D), fill, dtype=dt, device="cuda")
    tl = torch.full((B, T, H), fill, device="cuda") if lse else None
    dev = dev or cache.device(torch)
    tp = None if parents is None else torch.from_numpy(np.ascontiguousarray(parents)).cuda()
    tn = None if n_tok is None else torch.tensor(list(n_tok), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    xqattn.fa_tree(rows4(torch, tq, typ), dev, dst4(torch, out, typ), scale, parents=tp, n_tok=tn, lse=tl, stream=stream)
    torch.cuda.synchronize()
    return out.float().cpu().numpy(), None if tl is None else tl.cpu().numpy()


def check(got, glse, want, fill=7.0, n_tok=None):
    out, lse, tol, tol_lse = want
    live = ~np.isnan(lse[..., 0])
    assert np.all(got[~live] == fill) and (glse is None or np.all(glse[~live] == fill)), "padding tokens were written"
    err = np.abs(got[live] - out[live])
    bad = ~(err <= tol[live])
    assert not bad.any(), f"{bad.sum()} of {err.size} outside their tolerance (abs {err.max():.3e}, allowed {tol[live][bad].min():.3e})"
    if glse is not None and err.size:
        a, w, t = glse[live], lse[live], tol_lse[live]
        fin = np.isfinite(w)
        assert np.array_equal(a[~fin], w[~fin])
        assert np.all(np.abs(a[fin] - w[fin]) <= t[fin]), f"lse off by {np.max(np.abs(a[fin] - w[fin])):.3e}"


def setup(seed, kt, D, H, Hkv, P, rows, T, n_tok=None, **more):
    rng = np.random.default_rng(seed)
    n_tok = [T] * len(rows) if n_tok is None else n_tok
    c = Cache(rng, kt, D, Hkv, P, rows, n_tok, **more)
    q = rng.standard_normal((len(rows), T, H, D)).astype(np.float32)
    parents = np.stack([random_parents(rng, T) for _ in rows])
    return rng, c, q, parents, n_tok


SHAPES = [
    # D, H, Hkv, page rows, rows of each sequence, T, tokens of each sequence
    (256, 24, 4, 16, [377], 1, None),
    (128, 2, 2, 16, [0], 1, None),                       # nothing cached: the token sees itself
    (128, 16, 8, 16, [0, 1, 15, 16, 17], 3, [3, 1, 2, 3, 0]),
    (128, 32, 8, 48, [63, 64, 65, 200], 8, None),
    (256, 24, 4, 5, [31, 130], 16, [16, 9]),             # pages that end inside every tile
    (128, 8, 1, 64, [300], 25, None),
    (128, 32, 1, 1, [70], 2, None),                      # group 32, one row per page
    (128, 32, 8, 16, [1100, 3, 500], 64, [64, 64, 33]),
    (256, 24, 4, 100, [257, 900], 64, [64, 5]),
    (128, 12, 4, 32, [2050], 7, None),
]


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_fa_tree_shapes(torch_gpu, shape, kt, narrow):
    D, H, Hkv, P, rows, T, n_tok = SHAPES[shape]
    case_note(f"fa_tree {SHAPES[shape]} {kt} narrow {narrow}")
    rng, c, q, parents, n_tok = setup(100 + shape, TYPES[kt], D, H, Hkv, P, rows, T, n_tok, head_major=shape % 3 == 1, pad=(0, 0, 2, 0, 6)[shape % 5] if kt != "e5m2" else shape % 4)
    if narrow:
        q = bf16(q)
    scale = 1.0 / np.sqrt(D)
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, scale, narrow)
    check(got, lse, tree_f64(q, c, parents, n_tok, scale, narrow))


@pytest.mark.parametrize("seed", range(24))
def test_fa_tree_random(torch_gpu, seed):
    rng = np.random.default_rng(seed)
    D = int(rng.choice([128, 256]))
    Hkv = int(rng.choice([1, 2, 4, 8]))
    H = Hkv * int(rng.choice([1, 2, 3, 6, 8]))
    T = int(rng.integers(1, 65))
    B = int(rng.integers(1, 6))
    rows = [int(np.exp(rng.uniform(0, np.log(900)))) - 1 for _ in range(B)]
    n_tok = [int(rng.integers(0, T + 1)) for _ in range(B)]
    kt, narrow = list(TYPES)[seed % 4], bool(seed // 4 % 2)
    case_note(f"fa_tree random {seed}: D {D} H {H}/{Hkv} T {T} rows {rows} n_tok {n_tok} {kt} narrow {narrow}")
    _, c, q, parents, n_tok = setup(seed, TYPES[kt], D, H, Hkv, int(rng.choice([1, 3, 16, 32, 64, 77])), rows, T, n_tok)
    if narrow:
        q = bf16(q)
    scale = float(rng.choice([1.0 / np.sqrt(D), 0.5, 0.02]))
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, scale, narrow)
    check(got, lse, tree_f64(q, c, parents, n_tok, scale, narrow))


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
def test_fa_tree_chain_is_causal(torch_gpu, kt, narrow):
    """No parents: token i sees token i - 1 and all before it."""
    _, c, q, _, n_tok = setup(7, TYPES[kt], 128, 8, 4, 16, [130, 40], 6)
    q = bf16(q)
    got, lse = on_gpu(torch_gpu, q, c, None, None, 0.09, narrow)
    chain = np.tile(np.arange(-1, 5, dtype=np.int32), (2, 1))
    check(got, lse, tree_f64(q, c, chain, n_tok, 0.09, narrow))


def test_fa_tree_parents_out_of_range_count_as_none(torch_gpu):
    _, c, q, parents, n_tok = setup(8, wl.F16, 128, 4, 2, 16, [50], 9)
    bad = parents.copy()
    bad[0] = [-1, 1, 5, -9, 3, 2**31 - 1, -2**31, 6, 8]
    clean = bad.copy()
    clean[0] = [-1, -1, -1, -1, 3, -1, -1, 6, -1]
    got, lse = on_gpu(torch_gpu, q, c, bad, n_tok, 0.1, False)
    check(got, lse, tree_f64(q, c, clean, n_tok, 0.1, False))


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("D,T", [(128, 12), (256, 40)])
def test_fa_tree_unseen_rows_have_no_part(torch_gpu, kt, narrow, D, T):
    """NaN and Inf in rows that a token does not see (other branches, rows past the end, other
    pages) change nothing; in a branch's own rows they reach that branch only."""
    rng, c, q, parents, n_tok = setup(9, TYPES[kt], D, 12, 4, 16, [90, 33], T, [T - 1, T], spare=3)
    q = bf16(q)
    for b in range(2):
        parents[b] = np.arange(-2, T - 2)  # two interleaved chains
        parents[b][:2] = -1
    want = tree_f64(q, c, parents, n_tok, 0.08, narrow)
    junk = np.frombuffer(np.array([np.nan, np.inf, -np.inf], np.float16).tobytes(), np.uint8).reshape(3, 2)
    es = {"f16": 2, "q8_0": 34, "q4_0": 18, "e5m2": 1}[kt]
    live = {(int(c.table[b, r // 16]), r % 16) for b in range(2) for r in range(c.rows[b] + n_tok[b])}
    for buf in (c.k, c.v):
        v = c.view(buf)
        spots = [(p, i) for p in range(c.n_pages) for i in range(16) if (p, i) not in live]  # past the ends, spare pages
        odd = [c.place(b, int(c.rows[b]) + j) for b in range(2) for j in range(1, n_tok[b], 2)]  # the second chain
        for n, (p, i) in enumerate(spots + odd):
            for o in range(0, c.rec, es * 5):
                if es == 1:
                    v[p, i, :, o] = (0x7E, 0x7C, 0xFC)[n % 3]
                else:
                    v[p, i, :, o:o + 2] = junk[n % 3]
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, 0.08, narrow)
    out, wl_, tol, tol_lse = want
    even = np.arange(T) % 2 == 0
    for b in range(2):
        for i in range(n_tok[b]):
            if even[i]:
                assert np.all(np.abs(got[b, i] - out[b, i]) <= tol[b, i]), (b, i)
                assert np.all(np.abs(lse[b, i] - wl_[b, i]) <= tol_lse[b, i])
            else:
                assert not np.isfinite(got[b, i]).all(), "a row that is seen holds NaN or Inf"
    assert np.all(got[0, T - 1] == 7.0)


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
def test_fa_tree_infinite_value_of_one_element(torch_gpu, kt, narrow):
    """An infinite V element (or block scale) of one seen row makes its own dims non-finite and
    leaves the others."""
    _, c, q, parents, n_tok = setup(10, TYPES[kt], 128, 8, 4, 16, [100], 5)
    q = bf16(q)
    want = tree_f64(q, c, parents, n_tok, 0.08, narrow)
    p, i = c.place(0, 37)
    if kt == "e5m2":
        c.view(c.v)[p, i, 2, 40] = 0x7C
        dims = [40]
    else:
        o = {"f16": 80, "q8_0": 34, "q4_0": 18}[kt]
        c.view(c.v)[p, i, 2, o:o + 2] = (0x00, 0x7C)
        dims = [40] if kt == "f16" else list(range(32, 64))
    got, _ = on_gpu(torch_gpu, q, c, parents, n_tok, 0.08, narrow)
    hit = np.zeros((8, 128), bool)
    hit[4:6, dims] = True
    assert not np.isfinite(got[0][:, hit]).any()
    assert np.all(np.abs(got[0] - want[0][0])[:, ~hit] <= want[2][0][:, ~hit])


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kt", ["f16", "q8_0"])
def test_fa_tree_pages_out_of_range_are_not_seen(torch_gpu, kt, narrow):
    """Table entries that name no page, and rows past the table, have no part; a sequence of
    nothing else gives zeros and -inf."""
    _, c, q, parents, n_tok = setup(11, TYPES[kt], 128, 8, 4, 16, [200, 40, 64], 5)
    q = bf16(q)
    c.table[0, 2], c.table[0, 5], c.table[0, 12] = -1, c.n_pages, 2**31 - 1
    c.table[1] = -7
    c.rows[2] = c.cols * 16 + 1000  # the context fills the table; the tokens' rows lie past it
    c.table[2] = c.table[0]
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, 0.1, narrow)
    check(got, lse, tree_f64(q, c, parents, n_tok, 0.1, narrow))
    assert np.all(got[1] == 0.0) and np.all(lse[1] == -np.inf)


def test_fa_tree_negative_rows_are_none(torch_gpu):
    _, c, q, parents, n_tok = setup(12, wl.F16, 128, 4, 2, 16, [20, 30], 3)
    c.rows[1] = -5
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, 0.1, False)
    check(got, lse, tree_f64(q, c, parents, n_tok, 0.1, False))


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("power", [-20, -8, 6, 11])
def test_fa_tree_magnitudes(torch_gpu, kt, narrow, power):
    """K, V and Q far from 1 (powers of two): the scores stay, the outputs scale."""
    rng = np.random.default_rng(13)
    c = Cache(rng, TYPES[kt], 128, 4, 16, [150], [6])
    f = 2.0**power if kt != "e5m2" or power > -9 else 2.0**-8
    if kt in ("f16", "e5m2") and power == -20:
        f = 2.0**-8  # subnormal elements from here on: the decoded values are the operator's input either way
    for name in ("k", "v"):
        x = np.random.default_rng(14).standard_normal((c.n_pages, 16, 4, 128)).astype(np.float32) * np.float32(f)
        raw = oracle.quantize(c.kv_type, x).reshape(c.n_pages, 16, 4, c.rec)
        c.view(getattr(c, name))[...] = raw
    q = bf16(rng.standard_normal((1, 6, 8, 128)).astype(np.float32) / np.float32(f))
    parents = random_parents(rng, 6)[None]
    want = tree_f64(q, c, parents, [6], 0.09, narrow)
    got, lse = on_gpu(torch_gpu, q, c, parents, [6], 0.09, narrow)
    out, wlse, tol, tol_lse = want
    if narrow and kt in ("q8_0", "q4_0"):
        # d * q as one f16: below 2^-14 its step is 2^-24, half of it 2^-25 per value; scores alike
        ds = np.abs(q).sum(-1)[..., None] * 0.09 * 2.0**-25
        tol = tol + 2.0**-25 + np.abs(c.values(c.v, 0, 156)).max() * 2 * ds
        tol_lse = tol_lse + ds[..., 0]
    check(got, lse, (out, wlse, tol, tol_lse))


def test_fa_tree_offsets_past_32_bits(torch_gpu):
    """A pool whose pages lie more than 2^32 bytes apart."""
    torch = torch_gpu
    _, c, q, parents, n_tok = setup(15, wl.Q8_0, 128, 4, 2, 16, [60], 4, spare=0)
    stride = (1 << 31) + 4098
    assert stride * (c.n_pages - 1) > 1 << 32
    dev = c.device(torch)
    for name in ("k", "v"):
        big = torch.zeros(stride * (c.n_pages - 1) + c.page, dtype=torch.uint8, device="cuda")
        small = getattr(dev, name)
        for p in range(c.n_pages):
            big[p * stride:p * stride + c.page] = small.t[p * c.page:(p + 1) * c.page]
        setattr(dev, name, xqattn.DevTensor(c.kv_type, small.ne, (34, c.row, c.head, stride), big))
    got, lse = on_gpu(torch, q, c, parents, n_tok, 0.1, False, dev=dev)
    check(got, lse, tree_f64(q, c, parents, n_tok, 0.1, False))


def test_fa_tree_strided_q_and_dst(torch_gpu):
    """q as a slice of a wider row (an odd element offset), dst with gaps."""
    torch = torch_gpu
    _, c, q, parents, n_tok = setup(16, wl.F16, 128, 8, 4, 16, [77, 5], 5)
    wide = torch.zeros((2, 5, 8, 128 + 3), device="cuda")
    wide[..., 1:129] = torch.from_numpy(q).cuda()
    out = torch.full((2, 5, 8, 160), 7.0, device="cuda")
    tp = torch.from_numpy(parents).cuda()
    xqattn.fa_tree(rows4(torch, wide[..., 1:129], wl.F32), c.device(torch), dst4(torch, out[..., :128], wl.F32), 0.1, parents=tp)
    torch.cuda.synchronize()
    check(out[..., :128].cpu().numpy(), None, tree_f64(q, c, parents, n_tok, 0.1, False))
    assert torch.all(out[..., 128:] == 7.0)


def test_fa_tree_two_streams_and_one_workspace_in_two_graphs(torch_gpu):
    """Calls on two streams with workspaces of their own; two captured graphs that share one
    workspace, replayed in turn with the table, rows and parents changed between replays."""
    torch = torch_gpu
    sets = [setup(20 + i, wl.Q8_0, 128, 8, 4, 16, [300, 60], 6) for i in range(2)]
    want = [tree_f64(s[2], s[1], s[3], s[4], 0.09, False) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    runs = []
    for s in sets:
        c, q, parents = s[1], s[2], s[3]
        d = {"dev": c.device(torch), "q": torch.from_numpy(q).cuda(), "p": torch.from_numpy(parents).cuda(),
             "out": torch.zeros(q.shape, device="cuda"), "lse": torch.zeros(q.shape[:3], device="cuda")}
        d["args"] = (rows4(torch, d["q"], wl.F32), d["dev"], dst4(torch, d["out"], wl.F32), 0.09)
        runs.append(d)
    torch.cuda.synchronize()
    for _ in range(5):
        for d, st in zip(runs, streams):
            xqattn.fa_tree(*d["args"], parents=d["p"], lse=d["lse"], stream=st)
    torch.cuda.synchronize()
    for d, w in zip(runs, want):
        check(d["out"].cpu().numpy(), d["lse"].cpu().numpy(), w)
    ws = torch.empty(max(xqattn.fa_tree_workspace(*d["args"][:3]) for d in runs) + 256, dtype=torch.uint8, device="cuda")
    graphs = []
    for d in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            xqattn.fa_tree(*d["args"], parents=d["p"], lse=d["lse"], workspace=ws)
        graphs.append(g)
    for turn in range(4):
        for k, (g, d, s) in enumerate(zip(graphs, runs, sets)):
            c = s[1]
            rows = np.array([300 - 37 * turn, 60 - turn], np.int32)
            parents = np.stack([random_parents(np.random.default_rng(turn * 7 + k + j), 6) for j in range(2)])
            d["dev"].rows.copy_(torch.from_numpy(rows))
            d["p"].copy_(torch.from_numpy(parents))
            d["out"].fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            c.rows = rows
            w = tree_f64(s[2], c, parents, s[4], 0.09, False)
            check(d["out"].cpu().numpy(), d["lse"].cpu().numpy(), w)
        junk = torch.zeros(1 << 20, device="cuda") + turn
        torch.cuda.synchronize()
        del junk


def test_fa_tree_same_bits_again(torch_gpu):
    _, c, q, parents, n_tok = setup(30, wl.Q4_0, 128, 32, 8, 16, [700, 90, 5], 20)
    a = on_gpu(torch_gpu, q, c, parents, n_tok, 0.09, True)
    for _ in range(3):
        b = on_gpu(torch_gpu, q, c, parents, n_tok, 0.09, True)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_fa_tree_many_sequences(torch_gpu):
    """More sequences than a wave has lanes, most of them short, one long."""
    rows = [3] * 70 + [2500] + [0] * 30
    _, c, q, parents, n_tok = setup(31, wl.E5M2, 128, 4, 2, 16, rows, 2, [2] * 50 + [0] * 5 + [1] * 46)
    q = bf16(q)
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, 0.09, True)
    check(got, lse, tree_f64(q, c, parents, n_tok, 0.09, True))


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("D,H,Hkv,rows,T", [(128, 8, 4, [3, 1500], 2), (256, 8, 4, [1, 400], 12), (128, 8, 4, [2, 90], 30)])
def test_fa_tree_nan_queries_and_keys(torch_gpu, D, H, Hkv, rows, T, narrow, kt):
    """A NaN query makes its own row of dst and lse NaN; a NaN key (or block scale) those of the
    tokens that see it; the others stay as they were."""
    rng, c, q, parents, n_tok = setup(40 + T, TYPES[kt], D, H, Hkv, 16, rows, T)
    q = bf16(q)
    parents[:] = np.arange(T) - 1
    want = tree_f64(q, c, parents, n_tok, 0.08, narrow)
    hit = np.zeros((len(rows), T, H), bool)
    for b, t, h in ((0, 0, 1), (1, T - 1, H - 1), (1, 0, 4)):
        q[b, t, h, rng.integers(D)] = np.nan
        hit[b, t, h] = True
    p, i = c.place(0, rows[0] + T // 2)  # sequence 0, KV head 2: seen from token T / 2 on
    c.view(c.k)[p, i, 2, :2] = (0x7F, 0x7F) if kt == "e5m2" else (0x01, 0x7E)
    hit[0, T // 2:, 4:6] = True
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, 0.08, narrow)
    assert np.isnan(got[hit]).all() and np.isnan(lse[hit]).all()
    assert np.all(np.abs(got - want[0])[~hit] <= want[2][~hit]) and np.all(np.abs(lse - want[1])[~hit] <= want[3][~hit])


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kt", ["f16", "q4_0"])
def test_fa_tree_infinite_values_in_many_segments(torch_gpu, kt, narrow):
    """More segments than workgroups, each with an infinite value of a token's own row: a
    workgroup goes from one to the next with its flags set."""
    B, T = 96, 40
    rng, c, q, parents, n_tok = setup(50, TYPES[kt], 128, 8, 8, 16, [(7 * b) % 40 for b in range(B)], T)
    q = bf16(q)
    parents[:] = np.arange(T) - 1
    want = tree_f64(q, c, parents, n_tok, 0.08, narrow)
    hit = np.zeros(want[0].shape, bool)
    dims = slice(40, 41) if kt == "f16" else slice(32, 64)
    o = {"f16": 80, "q4_0": 18}[kt]
    for b in range(B):
        for h in range(8):
            t = int(rng.integers(1, T))
            p, i = c.place(b, int(c.rows[b]) + t)
            c.view(c.v)[p, i, h, o:o + 2] = (0x00, 0x7C)
            hit[b, t:, h, dims] = True
    got, _ = on_gpu(torch_gpu, q, c, parents, n_tok, 0.08, narrow)
    assert not np.isfinite(got[hit]).any()
    assert np.all(np.abs(got - want[0])[~hit] <= want[2][~hit])
