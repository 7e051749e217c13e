"""Norms and rotation of queries and keys into the paged cache, against float64.

Tolerances: y = x * inv * w has the sum of squares (D / 64 f32 steps a lane, 6 across lanes), a
division, a root and three products: under 16 roundings of 2^-24, halved by the root; the turn
two products and a sum of elements of at most sqrt(2) the larger, cos and sin within 2^-22:
together 2^-20 of the pair's length, plus the rounding of what is stored."""
import numpy as np
import pytest

import oracle
import xqattn
from conftest import case_note
from paged_cases import Cache, bf16, rope_f64
from test_gpu_fa_tree import rows4
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

TYPES = {"f32": wl.F32, "f16": wl.F16, "bf16": wl.BF16, "e5m2": wl.E5M2, "q8_0": wl.Q8_0, "q4_0": wl.Q4_0}
STEP = {"f32": 0.0, "f16": 2.0**-11, "bf16": 2.0**-8, "e5m2": 2.0**-3 + 2.0**-11}


def zero_cache(c):
    c.k[:] = 0xCD
    c.v[:] = 0xCD
    return c


def make_cache(rng, kt, D, Hkv, P, rows, n_tok, **more):
    """A cache of any stored type; its bytes are a pattern that a store overwrites."""
    real = oracle.quantize
    try:  # the content is replaced below: bf16 and f32 records need no quantizer of their own
        oracle.quantize = lambda typ, x, *a: np.zeros(x.size // D * wl.record_bytes(typ, D), np.uint8)
        c = Cache(rng, kt, D, Hkv, P, rows, n_tok, **more)
    finally:
        oracle.quantize = real
    return zero_cache(c)


def decode(c, raw):
    """float64 [..., D] of records uint8 [..., rec]."""
    shape = raw.shape[:-1] + (c.D,)
    flat = np.ascontiguousarray(raw).reshape(-1)
    if c.kv_type == wl.F32:
        return flat.view(np.float32).astype(np.float64).reshape(shape)
    if c.kv_type == wl.BF16:
        return (flat.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(shape)
    return oracle.dequant(c.kv_type, flat, int(np.prod(shape))).astype(np.float64).reshape(shape)


def run(torch, q, k, v, pos, w, c, params, n_tok=None, ff=None, tin="f32", tout="f32", in_place=False, gate=1, stream=None, dev=None):
    """q [B, T, H, D] ... -> (q_out, K bytes, V bytes). `gate`: query heads that many head dims apart."""
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}
    B, T, H, D = q.shape
    wide = torch.zeros((B, T, H, gate * D), dtype=dt[tin], device="cuda")
    wide[..., :D] = torch.from_numpy(q).cuda().to(dt[tin])
    tq = wide[..., :D]
    kv = torch.cat([torch.from_numpy(x).cuda().to(dt[tin]) for x in (k, v)], 2)  # fused: k heads, then v heads
    tk, tv = kv[:, :, :k.shape[2]], kv[:, :, k.shape[2]:]
    out = tq if in_place else torch.full((B, T, H, D), 7.0, dtype=dt[tout], device="cuda")
    dev = dev or c.device(torch)
    put = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    tp, tn, tw, tf = put(pos.astype(np.int32)), put(None if n_tok is None else np.array(n_tok, np.int32)), [put(x) for x in w], put(ff)
    torch.cuda.synchronize()
    xqattn.qk_norm_rope(rows4(torch, tq, TYPES[tin]), rows4(torch, tk, TYPES[tin]), rows4(torch, tv, TYPES[tin]), tp, params,
                        rows4(torch, out, TYPES[tin if in_place else tout]), dev, q_weight=tw[0], k_weight=tw[1], n_tok=tn,
                        freq_factors=tf, stream=stream)
    torch.cuda.synchronize()
    return out.float().cpu().numpy(), dev.k.t.cpu().numpy(), dev.v.t.cpu().numpy()


def expect_cache(c, kraw, vraw, want_k, want_v, n_tok, length_k):
    """Stored records of the new tokens; every other byte as it was."""
    name = {v: n for n, v in TYPES.items()}[c.kv_type]
    for buf, was, want, exact in ((kraw, c.k, want_k, False), (vraw, c.v, want_v, True)):
        touched = np.zeros(buf.shape, bool)
        mark, got = c.view(touched.view(np.uint8)), c.view(buf)
        for b in range(len(c.rows)):
            for i in range(n_tok[b]):
                r = int(c.rows[b]) + i
                if r < 0 or r // c.P >= c.cols or not 0 <= c.table[b, r // c.P] < c.n_pages:
                    continue
                p, j = c.place(b, r)
                mark[p, j] = 1
                w = want[b, i]
                g = decode(c, got[p, j])
                slack = 0.0 if exact else length_k[b, i] * 2.0**-20
                if name in STEP:
                    tol = slack * (1 + STEP[name]) + STEP[name] * np.abs(w) + (2.0**-25 if name == "f16" else 2.0**-17 if name == "e5m2" else 0)
                else:  # half a step of the block (q4_0: its largest element may take -8, the other end stops at 7)
                    amax = np.abs(w.reshape(w.shape[0], -1, 32)).max(-1, keepdims=True) * np.ones(32)
                    step = amax.reshape(w.shape) / (127 if name == "q8_0" else 8)
                    tol = slack * 2 + step * (0.5 if name == "q8_0" else 1.0) + (127 if name == "q8_0" else 8) * step * 2.0**-10 + 2.0**-16
                assert np.all(np.abs(g - w) <= tol), (b, i, np.max(np.abs(g - w) / np.maximum(tol, 1e-30)))
        assert np.array_equal(buf[~touched], was[~touched]), "bytes outside the new rows changed"


def pair_length(x, w, eps, n_rot, mode):
    """Per element, the length of the pair it turns in (its own size past n_rot)."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w
    n = np.abs(y)
    h = n_rot // 2
    a, b = (slice(0, h), slice(h, n_rot)) if mode == 0 else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    s = np.hypot(y[..., a], y[..., b])
    n[..., a], n[..., b] = s, s
    return n + 1e-30


CASES = [
    # D, H, Hkv, T, rows, n_tok, n_rot, mode, in, out
    (256, 24, 4, 1, [1000], None, 64, 0, "f32", "f32"),
    (128, 32, 8, 25, [900, 0, 31], [25, 1, 0], 128, 0, "bf16", "bf16"),
    (64, 6, 3, 5, [3, 17], None, 32, 1, "f32", "bf16"),      # heads that end inside a wave's load
    (64, 1, 1, 3, [0], None, 64, 0, "bf16", "f32"),
    (128, 5, 1, 7, [10, 2, 60], [7, 3, 5], 90, 1, "f32", "f32"),  # a turn that ends inside a lane
    (256, 2, 1, 33, [5], None, 256, 0, "bf16", "f32"),
    (128, 8, 4, 9, [40], None, 0, 0, "f32", "f32"),          # nothing turns
    (256, 24, 4, 130, [7, 300], None, 8, 0, "bf16", "bf16"),
    (128, 16, 8, 700, [0, 5], [700, 633], 128, 0, "bf16", "bf16"),  # several units per wave
]


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("case", range(len(CASES)))
def test_qk_norm_rope(torch_gpu, case, kt):
    D, H, Hkv, T, rows, n_tok, n_rot, mode, tin, tout = CASES[case]
    case_note(f"qk_norm_rope {CASES[case]} {kt}")
    rng = np.random.default_rng(case)
    B = len(rows)
    n_tok = n_tok or [T] * B
    c = make_cache(rng, TYPES[kt], D, Hkv, (16, 5, 64)[case % 3], rows, n_tok, head_major=case % 2 == 1,
                   pad=0 if case % 4 else 4)
    q, k, v = (rng.standard_normal((B, T, h, D)).astype(np.float32) * np.float32(3.0) for h in (H, Hkv, Hkv))
    if tin == "bf16":
        q, k, v = bf16(q), bf16(k), bf16(v)
    w = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
    pos = (np.array(rows)[:, None] + (0, 1, 131072, 1000003)[case % 4] + np.arange(T)).astype(np.int32)
    p = xqattn.rope_params(n_rot, 1e7 if D == 256 else 1e4, mode=mode)
    got, kraw, vraw = run(torch_gpu, q, k, v, pos, w, c, p, n_tok, tin=tin, tout=tout, gate=1 + case % 2)
    base = 1e7 if D == 256 else 1e4
    want = rope_f64(q, w[0], pos, n_rot, base, mode, 1e-6)
    tol = pair_length(q, w[0], 1e-6, n_rot, mode) * 2.0**-20
    if tout == "bf16":
        tol = tol + 2.0**-8 * (np.abs(want) + tol)
    for b in range(B):
        t = n_tok[b]
        assert np.all(np.abs(got[b, :t] - want[b, :t]) <= tol[b, :t]), np.max(np.abs(got[b, :t] - want[b, :t]) / tol[b, :t])
        assert np.all(got[b, t:] == 7.0), "padding tokens were written"
    expect_cache(c, kraw, vraw, rope_f64(k, w[1], pos, n_rot, base, mode, 1e-6), v.astype(np.float64), n_tok,
                 pair_length(k, w[1], 1e-6, n_rot, mode))


def _small(seed, kt=wl.F32, D=128, H=8, Hkv=4, T=6, rows=(20, 3), **more):
    rng = np.random.default_rng(seed)
    c = make_cache(rng, kt, D, Hkv, 16, list(rows), [T] * len(rows), **more)
    q, k, v = (rng.standard_normal((len(rows), T, h, D)).astype(np.float32) for h in (H, Hkv, Hkv))
    pos = (np.array(rows)[:, None] + np.arange(T)).astype(np.int32)
    w = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
    return rng, c, q, k, v, pos, w


@pytest.mark.parametrize("weights", [(True, False), (False, True), (False, False)])
def test_qk_norm_rope_without_norm(torch_gpu, weights):
    rng, c, q, k, v, pos, w = _small(40)
    w = [x if on else None for x, on in zip(w, weights)]
    got, kraw, _ = run(torch_gpu, q, k, v, pos, w, c, xqattn.rope_params(64, 1e4))
    want = rope_f64(q, w[0], pos, 64, 1e4, 0, 1e-6)
    assert np.all(np.abs(got - want) <= pair_length(q, w[0], 1e-6, 64, 0) * 2.0**-20)
    wk = rope_f64(k, w[1], pos, 64, 1e4, 0, 1e-6)
    view = c.view(kraw)
    for b in range(2):
        for i in range(6):
            g = decode(c, view[c.place(b, int(c.rows[b]) + i)])
            assert np.all(np.abs(g - wk[b, i]) <= pair_length(k, w[1], 1e-6, 64, 0)[b, i] * 2.0**-20)


@pytest.mark.parametrize("mode", [0, 1])
def test_qk_norm_rope_factors_scale_and_positions(torch_gpu, mode):
    """Frequency factors, position scale, attention factor; positions negative, zero, the largest."""
    rng, c, q, k, v, _, w = _small(41)
    pos = np.array([[-5, 0, 1, 2**31 - 1, -2**31, 262143], [7, 7, 7, 100000, 99999, 3]], np.int32)
    ff = np.exp(rng.uniform(0, 3, 32)).astype(np.float32)
    p = xqattn.rope_params(64, 5e5, freq_scale=0.25, attn_factor=1.125, mode=mode, eps=1e-5)
    got, kraw, vraw = run(torch_gpu, q, k, v, pos, w, c, p, ff=ff)
    args = (pos, 64, np.float32(5e5), mode, 1e-5, 0.25, ff, 1.125)
    # an angle of up to 2^29 rad: f64 keeps 2^-53 of it, twice over its factors (2^-22 rad)
    slack = 2.0**-20 + 2.0**-21
    assert np.all(np.abs(got - rope_f64(q, w[0], *args)) <= 1.125 * pair_length(q, w[0], 1e-5, 64, mode) * slack)
    expect_cache(c, kraw, vraw, rope_f64(k, w[1], *args), v.astype(np.float64), [6, 6], 2.25 * pair_length(k, w[1], 1e-5, 64, mode))


@pytest.mark.parametrize("tin", ["f32", "bf16"])
def test_qk_norm_rope_in_place(torch_gpu, tin):
    rng, c, q, k, v, pos, w = _small(42, T=40)
    q, k, v = bf16(q), bf16(k), bf16(v)
    p = xqattn.rope_params(128, 1e4)
    a, ka, va = run(torch_gpu, q, k, v, pos, w, c, p, tin=tin, tout=tin, gate=2)
    b, kb, vb = run(torch_gpu, q, k, v, pos, w, c, p, tin=tin, tout=tin, gate=2, in_place=True)
    assert np.array_equal(a, b) and np.array_equal(ka, kb) and np.array_equal(va, vb)


@pytest.mark.parametrize("kt", ["f16", "q8_0", "q4_0"])
def test_qk_norm_rope_stores_what_kv_store_stores(torch_gpu, kt):
    """Without norm and turn the cache rows are the KV append's, byte for byte, both q8_0 variants."""
    torch = torch_gpu
    for variant in (0, 1):
        rng, c, q, k, v, pos, _ = _small(43, TYPES[kt])
        p = xqattn.rope_params(0, 1e4, q8_variant=variant)
        _, kraw, vraw = run(torch, q, k, v, pos, (None, None), c, p)
        for x, raw in ((k, kraw), (v, vraw)):
            plane = torch.zeros(12 * 4 * c.rec, dtype=torch.uint8, device="cuda")
            at = torch.arange(12, dtype=torch.int32, device="cuda")
            xqattn.kv_store(torch.from_numpy(x).cuda().contiguous(), at, 4, 128, TYPES[kt], plane, 12, q8_variant=variant)
            torch.cuda.synchronize()
            want = plane.cpu().numpy().reshape(2, 6, 4, c.rec)
            for b in range(2):
                for i in range(6):
                    assert np.array_equal(c.view(raw)[c.place(b, int(c.rows[b]) + i)], want[b, i])


def test_qk_norm_rope_rows_without_a_page_are_not_stored(torch_gpu):
    rng, c, q, k, v, pos, w = _small(44, wl.F16, rows=(14, 30, 5, 40))
    c.table[0, 1] = c.n_pages  # rows 16.. of sequence 0
    c.table[1, 1:] = -1
    c.rows[2] = c.cols * 16 - 2  # the last rows of the table, then past it
    c.table[2] = -1
    c.rows[3] = -3
    got, kraw, vraw = run(torch_gpu, q, k, v, pos, w, c, xqattn.rope_params(64, 1e4))
    want = rope_f64(q, w[0], pos, 64, 1e4, 0, 1e-6)
    assert np.all(np.abs(got - want) <= pair_length(q, w[0], 1e-6, 64, 0) * 2.0**-20)
    expect_cache(c, kraw, vraw, rope_f64(k, w[1], pos, 64, 1e4, 0, 1e-6), v.astype(np.float64), [6] * 4, pair_length(k, w[1], 1e-6, 64, 0))


def test_qk_norm_rope_non_finite_rows_stay_their_own(torch_gpu):
    """An Inf or NaN in one head's row changes that row alone (norm: the whole row)."""
    rng, c, q, k, v, pos, w = _small(45)
    p = xqattn.rope_params(64, 1e4)
    clean, kc, vc = run(torch_gpu, q, k, v, pos, w, c, p)
    q2, k2 = q.copy(), k.copy()
    q2[0, 2, 3, 5], k2[1, 1, 2, 100] = np.inf, np.nan
    got, kraw, vraw = run(torch_gpu, q2, k2, v, pos, w, c, p)
    hit = np.zeros(q.shape[:3], bool)
    hit[0, 2, 3] = True
    assert np.array_equal(got[~hit], clean[~hit]) and np.isnan(got[0, 2, 3, 5]) and np.array_equal(vraw, vc)
    rows = decode(c, c.view(kraw)[c.place(1, int(c.rows[1]) + 1)])
    assert np.isnan(rows[2]).all() and np.isfinite(rows[[0, 1, 3]]).all()


def test_qk_norm_rope_graph_and_stream(torch_gpu):
    """A captured call replayed with other positions and rows; a call on another stream."""
    torch = torch_gpu
    rng, c, q, k, v, pos, w = _small(46, T=2, rows=(20, 3, 9))
    c = make_cache(rng, wl.F32, 128, 4, 16, [40, 40, 40], [2] * 3)
    dev = c.device(torch)
    t = [torch.from_numpy(x).cuda() for x in (q, k, v)]
    out = torch.zeros_like(t[0])
    tp, tw = torch.from_numpy(pos).cuda(), [torch.from_numpy(x).cuda() for x in w]
    p = xqattn.rope_params(64, 1e4)
    call = lambda **kw: xqattn.qk_norm_rope(*[rows4(torch, x, wl.F32) for x in t], tp, p, rows4(torch, out, wl.F32), dev, q_weight=tw[0], k_weight=tw[1], **kw)  # noqa: E731
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for turn in range(4):
        rows = np.array([turn, 3 * turn, 38], np.int32)
        pos2 = (rows[:, None] * 1000 + np.arange(2)).astype(np.int32)
        dev.rows.copy_(torch.from_numpy(rows))
        tp.copy_(torch.from_numpy(pos2))
        for x in (dev.k.t, dev.v.t):
            x.fill_(0xCD)
        out.fill_(7.0)
        torch.cuda.synchronize()
        if turn < 3:
            g.replay()
        else:
            call(stream=torch.cuda.Stream())
        torch.cuda.synchronize()
        c.rows = rows
        want = rope_f64(q, w[0], pos2, 64, 1e4, 0, 1e-6)
        assert np.all(np.abs(out.cpu().numpy() - want) <= pair_length(q, w[0], 1e-6, 64, 0) * 2.0**-20)
        expect_cache(c, dev.k.t.cpu().numpy(), dev.v.t.cpu().numpy(), rope_f64(k, w[1], pos2, 64, 1e4, 0, 1e-6), v.astype(np.float64),
                     [2] * 3, pair_length(k, w[1], 1e-6, 64, 0))
