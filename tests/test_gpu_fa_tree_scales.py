"""Attention of drafted tokens where the values of a row are far larger than the others: in a row
that a token does not see, and in one that it sees with next to no weight."""
import numpy as np
import pytest

import oracle
from conftest import case_note
from paged_cases import Cache, ancestors, bf16, tree_f64
from test_gpu_fa_tree import TYPES, check, on_gpu, setup

pytestmark = pytest.mark.gpu

BLOCK = {"q8_0": 34, "q4_0": 18}
# D, H, Hkv, T: up to 16, 32, 64, 128 pairs of a KV head, and more
FORMS = [(128, 8, 4, 8), (128, 8, 4, 13), (128, 8, 4, 24), (128, 8, 4, 40), (128, 16, 4, 40),
         (256, 12, 4, 5), (256, 12, 4, 10), (256, 12, 4, 20), (256, 12, 4, 40)]


def set_scale(c, buf, b, r, block, value):
    """The scale of a block of one row, in every KV head."""
    p, i = c.place(b, r)
    bb = c.rec // (c.D // 32)
    c.view(buf)[p, i, :, block * bb:block * bb + 2] = np.array([value], np.float16).view(np.uint8)


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kt", list(BLOCK))
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_large_scales_of_unseen_rows_change_no_bit(torch_gpu, form, kt, narrow):
    """Two chains of drafted tokens: finite scales of 32, 1024 and 65504 in the K and V rows of the
    second leave the first's results as they are without them, bit for bit."""
    D, H, Hkv, T = FORMS[form]
    case_note(f"unseen scales {FORMS[form]} {kt} narrow {narrow}")
    _, c, q, parents, n_tok = setup(60 + form, TYPES[kt], D, H, Hkv, 16, [90, 33], T, spare=0)
    if narrow:
        q = bf16(q)
    parents[:] = np.arange(-2, T - 2)
    parents[:, :2] = -1
    scale = D**-0.5
    want = tree_f64(q, c, parents, n_tok, scale, narrow)
    plain = on_gpu(torch_gpu, q, c, parents, n_tok, scale, narrow)
    first = np.arange(T) % 2 == 0
    assert np.all(np.abs(plain[0] - want[0])[:, first] <= want[2][:, first])
    for value in (32.0, 1024.0, 65504.0):
        for b in range(2):
            for j in range(1, T, 2):
                for n, buf in enumerate((c.k, c.v)):
                    set_scale(c, buf, b, int(c.rows[b]) + j, (j + n) % (D // 32), value)
        got = on_gpu(torch_gpu, q, c, parents, n_tok, scale, narrow)
        for x, y in zip(got, plain):
            assert np.array_equal(x[:, first], y[:, first]), (value, np.abs(x - y)[:, first].max())


def spread_case(seed, kt, D, H, Hkv, T, rows, power, v_scale):
    """Queries around one direction; row 37 lies against it, so that its weight is about 2^-power."""
    rng = np.random.default_rng(seed)
    c = Cache(rng, TYPES[kt], D, Hkv, 16, [rows], [T])
    u = rng.standard_normal(D)
    u /= np.linalg.norm(u)
    q = (8 * u + rng.standard_normal((1, T, H, D))).astype(np.float32)
    p, i = c.place(0, 37)
    against = np.tile((-power * np.log(2) * D**0.5 / 8 * u).astype(np.float32), (Hkv, 1))
    c.view(c.k)[p, i] = oracle.quantize(c.kv_type, against).reshape(Hkv, c.rec)
    v = (rng.standard_normal((c.n_pages, 16, Hkv, D)) * v_scale).astype(np.float32)
    c.view(c.v)[...] = oracle.quantize(c.kv_type, v).reshape(c.n_pages, 16, Hkv, c.rec)
    parents = (np.arange(T, dtype=np.int32) - 1)[None]
    return c, q, parents


def check_f32(c, q, parents, scale, got, lse, unit):
    """float64 and per-element bounds for f32 q: a score is off by its operands' 2^-21 and D + 8 f32
    operations, a weight by its score's and the sums' error and 2^-20, a term by that and one f32
    operation per row in the sum; `unit(w, b)`: the terms' absolute error, from the rows' weights and
    their decoded rows."""
    _, T, H, D = q.shape
    n0 = int(c.rows[0])
    K, V = (c.values(x, 0, n0 + T) for x in (c.k, c.v))
    tree = ancestors(parents[0])
    for t in range(T):
        rows = np.array([r for r in range(n0 + T) if r < n0 or tree[t, r - n0]])
        for h in range(H):
            k, v, x = K[rows, h // (H // c.Hkv)], V[rows, h // (H // c.Hkv)], q[0, t, h].astype(np.float64)
            s = k @ x * scale
            m = s.max()
            w = np.exp(s - m)
            z = w.sum()
            w /= z
            ds = np.abs(k) @ np.abs(x) * scale * (2.0**-21 + (D + 8) * 2.0**-24) + (np.abs(s) + abs(m)) * 2.0**-22
            rel = ds + w @ ds + 2.0**-20 + len(rows) * 2.0**-24
            tol = (w * rel) @ np.abs(v) + unit(w, rows, h // (H // c.Hkv)) + 2.0**-24 * np.abs(w @ v)
            err = np.abs(got[0, t, h] - w @ v)
            assert np.all(err <= tol), f"token {t} head {h}: off by {err.max():.3e}, {(err / tol).max():.1f} times its bound"
            assert abs(lse[0, t, h] - m - np.log(z)) <= w @ ds + 2.0**-19 + len(rows) * 2.0**-24 + abs(m) * 2.0**-22


@pytest.mark.parametrize("value,power", [(1024.0, 12), (1024.0, 30), (65504.0, 8), (65504.0, 20), (65504.0, 30), (65504.0, 60)])
@pytest.mark.parametrize("kt", list(BLOCK))
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_a_large_scale_of_next_to_no_weight(torch_gpu, form, kt, value, power):
    """A seen row with a block scale far above the others' and a weight of about 2^-power: the others
    keep their bits.

    With d the largest block scale of a row and M the largest w d: a weight times scale is an f16 high
    and low part at 2^11 or more for M, so one is off by 2^-25 / 2^11 of M at least, times an integer
    of up to 128; where the row's values are formed with their scales first, those scales are f16 at
    2^7 or more for d, off by 2^-25 / 2^7 of it."""
    D, H, Hkv, T = FORMS[form]
    case_note(f"large scale {FORMS[form]} {kt} {value} 2^-{power}")
    c, q, parents = spread_case(70 + form, kt, D, H, Hkv, T, 130, power, 1.0)
    set_scale(c, c.v, 0, 37, 1, value)
    d = np.stack([np.abs(np.ascontiguousarray(c.view(c.v)[c.place(0, r)].reshape(Hkv, -1, BLOCK[kt])[..., :2]).view(np.float16)[..., 0].astype(np.float64)).max(-1)
                  for r in range(130 + T)])

    def unit(w, rows, hk):
        wd = w * d[rows, hk]
        return 128 * (len(rows) * 2.0**-36 * wd.max() + 2.0**-32 * wd.sum())

    got, lse = on_gpu(torch_gpu, q, c, parents, None, D**-0.5, False)
    check_f32(c, q, parents, D**-0.5, got, lse, unit)


@pytest.mark.parametrize("power", [28, 30, 32, 34])
@pytest.mark.parametrize("kt", ["f16", "e5m2"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_large_values_of_little_weight(torch_gpu, form, kt, power):
    """Values of 2^15 and more at a weight of about 2^-power, the others near 2^-6: what they add up
    to keeps its bits.

    A weight is an f16 high and low part at 2^12 or more for the largest: one is off by 2^-25 / 2^12 of
    the largest at least, and that is at most the sum of all."""
    D, H, Hkv, T = FORMS[form]
    case_note(f"large values {FORMS[form]} {kt} 2^-{power}")
    c, q, parents = spread_case(80 + form, kt, D, H, Hkv, T, 130, power, 2.0**-6)
    p, i = c.place(0, 37)
    big = np.random.default_rng(form).choice([-57344.0, -32768.0, 32768.0, 57344.0], (Hkv, D)).astype(np.float32)
    c.view(c.v)[p, i] = oracle.quantize(c.kv_type, big).reshape(Hkv, c.rec)
    v = np.abs(c.values(c.v, 0, 130 + T))
    got, lse = on_gpu(torch_gpu, q, c, parents, None, D**-0.5, False)
    check_f32(c, q, parents, D**-0.5, got, lse, lambda w, rows, hk: 2.0**-37 * v[rows, hk].sum(0))


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kt", ["f16", "q8_0"])
@pytest.mark.parametrize("scale,power", [(3e38, -123), (-3e38, -123), (1e-40, 126), (-1e-40, 126), (3e38, 100)])
def test_scales_at_the_ends_of_f32(torch_gpu, kt, narrow, scale, power):
    """Scales whose product with log2(e) leaves f32's normal range, and queries that bring the scores
    back; where nothing can (the last), keys of zeros still score 0."""
    rng = np.random.default_rng(90)
    c = Cache(rng, TYPES[kt], 128, 4, 16, [100], [5])
    x = rng.standard_normal((c.n_pages, 16, 4, 128)).astype(np.float32) * {-123: 2.0**-8, 126: 2.0**5, 100: 0.0}[power]
    c.view(c.k)[...] = oracle.quantize(c.kv_type, x.astype(np.float32)).reshape(c.n_pages, 16, 4, c.rec)
    q = bf16((rng.standard_normal((1, 5, 8, 128)) * 2.0**power).astype(np.float32))
    assert np.isfinite(q).all()
    parents = (np.arange(5, dtype=np.int32) - 1)[None]
    scale = float(np.float32(scale))
    got, lse = on_gpu(torch_gpu, q, c, parents, None, scale, narrow)
    check(got, lse, tree_f64(q, c, parents, [5], scale, narrow))


SMALL = {"f16": -12, "q8_0": -12, "q4_0": -12, "e5m2": -10}


def small_case(kt, narrow):
    """K and V at a power of two where elements or block scales still hold several bits, queries that
    bring the scores back to 1; the bounds of tree_f64 without its absolute 2^-24."""
    rng = np.random.default_rng(95)
    c = Cache(rng, TYPES[kt], 128, 4, 16, [150], [6])
    for n, buf in enumerate((c.k, c.v)):
        x = np.random.default_rng(96 + n).standard_normal((c.n_pages, 16, 4, 128)) * 2.0**SMALL[kt]
        c.view(buf)[...] = oracle.quantize(c.kv_type, x.astype(np.float32)).reshape(c.n_pages, 16, 4, c.rec)
    q = bf16((rng.standard_normal((1, 6, 8, 128)) * 2.0**-SMALL[kt]).astype(np.float32))
    parents = (np.arange(6, dtype=np.int32) - 1)[None]
    out, lse, tol, tol_lse = tree_f64(q, c, parents, [6], 0.09, narrow)
    if not narrow:
        tol = tol - 2.0**-24 + 2.0**-24 * (np.abs(out) + tol)
    return c, q, parents, (out, lse, tol, tol_lse)


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
def test_small_values_and_keys(torch_gpu, kt, narrow):
    c, q, parents, want = small_case(kt, narrow)
    # (an output of zeros would not pass)
    assert np.mean(np.abs(want[0]) > want[2]) > (0.6 if narrow else 0.99)
    got, lse = on_gpu(torch_gpu, q, c, parents, None, 0.09, narrow)
    check(got, lse, want)


@pytest.mark.parametrize("T", [5, 40])
def test_a_score_of_minus_infinity_is_no_weight(torch_gpu, T):
    """bf16 Q and a key with an infinite element: where its score is -inf the row has no part, where it
    is +inf the result is NaN."""
    _, c, q, parents, n_tok = setup(99, TYPES["f16"], 128, 8, 4, 1, [100], T)
    q = bf16(q)
    assert np.all(q[..., 9] != 0)
    p, i = c.place(0, 37)
    c.view(c.k)[p, i, :, 18:20] = np.array([np.inf], np.float16).view(np.uint8)
    got, lse = on_gpu(torch_gpu, q, c, parents, n_tok, 0.08, True)
    c.table[0, 37] = -1  # (a page of that row alone) for the reference: not seen
    out, wlse, tol, tol_lse = tree_f64(q, c, parents, n_tok, 0.08, True)
    minus = q[..., 9] < 0
    assert np.all(np.abs(got - out)[minus] <= tol[minus]) and np.all(np.abs(lse - wlse)[minus] <= tol_lse[minus])
    assert np.isnan(got[~minus]).all() and np.isnan(lse[~minus]).all()
