"""The bias by distance of fa_chunk and kv_weights, with rows on both sides of a token: a prefix lets tokens see rows
behind their own, and what lies further away, on either side, gets less weight."""
import dataclasses

import numpy as np
import pytest

import chunk_cases
from chunk_cases import Params, chunk_f64, weights_f64
from conftest import case_note
from test_gpu_fa_chunk import on_gpu, setup
from test_gpu_fa_tree import TYPES, check
from test_gpu_kv_weights import check as check_weights, on_gpu as weights_on_gpu
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

unbiased = chunk_cases.scores


def scores(x, k, par, slope, at, op):
    """chunk_cases.scores with slope times the distance taken off on both sides; the roundings are the same."""
    s, ds = unbiased(x, k, dataclasses.replace(par, bias=0.0), 0.0, at, op)
    if par.bias:
        bias = slope * np.abs(np.arange(k.shape[0])[None, :] - at[:, None])
        s = s - bias
        ds = ds + bias * 2.0**-20 + np.abs(s) * 2.0**-22
    return s, ds


@pytest.fixture(autouse=True)
def _distance(monkeypatch):
    monkeypatch.setattr(chunk_cases, "scores", scores)


KINDS = [("f16", 128, 16, 4), ("q8_0", 256, 24, 4), ("q4_0", 128, 6, 2), ("e5m2", 256, 4, 4)]


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind,D,H,Hkv", KINDS)
@pytest.mark.parametrize("T", [1, 7, 15, 90])
def test_chunk(torch_gpu, T, kind, D, H, Hkv, narrow):
    rows, n_tok = [0, 100, 733], [T, max(T - 13, 0), T]
    rng, c, q, n_tok = setup(60 + T, TYPES[kind], D, H, Hkv, 16, rows, T, n_tok, narrow)
    first = np.stack([np.sort(rng.integers(-3, r + T, T)) for r in rows])
    first[:, ::7] = 1 << 20
    prefix = [T - 3, 150, 1 << 30]
    for window, cap, docs in ((0, 0.0, False), (0, 30.0, False), (100, 2.0, True)):
        case_note(f"fa_chunk bias beside a prefix {kind} T {T} narrow={narrow} window {window} cap {cap} documents {docs}")
        par = Params(D**-0.5, window, cap, 8.0)
        f = first if docs else None
        check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow, f, prefix), chunk_f64(q, c, n_tok, par, narrow, f, prefix))


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
def test_chunk_of_many_tokens(torch_gpu, narrow):
    """256 pairs a workgroup."""
    rng, c, q, n_tok = setup(61, wl.F16, 128, 16, 16, 64, [200], 300, None, narrow)
    par = Params(128**-0.5, 0, 0.0, 8.0)
    case_note(f"fa_chunk bias beside a prefix, 300 tokens narrow={narrow}")
    check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow, None, [350]), chunk_f64(q, c, n_tok, par, narrow, None, [350]))


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind,D,H,Hkv", KINDS)
@pytest.mark.parametrize("T", [1, 3, 40])
def test_weights(torch_gpu, T, kind, D, H, Hkv, narrow):
    rows, n_tok = [0, 100, 333], [T, T, (T + 1) // 2]
    rng, c, q, n_tok = setup(62 + T, TYPES[kind], D, H, Hkv, 16, rows, T, n_tok, narrow)
    prefix = [30, 120, 1 << 30]
    for window, cap in ((0, 0.0), (50, 30.0)):
        case_note(f"kv_weights bias beside a prefix {kind} T {T} narrow={narrow} window {window} cap {cap}")
        par = Params(D**-0.5, window, cap, 8.0)
        lse = np.nan_to_num(chunk_f64(q, c, n_tok, par, narrow, None, prefix)[1], nan=0.0).astype(np.float32)
        cols = max(rows) + T
        want = weights_f64(q, c, n_tok, par, lse, None, cols, 1.0, True, None, prefix)
        check_weights(weights_on_gpu(torch_gpu, q, c, par, n_tok, narrow, lse, None, cols, 1.0, True, None, prefix), want)


def test_equal_scores_fall_off_on_both_sides(torch_gpu):
    """Queries of 0: the first head's weights are e^(-|distance| / sqrt 2), worked out by geometric sums."""
    T, held, end = 64, 100, 164
    rng, c, q, n_tok = setup(63, wl.F16, 128, 16, 4, 16, [held], T)
    q[...] = 0.0
    case_note("fa_chunk bias beside a prefix, queries of 0")
    _, lse = on_gpu(torch_gpu, q, c, Params(0.1, 0, 0.0, 8.0), n_tok, False, None, [end])
    r = np.exp(-2.0**-0.5)
    for t in range(T):
        before, behind = held + t, end - 1 - held - t
        want = np.log(1.0 + r * (1 - r**before) / (1 - r) + r * (1 - r**behind) / (1 - r))
        # (a slope of 8 steps on a distance whose weight matters, up to 20; 164 sums; the logarithm)
        assert abs(lse[0, t, 0] - want) <= 20 * 2.0**-20 + 164 * 2.0**-24 + 2.0**-20
