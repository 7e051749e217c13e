"""Non-finite values in rows that some tokens of a chunk see and others do not, in every form of the kernel: exactly
the tokens that see such a row get its value, whether their own rows end inside its tile or only their neighbours' do."""
import numpy as np
import pytest

from chunk_cases import Params, chunk_f64
from conftest import case_note
from test_gpu_fa_chunk import on_gpu, setup
from test_gpu_fa_tree import TYPES
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

INF, NAN, NEG = 0x7C00, 0x7E00, 0xFC00

# Several waves of a workgroup with pairs of their own, so that a tile's rows can end for one wave's tokens and not for
# another's: 32 pairs a workgroup, 64, and 128 (heads of 256) or 256 (of 128), alone and as parts of a long cache.
SHAPES = [
    # D, H, Hkv, page rows, rows of each sequence, T, tokens of each sequence
    (128, 8, 8, 16, [300, 1000, 30, 77], 30, [30, 29, 30, 17]),    # 30 pairs, dealt by the lengths
    (128, 32, 8, 16, [90], 110, None),                             # 440 pairs, 32 a workgroup
    (256, 8, 8, 5, [1000, 500], 61, [61, 60]),                     # 61 pairs, dealt by the lengths
    (128, 16, 4, 32, [30], 300, None),                             # 1200 pairs, 64 a workgroup
    (256, 12, 4, 16, [30, 131], 260, [260, 201]),                  # 780 pairs, 128 a workgroup
    (128, 16, 16, 64, [200], 300, None),                           # 300 pairs, 256 a workgroup
    (128, 8, 2, 16, [30, 5], 512, [512, 70]),                      # 2048 pairs, 256 a workgroup
]
KINDS = [("f16", True), ("f16", False), ("e5m2", True), ("q8_0", False), ("q8_0", True), ("q4_0", False), ("q4_0", True), ("e5m2", False)]


def spoil(c, buf, b, row, head, element, bits):
    """One element (quantized: its block's scale) becomes what `bits` are in f16."""
    p, x = c.place(b, row)
    rec = c.view(buf)[p, x, head]
    if c.kv_type == wl.F16:
        rec[2 * element:2 * element + 2] = np.array([bits], np.uint16).view(np.uint8)
    elif c.kv_type == wl.E5M2:
        rec[element] = bits >> 8
    else:
        at = element // 32 * wl.TYPE_SIZE[c.kv_type]
        rec[at:at + 2] = np.array([bits], np.uint16).view(np.uint8)


def check(got, lse, want):
    out, wl_, tol, tol_lse = want
    live = ~np.isnan(wl_[..., 0])
    hit = ~np.isfinite(out[live])
    assert hit.any() and not hit.all()
    wrong = np.isfinite(got[live]) == hit
    assert not wrong.any(), f"{wrong.sum()} of {hit.sum()} non-finite elements are lost or reach others"
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(got[live] - out[live]) <= tol[live]) | hit)
    assert np.all(np.abs(lse[live] - wl_[live]) <= tol_lse[live])


@pytest.mark.parametrize("kind,narrow", KINDS, ids=lambda x: {True: "bf16", False: "f32"}.get(x, x))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[0]}h{s[1]}kv{s[2]}p{s[3]}t{s[5]}")
def test_values_reach_all_that_see_them(torch_gpu, shape, kind, narrow):
    D, H, Hkv, P, rows, T, n_tok = shape
    rng, c, q, n_tok = setup(70 + T, TYPES[kind], D, H, Hkv, P, rows, T, n_tok, narrow)
    for b, (r, t) in enumerate(zip(rows, n_tok)):
        # the first tile, inside the held rows, where windows of 100 end, among the tokens' own
        for i, row in enumerate(sorted({3, r // 2, max(r - 60, 1), r + t // 3, r + t - 3})):
            spoil(c, c.v, b, row, (b + i) % Hkv, (37 * i + 5) % D, (INF, NAN, NEG)[i % 3])
    docs = np.stack([np.where(np.arange(T) < T // 2, 0, r + T // 2 - 20) for r in rows])
    for window, first in ((0, None), (100, None), (0, docs)):
        case_note(f"fa_chunk non-finite values {kind} narrow={narrow} {shape} window {window} documents {first is not None}")
        par = Params(D**-0.5, window)
        check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow, first), chunk_f64(q, c, n_tok, par, narrow, first))


@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("shape", [SHAPES[1], SHAPES[4], SHAPES[6]], ids=lambda s: f"d{s[0]}h{s[1]}kv{s[2]}p{s[3]}t{s[5]}")
def test_products_beyond_f16_are_infinite_for_all_that_see_them(torch_gpu, shape, kind):
    """Beside BF16 q a quantized value d * q beyond 65504 is infinite."""
    D, H, Hkv, P, rows, T, n_tok = shape
    rng, c, q, n_tok = setup(71, TYPES[kind], D, H, Hkv, P, rows, T, n_tok, True)
    scale = np.array([1000.0 if kind == "q8_0" else 16000.0], np.float16).view(np.uint16)[0]
    for b, (r, t) in enumerate(zip(rows, n_tok)):
        for i, row in enumerate((3, r + t // 3)):
            spoil(c, c.v, b, row, i % Hkv, 40, int(scale))
    values = c.values
    c.values = lambda buf, b, n: np.where(np.abs(x := values(buf, b, n)) >= 65520.0, np.copysign(np.inf, x), x)
    case_note(f"fa_chunk products beyond f16 {kind} {shape}")
    par = Params(D**-0.5)
    check(*on_gpu(torch_gpu, q, c, par, n_tok, True), chunk_f64(q, c, n_tok, par, True))


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[3], SHAPES[4], SHAPES[6]], ids=lambda s: f"d{s[0]}h{s[1]}kv{s[2]}p{s[3]}t{s[5]}")
@pytest.mark.parametrize("kind,narrow", KINDS[:4], ids=lambda x: {True: "bf16", False: "f32"}.get(x, x))
def test_keys_reach_all_that_see_them(torch_gpu, shape, kind, narrow):
    """A NaN key makes every result of the tokens and heads that see it NaN, and no other one."""
    D, H, Hkv, P, rows, T, n_tok = shape
    rng, c, q, n_tok = setup(72 + T, TYPES[kind], D, H, Hkv, P, rows, T, n_tok, narrow)
    for b, (r, t) in enumerate(zip(rows, n_tok)):
        spoil(c, c.k, b, 3, 1, 9, NAN)
        spoil(c, c.k, b, r + t // 2, 0, 70, NAN)
    case_note(f"fa_chunk non-finite keys {kind} narrow={narrow} {shape}")
    par = Params(D**-0.5, 100)
    got, lse = on_gpu(torch_gpu, q, c, par, n_tok, narrow)
    out, wl_, tol, tol_lse = chunk_f64(q, c, n_tok, par, narrow)
    live = np.arange(T) < np.array(n_tok)[:, None]
    hit = np.isnan(wl_) & live[..., None]
    fine = ~hit & live[..., None]
    assert hit.any() and fine.any()
    assert np.all(np.isnan(lse[hit])) and np.all(np.isnan(got[hit]))
    assert np.all(np.abs(lse[fine] - wl_[fine]) <= tol_lse[fine]) and np.all(np.abs(got[fine] - out[fine]) <= tol[fine])
