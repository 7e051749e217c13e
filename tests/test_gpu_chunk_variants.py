"""Forms of the chunk operators that the ordinary sizes do not reach together: workgroups of 256 pairs under every mask, and row
weights of few and of many tokens under masks, caps and biases with either type of q."""
import numpy as np
import pytest

from chunk_cases import Params, chunk_f64, weights_f64
from conftest import case_note
from test_gpu_fa_chunk import on_gpu, setup
from test_gpu_fa_tree import TYPES, check
from test_gpu_kv_weights import check as check_weights, lse_of, on_gpu as weights_on_gpu

pytestmark = pytest.mark.gpu

MASKS = [
    # window, cap, bias, documents, prefix (a bias beside a prefix: test_gpu_chunk_distance.py)
    (1, 0.0, 0.0, False, False),
    (64, 30.0, 0.0, False, True),
    (0, 1.5, 8.0, True, False),
    (0, 0.0, 8.0, False, False),
    (130, 0.0, 0.0, True, True),
]
mask_id = lambda m: "w%d_cap%g_bias%g%s%s" % (m[0], m[1], m[2], "_docs" * m[3], "_prefix" * m[4])  # noqa: E731


def masks_of(rng, mask, rows, T):
    first = None
    if mask[3]:
        # documents: rising first rows, and tokens that see nothing (a first row behind their own)
        first = np.stack([np.sort(rng.integers(-3, r + T, T)) for r in rows])
        first[:, 2::7] = 1 << 20
    return first, [r // 2 + T - 2 for r in rows] if mask[4] else None


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("mask", MASKS, ids=mask_id)
def test_chunk_of_256_pairs_a_workgroup(torch_gpu, mask, kind, narrow):
    case_note(f"fa_chunk 256 pairs {mask} {kind} narrow={narrow}")
    rng, c, q, n_tok = setup(100, TYPES[kind], 128, 16, 16, 64, [200], 300, None, narrow)
    par = Params(128**-0.5, *mask[:3])
    first, prefix = masks_of(rng, mask, [200], 300)
    check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow, first, prefix), chunk_f64(q, c, n_tok, par, narrow, first, prefix))


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind,D,H,Hkv", [("f16", 128, 16, 4), ("q8_0", 256, 24, 4), ("q4_0", 128, 6, 2), ("e5m2", 256, 4, 4), ("q4_0", 256, 8, 2), ("f16", 256, 5, 5)])
@pytest.mark.parametrize("T", [1, 2, 40])
@pytest.mark.parametrize("mask", MASKS, ids=mask_id)
def test_weights_of_few_and_many_tokens(torch_gpu, mask, T, kind, D, H, Hkv, narrow):
    case_note(f"kv_weights {mask} T {T} {kind} {D} {H}/{Hkv} narrow={narrow}")
    rows, n_tok = [0, 100, 333], [T, (T + 1) // 2, T]
    rng, c, q, n_tok = setup(101 + T, TYPES[kind], D, H, Hkv, 16, rows, T, n_tok, narrow)
    par = Params(D**-0.5, *mask[:3])
    first, prefix = masks_of(rng, mask, rows, T)
    lse = lse_of(q, c, n_tok, par, narrow, first, prefix)
    cols = max(rows) + T
    scores = rng.random((3, cols)).astype(np.float32)
    want = weights_f64(q, c, n_tok, par, lse, scores, cols, 0.5, False, first, prefix)
    check_weights(weights_on_gpu(torch_gpu, q, c, par, n_tok, narrow, lse, scores, cols, 0.5, False, first, prefix), want)
