"""Row weights from the lse of the tree operator: over a chain all rows get their weights, over a tree the rows that
the sequences held before it."""
import numpy as np
import pytest

from chunk_cases import Params, weights_f64
from conftest import case_note
from paged_cases import random_parents
from test_gpu_fa_chunk import setup
from test_gpu_fa_tree import TYPES, on_gpu as tree_on_gpu
from test_gpu_kv_weights import on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("T", [1, 4, 33])
def test_weights_from_the_trees_lse(torch_gpu, T, kind, narrow):
    H, rows, n_tok = 16, [333, 0, 20], [T, T, (T + 1) // 2]
    rng, c, q, n_tok = setup(90 + T, TYPES[kind], 128, H, 8, 16, rows, T, n_tok, narrow)
    par, cols = Params(128**-0.5), 333 + T
    scores = rng.random((3, cols)).astype(np.float32)
    tree = np.stack([random_parents(rng, T) for _ in rows])
    for parents in (None, tree):
        case_note(f"kv_weights from fa_tree's lse {kind} narrow={narrow} T {T} {'chain' if parents is None else 'tree'}")
        _, lse = tree_on_gpu(torch_gpu, q, c, parents, n_tok, par.scale, narrow)
        got = on_gpu(torch_gpu, q, c, par, n_tok, narrow, lse, scores, cols, 0.5)
        want, tol = weights_f64(q, c, n_tok, par, lse, scores, cols, 0.5, True)
        for b, (r, t) in enumerate(zip(rows, n_tok)):
            n = r + t if parents is None else r
            assert np.all(np.abs(got[b, :n] - want[b, :n]) <= tol[b, :n])
            if parents is None:
                # A token's weights are 1 in all, but for the scores' errors on both sides: |q|.|k| scale is up to 9 here, times 2^-21 and
                # 136 * 2^-24 each. Beside BF16 q the attention has quantized keys rounded to f16 (2^-11), and these weights have not.
                own = got[b, :n].astype(np.float64).copy()
                own[:r] -= 0.5 * scores[b, :r]
                assert abs(own.sum() - H * t) <= H * t * (2.0**-6 if narrow and kind in ("q8_0", "q4_0") else 2.0**-12) + n * 2.0**-23
            else:
                assert np.all(got[b, r + t:] == -7.0)
