"""Caps of the scores at the ends of f32: a score of 0 stays 0 however small the cap, and a cap far above the scores does nothing."""
import numpy as np
import pytest

from chunk_cases import Params, chunk_f64, weights_f64
from conftest import case_note
from test_gpu_fa_chunk import on_gpu, setup
from test_gpu_fa_tree import check
from test_gpu_kv_weights import check as check_weights, on_gpu as weights_on_gpu
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu

# 2^-149 and 2^-130 are subnormal (their reciprocals are beyond f32), 2^-126 the smallest normal number
CAPS = [2.0**-149, 2.0**-130, 2.0**-126, 1e-30, 2.0**-10, 1e6, 2.0**127]


@pytest.mark.parametrize("cap", CAPS, ids=lambda c: "%.0e" % c)
@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 20, 150])
def test_caps(torch_gpu, T, narrow, cap):
    rng, c, q, n_tok = setup(80 + T, wl.F16, 128, 16, 4, 16, [70, 300], T, None, narrow)
    q[:, :, ::2] = 0.0  # every other head: scores of 0
    par = Params(128**-0.5, 0, cap, 0.0)
    case_note(f"fa_chunk cap {cap} T {T} narrow={narrow}")
    want = chunk_f64(q, c, n_tok, par, narrow)
    assert np.isfinite(want[0]).all()
    check(*on_gpu(torch_gpu, q, c, par, n_tok, narrow), want)
    case_note(f"kv_weights cap {cap} T {T} narrow={narrow}")
    cols = 300 + T
    lse = want[1].astype(np.float32)
    check_weights(weights_on_gpu(torch_gpu, q, c, par, n_tok, narrow, lse, None, cols), weights_f64(q, c, n_tok, par, lse, None, cols, 1.0, True))
