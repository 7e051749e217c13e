"""Verification where the oracle's own answers are known to hold what the cases are for: drafted tokens that stand, tokens
that are rejected, and a next token from what is left after that."""
import numpy as np
import pytest

from chunk_cases import verify
from conftest import case_note
from paged_cases import bf16
from test_gpu_verify_tokens import check, on_gpu, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("mode", ["greedy", "target", "chain", "draft"])
@pytest.mark.parametrize("shape", [(24, 12, 700), (12, 40, 9000)], ids=lambda s: "b%dt%dv%d" % s)
def test_some_stand_and_some_do_not(torch_gpu, shape, mode, narrow):
    B, T, V = shape
    rng, x, tokens, parents = setup(7 * T, B, T, V, 6.0, narrow, mode in ("chain", "draft"))
    heat = None if mode == "greedy" else rng.uniform(0.5, 1.2, B).astype(np.float32)
    u = None if mode == "greedy" else rng.random((B, T + 1)).astype(np.float32)
    n_tok = rng.integers(2, T + 1, B).astype(np.int32)
    draft = None
    if mode == "draft":
        y = x.astype(np.float64) + 0.5 * rng.standard_normal(x.shape)
        draft = np.exp(y - y.max(-1, keepdims=True))
        draft = (draft / draft.sum(-1, keepdims=True)).astype(np.float32)
        draft = bf16(draft) if narrow else draft
        for b in range(B):
            for c in range(1, T):
                tokens[b, c] = rng.choice(V, p=draft[b, c - 1].astype(np.float64) / draft[b, c - 1].astype(np.float64).sum())
    want = verify(x, tokens, parents, n_tok, heat, u, draft)
    path, n_path, nxt, _ = want
    up = np.tile(np.arange(-1, T - 1), (B, 1)) if parents is None else parents
    last = path[np.arange(B), n_path - 1]
    kids = np.array([(up[b, 1:n_tok[b]] == last[b]).any() for b in range(B)])
    assert (n_path > 2).any() and kids.any() and (n_path[kids] > 1).any()
    assert mode == "greedy" or len(set(nxt)) > 2
    case_note(f"verify_tokens {mode} {shape} narrow={narrow}: {n_path.tolist()}")
    check(on_gpu(torch_gpu, x, tokens, parents, n_tok, heat, u, draft, narrow), want, V, np.abs(x).max() * 2 / 0.5)
