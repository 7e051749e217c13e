"""Verification of drafted tokens from given random numbers, against the walk in float64."""
import numpy as np
import pytest

import xqattn
from chunk_cases import verify
from conftest import case_note
from paged_cases import bf16, random_parents
from xqattn import workloads as wl

pytestmark = pytest.mark.gpu


def rows3(torch, x, typ):
    """[B, T, V] device tensor -> [V, T, B] descriptor."""
    es = x.element_size()
    B, T, V = x.shape
    return xqattn.DevTensor(typ, (V, T, B, 1), (es, x.stride(1) * es, x.stride(0) * es, B * x.stride(0) * es), x)


def on_gpu(torch, logits, tokens, parents, n_tok, heat, u, draft=None, narrow=False, stream=None, wide=0):
    dt, typ = (torch.bfloat16, wl.BF16) if narrow else (torch.float32, wl.F32)
    B, T, V = logits.shape

    def rows(x):
        if x is None:
            return None
        y = torch.full((B, T, V + wide), 1e30, dtype=dt, device="cuda")[..., :V]
        y.copy_(torch.from_numpy(x))
        return rows3(torch, y, typ)

    def dev(x, t):
        return None if x is None else torch.from_numpy(np.ascontiguousarray(x, t)).cuda()

    path, n_path, nxt = (torch.full(s, 77, dtype=torch.int32, device="cuda") for s in ((B, T), (B,), (B,)))
    logp = torch.full((B, T + 1), 77.0, device="cuda")
    args = rows(logits), dev(tokens, np.int32), path, n_path, nxt, dev(u, np.float32), rows(draft), dev(parents, np.int32), dev(n_tok, np.int32), dev(heat, np.float32), logp
    torch.cuda.synchronize()
    xqattn.verify_tokens(*args, stream=stream)
    torch.cuda.synchronize()
    return path.cpu().numpy(), n_path.cpu().numpy(), nxt.cpu().numpy(), logp.cpu().numpy()


def check(got, want, V, biggest):
    """Whole numbers are equal. logp: f32 exponentials (2^-22 and the argument's 2^-23 of it) and their sums over
    up to V / 256 terms a lane, a logarithm, one rounding."""
    for a, b, what in zip(got[:3], want[:3], ("path", "n_path", "next")):
        assert np.array_equal(a, b), f"{what}: {a.tolist()} for {b.tolist()}"
    a, b = got[3], want[3]
    fin = np.isfinite(b)
    assert np.array_equal(a[~fin], b[~fin])
    tol = 2.0**-21 + biggest * 2.0**-22 + 48 * 2.0**-24 + np.abs(b[fin]) * 2.0**-23
    assert np.all(np.abs(a[fin] - b[fin]) <= tol), f"logp off by {np.abs(a[fin] - b[fin]).max():.3e}"


def setup(seed, B, T, V, sharp=2.0, narrow=False, chain=False):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((B, T, V)) * sharp).astype(np.float32)
    x = bf16(x) if narrow else x
    parents = None if chain else np.stack([random_parents(rng, T) for _ in range(B)])
    up = np.tile(np.arange(-1, T - 1), (B, 1)) if chain else parents
    tokens = rng.integers(0, V, (B, T))
    for b in range(B):
        for c in range(1, T):
            p = max(0, int(up[b, c]))
            k = int((up[b, :c] == up[b, c]).sum())
            if rng.random() < 0.85:
                tokens[b, c] = np.argsort(-x[b, p], kind="stable")[min(k, V - 1)]
    return rng, x, tokens.astype(np.int32), parents


SHAPES = [(1, 1, 1), (2, 2, 3), (3, 5, 100), (1, 64, 513), (4, 25, 8192), (2, 8, 8193), (2, 7, 20001), (40, 3, 64)]


@pytest.mark.parametrize("narrow", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("mode", ["greedy", "target", "chain", "draft", "mixed"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "b%dt%dv%d" % s)
def test_walks(torch_gpu, shape, mode, narrow):
    B, T, V = shape
    case_note(f"verify_tokens {mode} {shape} narrow={narrow}")
    for seed in range(3):
        rng, x, tokens, parents = setup(100 * seed + T, B, T, V, (1.0, 3.0, 8.0)[seed], narrow, mode in ("chain", "draft"))
        heat = rng.uniform(0.3, 1.5, B).astype(np.float32)
        if mode == "mixed":
            heat[::2] = (0.0, -1.0, np.float32(np.nan))[seed]
        u = None if mode == "greedy" else rng.random((B, T + 1)).astype(np.float32)
        n_tok = rng.integers(0, T + 1, B).astype(np.int32)
        n_tok[0] = T
        draft = None
        if mode == "draft":
            y = x.astype(np.float64) + rng.standard_normal(x.shape)
            draft = np.exp(y - y.max(-1, keepdims=True))
            draft = (draft / draft.sum(-1, keepdims=True)).astype(np.float32)
            draft = bf16(draft) if narrow else draft
            for b in range(B):
                for c in range(1, T):
                    tokens[b, c] = rng.choice(V, p=draft[b, c - 1].astype(np.float64) / draft[b, c - 1].astype(np.float64).sum())
        want = verify(x, tokens, parents, n_tok, heat, u, draft)
        got = on_gpu(torch_gpu, x, tokens, parents, n_tok, heat, u, draft, narrow, wide=seed)
        check(got, want, V, np.abs(x).max() * 2 / 0.3)
        assert seed or mode == "greedy" or T < 5 or (want[1] > 0).any()


def test_token_zero_alone_and_nothing(torch_gpu):
    rng, x, tokens, parents = setup(1, 3, 4, 50)
    u = rng.random((3, 5)).astype(np.float32)
    case_note("verify_tokens n_tok 0, 1, above n_q")
    want = verify(x, tokens, parents, [0, 1, 4], None, u)
    check(on_gpu(torch_gpu, x, tokens, parents, [-2, 1, 9], None, u), want, 50, 20)
    assert want[2][0] == -1 and want[1].tolist()[:2] == [0, 1]


def test_bad_parents_and_tokens_are_never_reached(torch_gpu):
    rng, x, tokens, parents = setup(2, 4, 12, 200)
    parents[0] = [-1, 0, 1, 7, 12, 4, -5, 1 << 30, 2, 8, 9, 10]
    tokens[1, 1:] = [-1, 200, 1 << 30, -(1 << 31)] + [5] * 7
    u = np.zeros((4, 13), np.float32)
    u[:, -1] = 0.5
    case_note("verify_tokens bad parents and tokens")
    want_parents = parents.copy()
    bad = (want_parents < 0) | (want_parents >= np.arange(12))
    want_parents[bad] = -1
    check(on_gpu(torch_gpu, x, tokens, parents, [12] * 4, None, u), verify(x, tokens, want_parents, [12] * 4, None, u), 200, 20)


def test_siblings_with_the_same_token(torch_gpu):
    """A token that is tried again has no mass left, whatever the number."""
    x = np.log(np.array([0.6, 0.2, 0.1, 0.1], np.float32))[None, None].repeat(6, 1).repeat(50, 0)
    tokens = np.tile(np.array([0, 1, 1, 0, 1, 2], np.int32), (50, 1))
    parents = np.tile(np.array([-1, 0, 0, 0, 0, 0], np.int32), (50, 1))
    u = np.random.default_rng(5).random((50, 7)).astype(np.float32)
    case_note("verify_tokens same token twice")
    want = verify(x, tokens, parents, [6] * 50, None, u)
    assert {tuple(p[:2]) for p in want[0].tolist()} >= {(0, 1), (0, 3), (0, 5), (0, -1)} and not {2, 4} & set(want[0].ravel().tolist())
    check(on_gpu(torch_gpu, x, tokens, parents, [6] * 50, None, u), want, 4, 10)


def test_ties_infinities_and_nan(torch_gpu):
    """The lowest index of equal maxima; NaN as -inf; +inf shares the mass; rows without any; nothing next."""
    V = 9000
    x = np.full((7, 2, V), -2.0, np.float32)
    x[0, :, [5, 8500]] = 4.0
    x[1, :, 100:] = -np.inf
    x[2, :, 0:50] = np.nan
    x[3, :, [7, 8999]] = np.inf
    x[4] = -np.inf
    x[5] = np.nan
    x[6, 0], x[6, 1] = np.inf, -np.inf
    tokens = np.array([[0, 5], [0, 200], [0, 60], [0, 7], [0, 3], [0, 3], [0, 11]], np.int32)
    rng = np.random.default_rng(6)
    for u in (None, np.full((7, 3), 0.0, np.float32), np.full((7, 3), 1.0 - 2.0**-24, np.float32), rng.random((7, 3)).astype(np.float32)):
        for narrow in (False, True):
            case_note(f"verify_tokens infinities u={None if u is None else u[0]} narrow={narrow}")
            want = verify(x, tokens, None, [2] * 7, None, u)
            check(on_gpu(torch_gpu, x, tokens, None, [2] * 7, None, u, narrow=narrow), want, V, 10)


def test_draft_that_equals_the_target_and_numbers_at_the_ends(torch_gpu):
    """max(p - q, 0) without mass gives p; u of 0, of next to 1, NaN and above 1."""
    V = 300
    rng = np.random.default_rng(8)
    p = np.zeros((4, 3, V), np.float32)
    p[..., :4] = 0.25
    with np.errstate(divide="ignore"):
        x = np.log(p)
    tokens = np.array([[0, 7, 1]] * 4, np.int32)  # 7 has no mass: rejected, and p - q is 0 everywhere
    u = np.array([[0.5, 0.5, 0.5, 0.0], [0.5, 0.5, 0.5, 0.26], [0.5, 0.5, 0.5, 0.99], [0.5, 0.5, 0.5, 0.5]], np.float32)
    case_note("verify_tokens draft equals target")
    want = verify(x, tokens, None, [3] * 4, None, u, p)
    assert want[2].tolist() == [0, 1, 3, 2] and want[1].tolist() == [1] * 4
    check(on_gpu(torch_gpu, x, tokens, None, [3] * 4, None, u, p), want, V, 10)
    u[:, 3] = [np.nan, -1.0, 1.0, 7.0]
    got = on_gpu(torch_gpu, x, tokens, None, [3] * 4, None, u, p)
    assert got[2].tolist() == [0, 0, 3, 3]


def test_temperatures_at_the_ends(torch_gpu):
    rng, x, tokens, _ = setup(9, 4, 3, 500, chain=True)
    x[:, :, 10:20] = -np.inf
    heat = np.array([1e-30, 1e-3, 1e4, np.inf], np.float32)
    u = rng.random((4, 4)).astype(np.float32)
    case_note("verify_tokens temperatures")
    want = verify(x, tokens, None, [3] * 4, np.minimum(heat, 1e30), u)
    got = on_gpu(torch_gpu, x, tokens, None, [3] * 4, heat, u)
    for a, b in zip(got[:3], want[:3]):
        assert np.array_equal(a, b)


def test_distribution_of_what_stands(torch_gpu):
    """Over many draws the first drawn token of chain and tree is the target's distribution: the counts of
    20 000 walks within 5 standard deviations."""
    n, V = 20000, 4
    p = np.array([0.5, 0.3, 0.15, 0.05])
    rng = np.random.default_rng(10)
    x = np.log(p).astype(np.float32)[None, None].repeat(3, 1).repeat(n, 0)
    u = rng.random((n, 4)).astype(np.float32)
    parents = np.tile(np.array([-1, 0, 0], np.int32), (n, 1))
    tokens = np.tile(np.array([0, 1, 3], np.int32), (n, 1))
    q = np.array([0.1, 0.6, 0.1, 0.2], np.float32)
    drawn = np.concatenate([np.zeros((n, 1), np.int64), rng.choice(V, (n, 2), p=q.astype(np.float64) / q.astype(np.float64).sum())], 1)
    for name, args in (("tree", (tokens, parents, None)), ("draft", (drawn, None, q[None, None].repeat(3, 1).repeat(n, 0)))):
        case_note(f"verify_tokens distribution, {name}")
        t, up, d = args
        path, n_path, nxt, _ = on_gpu(torch_gpu, x, t, up, [3] * n, None, u, d)
        first = np.where(n_path > 1, np.take_along_axis(np.asarray(t), np.maximum(path[:, 1:2], 0), 1)[:, 0], nxt)
        count = np.bincount(first, minlength=V)
        assert np.all(np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p))), count


def test_replays_and_streams(torch_gpu):
    torch = torch_gpu
    B, T, V = 3, 6, 9001
    path, n_path, nxt = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((B, T), (B,), (B,)))
    logp = torch.zeros((B, T + 1), device="cuda")
    lg, tk, up = torch.zeros((B, T, V), device="cuda"), torch.zeros((B, T), dtype=torch.int32, device="cuda"), torch.zeros((B, T), dtype=torch.int32, device="cuda")
    u, heat, tn = torch.zeros((B, T + 1), device="cuda"), torch.ones(B, device="cuda"), torch.full((B,), T, dtype=torch.int32, device="cuda")
    args = (rows3(torch, lg, wl.F32), tk, path, n_path, nxt, u, None, up, tn, heat, logp)
    case_note("verify_tokens capture")
    ws = xqattn.verify_tokens(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xqattn.verify_tokens(*args, workspace=ws)
    side = torch.cuda.Stream()
    for seed in range(4):
        rng, x, tokens, parents = setup(60 + seed, B, T, V)
        lg.copy_(torch.from_numpy(x)), tk.copy_(torch.from_numpy(tokens)), up.copy_(torch.from_numpy(parents))
        un = rng.random((B, T + 1)).astype(np.float32)
        u.copy_(torch.from_numpy(un)), heat.copy_(torch.tensor([0.0, 0.7, 1.0]))
        path.fill_(5), n_path.fill_(5), nxt.fill_(5), logp.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (path, n_path, nxt, logp)]
        check([t.cpu().numpy() for t in got], verify(x, tokens, parents, [T] * B, np.array([0.0, 0.7, 1.0], np.float32), un), V, 40)
        path.fill_(6), n_path.fill_(6), nxt.fill_(6), logp.fill_(6.0)
        torch.cuda.synchronize()
        xqattn.verify_tokens(*args, stream=side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (path, n_path, nxt, logp)))
