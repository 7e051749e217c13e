"""The chunk operators, eviction and verification on the host: what they refuse, and their workspace
sizes. No GPU: every call here is refused before a launch."""
import ctypes
import math

import numpy as np
import pytest

import xqattn
from chunk_cases import evict, seen, verify
from test_cpu_paged import BAD_ARG, BAD_SHAPE, DATA, OK, UNSUPPORTED, WORKSPACE, cache, tensor, tree_args, with_nb, with_ne
from xqattn import workloads as wl


def par(scale=0.1, **kw):
    p = xqattn.chunk_params(scale)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def call_chunk(q, c, d, p=None, first=None, prefix=None, n_tok=None, lse=None, ws=DATA, ws_bytes=1 << 40):
    return xqattn.load().xq_fa_chunk(ctypes.byref(q), ctypes.byref(c), ctypes.byref(p or par()), first, prefix, n_tok, ctypes.byref(d), lse,
                                     ws, ws_bytes, None)


def call_weights(q, c, p=None, first=None, prefix=None, n_tok=None, lse=DATA, scores=DATA, out=DATA, cols=100, decay=1.0, fresh=1, ws=DATA,
                 ws_bytes=1 << 40):
    return xqattn.load().xq_kv_weights(ctypes.byref(q), ctypes.byref(c), ctypes.byref(p or par()), first, prefix, n_tok, lse, scores, out,
                                       cols, decay, fresh, ws, ws_bytes, None)


BAD_PARAMS = [dict(scale=math.inf), dict(scale=math.nan), dict(logit_softcap=-1.0), dict(logit_softcap=math.nan), dict(logit_softcap=math.inf),
              dict(max_bias=-1.0), dict(max_bias=math.nan), dict(window=-1)]


def test_fa_chunk_refusals():
    lib = xqattn.load()

    def refused(want, q, c, d, **kw):
        assert call_chunk(q, c, d, **kw) == want, lib.xq_last_error()
        assert lib.xq_last_error()
        if not kw and want in (UNSUPPORTED, BAD_SHAPE) and q.data and c.k.data:
            assert not lib.xq_supports_fa_chunk(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d))

    q, c, d = tree_args(T=100)
    assert lib.xq_supports_fa_chunk(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d))
    long = cache(cols=200)  # in parts
    refused(WORKSPACE, q, long, d, ws=None)
    refused(WORKSPACE, q, long, d, ws_bytes=16)
    refused(WORKSPACE, q, long, d, ws=DATA + 16)
    for bad in BAD_PARAMS:
        refused(BAD_ARG, q, c, d, p=par(**bad))
    p = par()
    p.reserved[2] = 1
    refused(BAD_ARG, q, c, d, p=p)
    for kw in (dict(first=DATA + 2), dict(prefix=DATA + 1), dict(n_tok=DATA + 2), dict(lse=DATA + 2)):
        refused(UNSUPPORTED, q, c, d, **kw)
    for typ in (wl.F16, wl.Q8_0):
        q2, _, d2 = tree_args(typ)
        refused(UNSUPPORTED, q2, c, d2)
    for D in (64, 96, 512):
        refused(UNSUPPORTED, *tree_args(D=D, c=cache(D=D)))
    for typ in (wl.F32, wl.BF16):
        refused(UNSUPPORTED, q, cache(typ), d)
    refused(UNSUPPORTED, q, c, tree_args(wl.BF16, T=100)[2])
    refused(BAD_SHAPE, q, c, with_ne(tree_args(T=100)[2], 2, 99))
    refused(BAD_SHAPE, *tree_args(B=3))
    refused(BAD_SHAPE, *tree_args(H=6))
    refused(UNSUPPORTED, *tree_args(H=33, c=cache(Hkv=1)))
    refused(UNSUPPORTED, with_nb(tree_args(T=100)[0], 0, 8), c, d)
    refused(UNSUPPORTED, with_nb(tree_args(T=100)[0], 1, 514), c, d)
    refused(UNSUPPORTED, q, c, with_nb(tree_args(T=100)[2], 1, 8 * 128 * 4 + 4))
    big = cache()
    big.k.nb[3] = 1 << 32
    refused(UNSUPPORTED, q, big, d)
    refused(UNSUPPORTED, *tree_args(T=1 << 24))
    refused(UNSUPPORTED, *tree_args(T=1, H=1, B=1 << 23, c=cache(Hkv=1, n_seq=1 << 23)))
    refused(BAD_ARG, q, cache(table=None), d)
    refused(BAD_ARG, q, cache(table_cols=0), d)
    q.data = None
    refused(BAD_ARG, q, c, d)


def test_kv_weights_refusals():
    lib = xqattn.load()

    def refused(want, q, c, **kw):
        assert call_weights(q, c, **kw) == want, lib.xq_last_error()
        assert lib.xq_last_error()

    q, c, _ = tree_args(T=100)
    refused(WORKSPACE, q, c, ws=None)
    refused(WORKSPACE, q, c, ws_bytes=16)
    refused(WORKSPACE, q, c, ws=DATA + 16)
    for bad in BAD_PARAMS:
        refused(BAD_ARG, q, c, p=par(**bad))
    for kw in (dict(lse=None), dict(out=None), dict(cols=0), dict(decay=math.nan), dict(decay=math.inf), dict(fresh=2)):
        refused(BAD_ARG, q, c, **kw)
    for kw in (dict(lse=DATA + 2), dict(out=DATA + 2), dict(scores=DATA + 1), dict(first=DATA + 2)):
        refused(UNSUPPORTED, q, c, **kw)
    refused(UNSUPPORTED, tree_args(wl.F16)[0], c)
    refused(UNSUPPORTED, q, cache(wl.BF16))
    refused(UNSUPPORTED, tree_args(T=1, H=1, B=65536)[0], cache(Hkv=1, n_seq=65536))


def test_workspaces_follow_the_shapes():
    lib = xqattn.load()
    n = ctypes.c_size_t(0)
    q, c, d = tree_args(T=100)
    assert lib.xq_fa_chunk_workspace(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d), None) == BAD_ARG
    assert lib.xq_kv_weights_workspace(ctypes.byref(q), ctypes.byref(c), None) == BAD_ARG
    # a prompt that fills the card needs no parts
    q, c, d = tree_args(wl.BF16, T=8191, H=32, c=cache(Hkv=8, pages=1000, cols=512))
    assert lib.xq_fa_chunk_workspace(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d), ctypes.byref(n)) == OK and n.value == 0
    assert lib.xq_kv_weights_workspace(ctypes.byref(q), ctypes.byref(c), ctypes.byref(n)) == OK and n.value >= 2 * 8191 * 32 * 128 * 2
    assert lib.xq_kv_pages_evict_workspace(3, 0, ctypes.byref(n)) == BAD_ARG
    assert lib.xq_kv_pages_evict_workspace(3, 1000, ctypes.byref(n)) == OK and n.value >= 3 * 500 * 24
    assert lib.xq_verify_tokens_workspace(ctypes.byref(tensor(wl.F32, (1000, 65, 2, 1))), ctypes.byref(n)) == UNSUPPORTED


def pools(n=2, typ=wl.F16, D=128, P=16, Hkv=4, pages=10, step=1 << 20):
    return (xqattn.XqTensor * n)(*[tensor(typ, (D, P, Hkv, pages), data=DATA + i * step) for i in range(n)])


def test_evict_refusals():
    lib = xqattn.load()

    def refused(want, ps=None, table=DATA, rows=DATA, refs=DATA, n_seq=2, cols=3, keep=DATA, first=0, last=0, scores=DATA, positions=None,
                score_cols=48, scores_out=None, positions_out=None, rows_out=DATA + 64, ws=DATA, ws_bytes=1 << 40):
        ps = pools() if ps is None else ps
        got = lib.xq_kv_pages_evict(ps, len(ps), table, rows, refs, n_seq, cols, keep, first, last, scores, positions, score_cols, scores_out,
                                    positions_out, rows_out, ws, ws_bytes, None)
        assert got == want, lib.xq_last_error()
        assert lib.xq_last_error()

    for kw in (dict(table=None), dict(rows=None), dict(keep=None), dict(scores=None), dict(rows_out=None), dict(rows_out=DATA), dict(n_seq=0),
               dict(cols=0), dict(score_cols=0), dict(first=-1), dict(last=-1), dict(ps=pools(2, step=0))):
        refused(BAD_ARG, **kw)
    for kw in (dict(n_seq=65536), dict(score_cols=(1 << 30) + 1), dict(scores=DATA + 2), dict(positions=DATA + 1), dict(refs=DATA + 2),
               dict(ps=pools(D=48))):
        refused(UNSUPPORTED, **kw)
    for kw in (dict(ws=None), dict(ws_bytes=64), dict(ws=DATA + 8)):
        refused(WORKSPACE, **kw)


def test_verify_refusals():
    lib = xqattn.load()

    def logits(typ=wl.F32, V=1000, T=5, B=2):
        return tensor(typ, (V, T, B, 1))

    def refused(want, l=None, q=None, tokens=DATA, parents=None, n_tok=None, heat=None, u=DATA, path=DATA, n_path=DATA, nxt=DATA, logp=None,
                ws=DATA, ws_bytes=1 << 40):
        l = logits() if l is None else l
        got = lib.xq_verify_tokens(ctypes.byref(l), None if q is None else ctypes.byref(q), tokens, parents, n_tok, heat, u, path, n_path, nxt,
                                   logp, ws, ws_bytes, None)
        assert got == want, lib.xq_last_error()
        assert lib.xq_last_error()

    for kw in (dict(tokens=None), dict(path=None), dict(n_path=None), dict(nxt=None), dict(q=logits(), u=None)):
        refused(BAD_ARG, **kw)
    for kw in (dict(l=logits(wl.F16)), dict(l=logits(T=65)), dict(l=logits(V=(1 << 24) + 1)), dict(l=logits(B=65536)), dict(q=logits(wl.BF16)),
               dict(q=logits(), parents=DATA), dict(tokens=DATA + 2), dict(u=DATA + 1), dict(logp=DATA + 2), dict(l=with_nb(logits(), 0, 8)),
               dict(l=with_nb(logits(), 1, 4002))):
        refused(UNSUPPORTED, **kw)
    for kw in (dict(q=logits(V=999)), dict(q=logits(T=4)), dict(l=with_ne(logits(), 3, 2)), dict(l=with_ne(logits(), 2, 0))):
        refused(BAD_SHAPE, **kw)
    for kw in (dict(ws=None), dict(ws_bytes=64), dict(ws=DATA + 8)):
        refused(WORKSPACE, **kw)


def test_binding_checks_shapes():
    torch = pytest.importorskip("torch")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    l = xqattn.DevTensor(wl.F32, (1000, 5, 2, 1), (4, 4000, 20000, 40000), torch.zeros(10000))
    with pytest.raises(ValueError, match="tokens"):
        xqattn.verify_tokens(l, i32(9), i32(10), i32(2), i32(2))
    with pytest.raises(ValueError, match="uniform"):
        xqattn.verify_tokens(l, i32(10), i32(10), i32(2), i32(2), uniform=torch.zeros(11))
    with pytest.raises(ValueError, match="device tensors"):
        xqattn.verify_tokens(l, i32(10), i32(10), i32(2), i32(2))
    with pytest.raises(ValueError, match="scores"):
        xqattn.kv_pages_evict([l], i32(2, 3), i32(2), None, i32(2), torch.zeros(3, 10), i32(2))
    with pytest.raises(ValueError, match="positions"):
        xqattn.kv_pages_evict([l], i32(2, 3), i32(2), None, i32(2), torch.zeros(2, 10), i32(2), positions=i32(2, 9))


def test_oracle_masks_and_walks():
    """The oracle against cases worked out by hand."""
    s = seen(3, 2, 5, 2, None, None)
    assert np.array_equal(s, [[0, 0, 1, 1, 0], [0, 0, 0, 1, 1]])
    assert np.array_equal(seen(3, 2, 5, 0, [4, 0], 5), [[0, 0, 0, 0, 1], [1, 1, 1, 1, 1]])
    # rows 0..5 with a budget of 3: row 0 is protected, then 4 and 3 by weight; 3 and 4 go to 1 and 2
    table, refs, rows, moves, order = evict(np.array([[2, 0, 1]], np.int32), np.array([6], np.int32), np.array([1, 1, 1], np.int32), [3], 1, 0,
                                            np.array([[0.0, 1, 2, 3, 4, 3]], np.float32), None, 2, 3)
    assert order == [[0, 3, 4]] and rows.tolist() == [3] and refs.tolist() == [1, 0, 1] and table.tolist() == [[2, 0, -1]]
    assert moves == [(0, (0, 1), (2, 1)), (0, (1, 0), (0, 0))]
    # two children of the root: the first has p 1/2 and is rejected by u = 0.6, the second has half of what is left
    l = np.log(np.array([[[0.5, 0.25, 0.25]] * 3]))
    path, n, nxt, _ = verify(l, np.array([[0, 0, 1]]), np.array([[-1, 0, 0]]), [3], None, np.array([[0, 0.6, 0.49, 0.9]]))
    assert path.tolist() == [[0, 2, -1]] and n.tolist() == [2] and nxt.tolist() == [2]
    path, n, nxt, _ = verify(l, np.array([[0, 0, 1]]), np.array([[-1, 0, 0]]), [3], None, np.array([[0, 0.6, 0.51, 0.9]]))
    assert n.tolist() == [1] and nxt.tolist() == [2]
