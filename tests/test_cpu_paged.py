"""The paged entry points on the host: what they refuse, and their workspace sizes. No GPU: every
call here is refused before a launch."""
import ctypes

import numpy as np
import pytest

import xqattn
from paged_cases import Cache, Pages, ancestors
from xqattn import workloads as wl

OK, UNSUPPORTED, BAD_SHAPE, BAD_ARG, WORKSPACE = 0, 1, 2, 3, 4
DATA = 0x10000  # a pointer that is never followed


def tensor(typ, ne, nb=None, data=DATA):
    t = xqattn.XqTensor()
    t.type, t.data = typ, data
    if nb is None:
        nb = [wl.TYPE_SIZE[typ], wl.record_bytes(typ, ne[0])]
        nb += [nb[1] * ne[1], nb[1] * ne[1] * ne[2]]
    for i in range(4):
        t.ne[i], t.nb[i] = ne[i], nb[i]
    return t


def cache(typ=wl.F16, D=128, P=16, Hkv=4, pages=10, n_seq=2, cols=3, **over):
    c = xqattn.XqKvPages()
    c.k, c.v = tensor(typ, (D, P, Hkv, pages)), tensor(typ, (D, P, Hkv, pages))
    c.table, c.rows, c.n_seq, c.table_cols = DATA, DATA, n_seq, cols
    for name, v in over.items():
        setattr(c, name, v)
    return c


def tree_args(typ=wl.F32, D=128, T=4, H=8, B=2, c=None):
    return tensor(typ, (D, T, H, B)), c or cache(), tensor(typ, (D, H, T, B))


def call_tree(q, c, d, scale=0.1, parents=None, n_tok=None, lse=None, ws=DATA, ws_bytes=1 << 40):
    return xqattn.load().xq_fa_tree(ctypes.byref(q), ctypes.byref(c), parents, n_tok, ctypes.byref(d), lse, scale, ws, ws_bytes, None)


def with_nb(t, i, v):
    t.nb[i] = v
    return t


def with_ne(t, i, v):
    t.ne[i] = v
    return t


def test_fa_tree_refusals():
    lib = xqattn.load()

    def refused(want, q, c, d, **kw):
        assert call_tree(q, c, d, **kw) == want, lib.xq_last_error()
        assert lib.xq_last_error()
        if not kw and want in (UNSUPPORTED, BAD_SHAPE) and q.data and c.k.data:
            assert lib.xq_supports_fa_tree(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d)) == 0

    q, c, d = tree_args()
    assert lib.xq_supports_fa_tree(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d)) == 1
    assert lib.xq_supports_fa_tree(None, ctypes.byref(c), ctypes.byref(d)) == 0
    refused(UNSUPPORTED, *tree_args(wl.F16))
    refused(UNSUPPORTED, tensor(wl.F32, (128, 4, 8, 2)), cache(), tensor(wl.BF16, (128, 8, 4, 2)))
    refused(UNSUPPORTED, *tree_args(D=64, c=cache(D=64)))
    refused(UNSUPPORTED, *tree_args(T=65))
    refused(BAD_SHAPE, *tree_args(T=0))
    refused(BAD_SHAPE, q, c, tensor(wl.F32, (128, 4, 8, 2)))
    refused(BAD_SHAPE, *tree_args(H=6))                        # 6 heads over 4
    refused(UNSUPPORTED, *tree_args(H=33, c=cache(Hkv=1)))     # a group of 33
    refused(BAD_SHAPE, *tree_args(c=cache(D=256)))
    refused(BAD_SHAPE, *tree_args(c=cache(n_seq=3)))
    refused(BAD_ARG, *tree_args(c=cache(cols=0)))
    for t in (wl.F32, wl.BF16, 77):
        refused(UNSUPPORTED, *tree_args(c=cache(typ=t) if t != 77 else cache(k=with_type(77), v=with_type(77))))
    refused(UNSUPPORTED, *tree_args(c=cache(v=tensor(wl.Q8_0, (128, 16, 4, 10)))))
    refused(BAD_SHAPE, *tree_args(c=cache(v=tensor(wl.F16, (128, 16, 4, 11)))))
    refused(BAD_SHAPE, *tree_args(c=cache(pages=0)))
    refused(UNSUPPORTED, *tree_args(c=cache(k=with_nb(tensor(wl.F16, (128, 16, 4, 10)), 0, 4))))
    refused(UNSUPPORTED, *tree_args(c=cache(k=with_nb(tensor(wl.F16, (128, 16, 4, 10)), 1, 257))))
    refused(UNSUPPORTED, with_nb(tree_args()[0], 0, 8), c, d)
    refused(UNSUPPORTED, with_nb(tree_args()[0], 1, 514), c, d)
    refused(UNSUPPORTED, q, c, with_nb(tree_args()[2], 1, 520))
    refused(UNSUPPORTED, q, c, tensor(wl.F32, (128, 8, 4, 2), data=DATA + 8))
    refused(BAD_ARG, q, cache(table=None), d)
    refused(BAD_ARG, q, cache(rows=None), d)
    refused(BAD_ARG, tensor(wl.F32, (128, 4, 8, 2), data=None), c, d)
    for bad in (float("nan"), float("inf"), -float("inf")):
        refused(BAD_ARG, q, c, d, scale=bad)
    refused(UNSUPPORTED, q, c, d, parents=DATA + 2)
    refused(UNSUPPORTED, q, c, d, lse=DATA + 1)
    n = ctypes.c_size_t(0)
    assert lib.xq_fa_tree_workspace(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d), ctypes.byref(n)) == OK and n.value > 0
    assert lib.xq_fa_tree_workspace(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d), None) == BAD_ARG
    refused(WORKSPACE, q, c, d, ws=None)
    refused(WORKSPACE, q, c, d, ws_bytes=n.value - 1)
    refused(WORKSPACE, q, c, d, ws=DATA + 128)


def with_type(t):
    x = tensor(wl.F16, (128, 16, 4, 10))
    x.type = t
    return x


def test_qk_norm_rope_refusals():
    lib = xqattn.load()

    def args(typ=wl.F32, D=128, T=4, H=8, Hkv=4, B=2, out=None):
        return [tensor(typ, (D, T, h, B)) for h in (H, Hkv, Hkv)] + [tensor(typ if out is None else out, (D, T, H, B))]

    def refused(want, a, c=None, p=None, positions=DATA, **kw):
        c, p = c or cache(), p or xqattn.rope_params(64, 1e4)
        r = [ctypes.byref(x) for x in a]
        st = lib.xq_qk_norm_rope(r[0], r[1], r[2], positions, kw.get("n_tok"), kw.get("qw"), kw.get("kw"), kw.get("ff"), ctypes.byref(p),
                                 r[3], ctypes.byref(c), None)
        assert st == want and lib.xq_last_error(), (st, lib.xq_last_error())

    a, c, p = args(), cache(), xqattn.rope_params(64, 1e4)
    assert lib.xq_supports_qk_norm_rope(*map(ctypes.byref, a[:3]), ctypes.byref(p), ctypes.byref(a[3]), ctypes.byref(c)) == 1
    refused(UNSUPPORTED, args(wl.F16))
    refused(UNSUPPORTED, args(out=wl.F16))
    refused(UNSUPPORTED, [a[0], tensor(wl.BF16, (128, 4, 4, 2)), a[2], a[3]])
    refused(UNSUPPORTED, args(D=96), cache(D=96))
    refused(BAD_SHAPE, args(T=0))
    refused(BAD_SHAPE, [a[0], a[1], tensor(wl.F32, (128, 4, 5, 2)), a[3]])
    refused(BAD_SHAPE, [a[0], a[1], a[2], tensor(wl.F32, (128, 8, 4, 2))])
    refused(BAD_SHAPE, a, cache(Hkv=8))
    refused(BAD_SHAPE, a, cache(n_seq=1))
    refused(UNSUPPORTED, [with_nb(args()[0], 0, 8)] + a[1:])
    refused(UNSUPPORTED, [with_nb(args()[0], 2, 514)] + a[1:])
    refused(UNSUPPORTED, a[:3] + [with_nb(args()[3], 1, 2050)])
    refused(BAD_ARG, a, positions=None)
    refused(UNSUPPORTED, a, positions=DATA + 1)
    refused(UNSUPPORTED, a, qw=DATA + 2)
    refused(BAD_ARG, a, cache(rows=None))
    for bad in (dict(n_rot=130), dict(n_rot=-2), dict(n_rot=7), dict(freq_base=0.0), dict(freq_base=float("inf")), dict(freq_scale=float("nan")),
                dict(attn_factor=float("inf")), dict(eps=-1.0), dict(mode=2), dict(q8_variant=2)):
        refused(BAD_ARG, a, p=xqattn.rope_params(**{"n_rot": 64, "freq_base": 1e4, **bad}))
    refused(UNSUPPORTED, a, p=xqattn.rope_params(60, 1e4))


def test_kv_pages_refusals():
    lib = xqattn.load()
    pools = (xqattn.XqTensor * 2)(tensor(wl.F16, (128, 16, 4, 10)), tensor(wl.Q8_0, (128, 16, 4, 10)))
    X = DATA

    def err(want, st):
        assert st == want and lib.xq_last_error(), (st, lib.xq_last_error())

    err(BAD_ARG, lib.xq_kv_pages_copy(None, 1, X, X, 1, None))
    err(BAD_ARG, lib.xq_kv_pages_copy(pools, 0, X, X, 1, None))
    err(BAD_ARG, lib.xq_kv_pages_copy(pools, 2, X, X, -1, None))
    err(BAD_ARG, lib.xq_kv_pages_copy(pools, 2, None, X, 1, None))
    err(UNSUPPORTED, lib.xq_kv_pages_copy(pools, 2, X + 1, X, 1, None))
    assert lib.xq_kv_pages_copy(pools, 2, None, None, 0, None) == OK
    for bad, want in ((tensor(wl.F16, (128, 8, 4, 10)), BAD_SHAPE), (tensor(wl.F16, (128, 16, 4, 11)), BAD_SHAPE),
                      (tensor(wl.F16, (100, 16, 4, 10)), UNSUPPORTED), (tensor(wl.F16, (128, 16, 0, 10)), BAD_SHAPE), (with_type(99), UNSUPPORTED),
                      (with_nb(tensor(wl.F16, (128, 16, 4, 10)), 0, 4), UNSUPPORTED), (tensor(wl.F16, (128, 16, 4, 10), data=None), BAD_ARG)):
        err(want, lib.xq_kv_pages_copy((xqattn.XqTensor * 2)(pools[0], bad), 2, X, X, 1, None))
    err(UNSUPPORTED, lib.xq_kv_pages_copy((xqattn.XqTensor * 1)(tensor(wl.F16, (65536, 16384, 4, 10))), 1, X, X, 1, None))  # 2^33 byte pages
    Y = DATA + 4096
    err(BAD_ARG, lib.xq_kv_pages_compact(pools, 2, X, X, 2, 3, X, X, 4, X, None))           # rows_out is rows
    err(BAD_ARG, lib.xq_kv_pages_compact(pools, 2, X, X, 0, 3, X, X, 4, Y, None))
    err(BAD_ARG, lib.xq_kv_pages_compact(pools, 2, X, X, 2, 3, X, X, 0, Y, None))
    err(UNSUPPORTED, lib.xq_kv_pages_compact(pools, 2, X, X, 65536, 3, X, X, 4, Y, None))
    err(BAD_ARG, lib.xq_kv_pages_compact(pools, 2, X, X, 2, 3, None, X, 4, Y, None))
    err(UNSUPPORTED, lib.xq_kv_pages_compact(pools, 2, X, X, 2, 3, X + 2, X, 4, Y, None))
    n = ctypes.c_size_t(0)
    assert lib.xq_kv_pages_reserve_workspace(7, 100, ctypes.byref(n)) == OK and n.value >= 4 * 107
    err(BAD_ARG, lib.xq_kv_pages_reserve_workspace(0, 100, ctypes.byref(n)))
    err(WORKSPACE, lib.xq_kv_pages_reserve(X, X, 7, 3, 100, 16, X, X, X, 4 * 107 - 1, None))
    err(WORKSPACE, lib.xq_kv_pages_reserve(X, X, 7, 3, 100, 16, X, X, X + 4, 1 << 20, None))
    err(BAD_ARG, lib.xq_kv_pages_reserve(X, X, 7, 3, 100, 0, X, X, X, 1 << 20, None))
    err(BAD_ARG, lib.xq_kv_pages_reserve(X, X, 7, 0, 100, 16, X, X, X, 1 << 20, None))
    err(BAD_ARG, lib.xq_kv_pages_reserve(X, None, 7, 3, 100, 16, X, X, X, 1 << 20, None))
    assert lib.xq_kv_pages_fork_workspace(5, ctypes.byref(n)) == OK and n.value >= 60
    err(BAD_ARG, lib.xq_kv_pages_fork_workspace(1025, ctypes.byref(n)))
    err(BAD_ARG, lib.xq_kv_pages_fork(pools, 2, X, X, X, 4, 3, X, X, 1025, X, X, 1 << 20, None))
    err(WORKSPACE, lib.xq_kv_pages_fork(pools, 2, X, X, X, 4, 3, X, X, 5, X, X, 59, None))
    err(WORKSPACE, lib.xq_kv_pages_fork(pools, 2, X, X, X, 4, 3, X, X, 5, X, None, 1 << 20, None))
    err(BAD_ARG, lib.xq_kv_pages_fork(pools, 2, X, None, X, 4, 3, X, X, 5, X, X, 1 << 20, None))
    assert lib.xq_kv_pages_fork(pools, 2, None, None, None, 4, 3, None, None, 0, None, None, 1 << 20, None) == OK
    err(BAD_ARG, lib.xq_kv_pages_release(X, X, X, 4, 3, 10, X, -1, None))
    err(BAD_ARG, lib.xq_kv_pages_release(X, X, X, 4, 3, 0, X, 1, None))
    err(UNSUPPORTED, lib.xq_kv_pages_release(X, X, X, 4, 3, 10, X, 65536, None))
    err(BAD_ARG, lib.xq_kv_pages_release(X, X, X, 4, 3, 10, None, 1, None))
    assert lib.xq_kv_pages_release(None, None, None, 4, 3, 10, None, 0, None) == OK


def test_limits_of_strides_and_counts():
    """Sizes whose products the kernels hold in 32 bits, at and past their bounds."""
    lib = xqattn.load()

    def tree(want, q, c, d):
        assert call_tree(q, c, d) == want and lib.xq_last_error(), lib.xq_last_error()
        assert lib.xq_supports_fa_tree(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d)) == 0

    for i in (1, 3):  # row, page
        for name in "kv":
            tree(UNSUPPORTED, *tree_args(c=cache(**{name: with_nb(tensor(wl.F16, (128, 16, 4, 10)), i, 1 << 32)})))
    tree(UNSUPPORTED, *tree_args(T=64, H=32, B=4096, c=cache(n_seq=4096)))                                 # 2^23 query rows
    big = (1 << 31) - 1
    tree(UNSUPPORTED, *tree_args(T=64, H=big, B=big, c=cache(n_seq=big, k=tensor(wl.F16, (128, 16, big, 10)), v=tensor(wl.F16, (128, 16, big, 10)))))
    tree(UNSUPPORTED, *tree_args(T=1, H=8, B=1024, c=cache(n_seq=1024, P=1 << 20, cols=2000, Hkv=8)))         # 2^25 tiles of 8192 segments
    q, c, d = tree_args(T=1, H=8, B=4, c=cache(n_seq=4, P=1 << 20, cols=2000, Hkv=8))
    assert lib.xq_supports_fa_tree(ctypes.byref(q), ctypes.byref(c), ctypes.byref(d)) == 1

    def rope(ok, T=4, B=2, H=8, nb=None):
        a = [tensor(wl.F32, (128, T, h, B), nb=(4, 512 * h, 512, 512 * h * T)) for h in (H, 4, 4, H)]  # a token's heads together
        if nb:
            a[nb[0]].nb[2] = nb[1]
        c, p = cache(n_seq=B), xqattn.rope_params(64, 1e4)
        r = [ctypes.byref(x) for x in a]
        assert lib.xq_supports_qk_norm_rope(r[0], r[1], r[2], ctypes.byref(p), r[3], ctypes.byref(c)) == ok
        if not ok:
            assert lib.xq_qk_norm_rope(r[0], r[1], r[2], DATA, None, None, None, None, ctypes.byref(p), r[3], ctypes.byref(c), None) == UNSUPPORTED

    for i in range(4):
        rope(0, nb=(i, 1 << 32))
        rope(1, nb=(i, (1 << 32) - 4))
    rope(1, T=(1 << 25) - 1)
    rope(0, T=1 << 25)
    rope(0, T=(1 << 31) - 1, B=(1 << 31) - 1)
    two = (xqattn.XqTensor * 2)(tensor(wl.F16, (128, 16, 4, 10)), tensor(wl.F16, (128, 16, 4, 10)))
    assert lib.xq_kv_pages_compact(two, 2, DATA, DATA, 2, 3, DATA, DATA, 4, DATA + 4096, None) == BAD_ARG   # one pool twice
    many = (xqattn.XqTensor * 1025)(*[tensor(wl.F16, (128, 16, 4, 10), data=DATA + 4096 * i) for i in range(1025)])
    assert lib.xq_kv_pages_copy(many, 1025, DATA, DATA, 1, None) == BAD_ARG
    assert lib.xq_kv_pages_copy(many, 1024, DATA, DATA, 0, None) == OK


def test_binding_refuses_tensors_that_do_not_fit():
    import torch
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pool = xqattn.pool_tensor(torch.zeros(16 * 4 * 256 * 3, dtype=torch.uint8), wl.F16, 128, 16, 4, 3)
    with pytest.raises(ValueError, match="int32"):
        xqattn.kv_pages_copy([pool], torch.zeros(2), i32(2))
    with pytest.raises(ValueError, match="hold 2"):
        xqattn.kv_pages_copy([pool], i32(2), i32(1))
    with pytest.raises(ValueError, match="device"):
        xqattn.kv_pages_copy([pool], i32(2), i32(2))
    with pytest.raises(ValueError, match="one row per sequence"):
        xqattn.kv_pages_compact([pool], i32(2, 3), i32(2), i32(3, 4), i32(2), i32(2))
    with pytest.raises(ValueError, match="one number per page"):
        xqattn.kv_pages_fork([pool], i32(2, 3), i32(2), i32(4), i32(1), i32(1), i32(1))
    with pytest.raises(ValueError, match="2 dimensions"):
        xqattn.kv_pages_release(i32(6), i32(2), i32(3), i32(1))
    c = xqattn.KvPages(pool, pool, i32(2, 3), i32(1))
    with pytest.raises(ValueError, match="per sequence"):
        c.struct()


def test_host_models_agree_with_themselves():
    """The oracle's pieces on cases small enough to read."""
    assert ancestors([-1, 0, 0, 1, 3]).tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0], [1, 1, 0, 1, 1]]
    m = Pages(np.array([[4, 1], [-1, -1], [-1, -1]], np.int32), np.array([6, 0, 0], np.int32), np.array([0, 1, 0, 0, 1], np.int32), 4)
    done, copies = m.fork([0, 0], [1, 2])
    assert done.tolist() == [1, 1] and copies == [(1, 0, 2), (1, 2, 2)]
    assert m.table.tolist() == [[4, 1], [4, 0], [4, 2]] and m.refs.tolist() == [1, 1, 1, 0, 3] and m.rows.tolist() == [6, 6, 6]
    m.release([0])
    assert m.refs.tolist() == [1, 0, 1, 0, 2] and m.reserve([5, 0, 0]).tolist() == [8, 8, 8] and m.table[0].tolist() == [1, 3]
    c = Cache(np.random.default_rng(0), wl.Q4_0, 128, 2, 3, [4], [1], head_major=True, pad=2)
    assert c.values(c.k, 0, 5).shape == (5, 2, 128) and c.has(0, 9).tolist() == [True] * 6 + [False] * 3
