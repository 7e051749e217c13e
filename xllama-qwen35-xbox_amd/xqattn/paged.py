"""Host binding of the paged KV cache (``include/xq_attn.h``, "A KV cache in pages"):
norms and rotation of queries and keys into the cache, attention of drafted tokens and of
whole chunks over it, the weight its rows get, the verification of drafted tokens, and the
pages themselves. Like the rest of the binding it only fills descriptors
and hands over workspaces and the stream; torch holds the memory.

``KvPages`` is one layer's cache; the page operations take a list of pools (K and V of
every layer) that one page table addresses. A call runs on the device of its tensors:
on that device's current stream unless ``stream`` is given.
"""
from __future__ import annotations

import contextlib
import ctypes
import dataclasses

from . import DevTensor, XqError, XqTensor, _aligned_ptr, _check, load  # noqa: F401
from .workloads import TYPE_SIZE, record_bytes

ROPE_HALVES, ROPE_PAIRS = 0, 1


class XqKvPages(ctypes.Structure):
    _fields_ = [
        ("k", XqTensor),
        ("v", XqTensor),
        ("table", ctypes.c_void_p),
        ("rows", ctypes.c_void_p),
        ("n_seq", ctypes.c_int32),
        ("table_cols", ctypes.c_int32),
    ]


class XqRopeParams(ctypes.Structure):
    _fields_ = [
        ("n_rot", ctypes.c_int32),
        ("mode", ctypes.c_int32),
        ("freq_base", ctypes.c_float),
        ("freq_scale", ctypes.c_float),
        ("attn_factor", ctypes.c_float),
        ("eps", ctypes.c_float),
        ("q8_variant", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


def rope_params(n_rot, freq_base, freq_scale=1.0, attn_factor=1.0, mode=ROPE_HALVES, eps=1e-6, q8_variant=0) -> XqRopeParams:
    return XqRopeParams(n_rot, mode, freq_base, freq_scale, attn_factor, eps, q8_variant, 0)


class XqChunkParams(ctypes.Structure):
    _fields_ = [
        ("scale", ctypes.c_float),
        ("max_bias", ctypes.c_float),
        ("logit_softcap", ctypes.c_float),
        ("window", ctypes.c_int32),
        ("reserved", ctypes.c_int32 * 4),
    ]


def chunk_params(scale, window=0, logit_softcap=0.0, max_bias=0.0) -> XqChunkParams:
    return XqChunkParams(scale, max_bias, logit_softcap, window)


def pool_tensor(t, kv_type: int, head_dim: int, page_rows: int, n_head_kv: int, n_pages: int, head_major=False) -> DevTensor:
    """A pool over a device buffer: pages of [page_rows][n_head_kv][record], or
    (head_major) of [n_head_kv][page_rows][record]."""
    rec = record_bytes(kv_type, head_dim)
    row, head = (rec, page_rows * rec) if head_major else (n_head_kv * rec, rec)
    return DevTensor(kv_type, (head_dim, page_rows, n_head_kv, n_pages), (TYPE_SIZE[kv_type], row, head, page_rows * n_head_kv * rec), t)


@dataclasses.dataclass
class KvPages:
    """One layer's cache: K and V pools, the page table int32 [n_seq, cols] and the rows
    that each sequence holds, int32 [n_seq]."""
    k: DevTensor
    v: DevTensor
    table: "object"
    rows: "object"

    def struct(self) -> XqKvPages:
        _i32("table", self.table, 2)
        _i32("rows", self.rows, 1)
        c = XqKvPages()
        c.k, c.v = self.k.desc(), self.v.desc()
        c.table, c.rows = self.table.data_ptr(), self.rows.data_ptr()
        c.n_seq, c.table_cols = self.table.shape
        if self.rows.numel() != c.n_seq:
            raise ValueError("rows must hold one number per sequence of the table")
        return c


def _i32(name, t, dims=None):
    import torch
    if t is None:
        return
    if t.dtype != torch.int32 or not t.is_contiguous() or (dims is not None and t.dim() != dims):
        raise ValueError(f"{name} must be a contiguous int32 tensor" + (f" of {dims} dimensions" if dims else ""))


def _f32(name, t, n):
    import torch
    if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < n):
        raise ValueError(f"{name} must be a contiguous float32 tensor of {n} elements")


def _size(name, t, n):
    if t is not None and t.numel() < n:
        raise ValueError(f"{name} must hold {n} numbers")


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


@contextlib.contextmanager
def _on(stream, *tensors):
    """The device of the tensors made current, and the stream to launch on."""
    import torch
    devs = {t.device for t in tensors if t is not None}
    if len(devs) != 1:
        raise ValueError(f"all tensors of a call must be on one device, got {sorted(map(str, devs))}")
    dev = devs.pop()
    if dev.type != "cuda":
        raise ValueError(f"device tensors are needed, got {dev}")
    if stream is not None and stream.device != dev:
        raise ValueError(f"stream of {stream.device}, tensors on {dev}")
    # (a workspace made inside belongs to the stream that uses it)
    with torch.cuda.device(dev), torch.cuda.stream(stream):
        yield ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _space(nbytes, workspace, like):
    import torch
    if workspace is None:
        workspace = torch.empty(nbytes + 256, dtype=torch.uint8, device=like.device)
    return workspace, *_aligned_ptr(workspace)


def _memory(pools):
    return [None if isinstance(p, XqTensor) else p.t for p in pools]


def _pools(pools):
    """Descriptors of the pools; one may be given as its descriptor, its memory is the caller's then."""
    if not pools:
        raise ValueError("at least one pool is needed")
    return (XqTensor * len(pools))(*[p if isinstance(p, XqTensor) else p.desc() for p in pools]), len(pools)


def supports_qk_norm_rope(q, k, v, params, q_out, cache: KvPages) -> bool:
    ds = [x.desc() for x in (q, k, v)]
    o, c = q_out.desc(), cache.struct()
    return bool(load().xq_supports_qk_norm_rope(*map(ctypes.byref, ds), ctypes.byref(params), ctypes.byref(o), ctypes.byref(c)))


def qk_norm_rope(q: DevTensor, k: DevTensor, v: DevTensor, positions, params: XqRopeParams, q_out: DevTensor, cache: KvPages,
                 q_weight=None, k_weight=None, n_tok=None, freq_factors=None, stream=None):
    """Per-head RMS norm and rotation of q and k; q to q_out, k and v into the cache."""
    d, n_q, _, n_seq = q.ne
    _i32("positions", positions)
    _size("positions", positions, n_q * n_seq)
    _i32("n_tok", n_tok)
    _size("n_tok", n_tok, n_seq)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        _f32(name, w, d)
    _f32("freq_factors", freq_factors, params.n_rot // 2)
    ds = [x.desc() for x in (q, k, v)]
    o, c = q_out.desc(), cache.struct()
    with _on(stream, q.t, k.t, v.t, q_out.t, positions, n_tok, q_weight, k_weight, freq_factors, cache.table, cache.rows, cache.k.t, cache.v.t) as s:
        _check(load().xq_qk_norm_rope(*map(ctypes.byref, ds), _ptr(positions), _ptr(n_tok), _ptr(q_weight), _ptr(k_weight),
                                      _ptr(freq_factors), ctypes.byref(params), ctypes.byref(o), ctypes.byref(c), s), "qk_norm_rope")


def supports_fa_tree(q, cache: KvPages, dst) -> bool:
    dq, c, dd = q.desc(), cache.struct(), dst.desc()
    return bool(load().xq_supports_fa_tree(ctypes.byref(dq), ctypes.byref(c), ctypes.byref(dd)))


def fa_tree_workspace(q, cache: KvPages, dst) -> int:
    dq, c, dd = q.desc(), cache.struct(), dst.desc()
    n = ctypes.c_size_t(0)
    _check(load().xq_fa_tree_workspace(ctypes.byref(dq), ctypes.byref(c), ctypes.byref(dd), ctypes.byref(n)), "fa_tree_workspace")
    return int(n.value)


def fa_tree(q: DevTensor, cache: KvPages, dst: DevTensor, scale: float, parents=None, n_tok=None, lse=None, workspace=None, stream=None):
    """Attention of each sequence's tokens (a tree by `parents`, or a chain) over its cached
    rows and their own. Returns the workspace, for the next call of these shapes."""
    _, n_q, h, n_seq = q.ne
    _i32("parents", parents)
    _size("parents", parents, n_q * n_seq)
    _i32("n_tok", n_tok)
    _size("n_tok", n_tok, n_seq)
    _f32("lse", lse, n_q * h * n_seq)
    dq, c, dd = q.desc(), cache.struct(), dst.desc()
    refs = [ctypes.byref(x) for x in (dq, c, dd)]
    n = ctypes.c_size_t(0)
    _check(load().xq_fa_tree_workspace(*refs, ctypes.byref(n)), "fa_tree_workspace")
    with _on(stream, q.t, dst.t, parents, n_tok, lse, cache.table, cache.rows, cache.k.t, cache.v.t, workspace) as s:
        ws, wp, wn = _space(n.value, workspace, dst.t)
        _check(load().xq_fa_tree(refs[0], refs[1], _ptr(parents), _ptr(n_tok), refs[2], _ptr(lse), scale, ctypes.c_void_p(wp), wn, s), "fa_tree")
    return ws


def supports_fa_chunk(q, cache: KvPages, dst) -> bool:
    dq, c, dd = q.desc(), cache.struct(), dst.desc()
    return bool(load().xq_supports_fa_chunk(ctypes.byref(dq), ctypes.byref(c), ctypes.byref(dd)))


def fa_chunk_workspace(q, cache: KvPages, dst) -> int:
    dq, c, dd = q.desc(), cache.struct(), dst.desc()
    n = ctypes.c_size_t(0)
    _check(load().xq_fa_chunk_workspace(ctypes.byref(dq), ctypes.byref(c), ctypes.byref(dd), ctypes.byref(n)), "fa_chunk_workspace")
    return int(n.value)


def _chunk_masks(q, first, prefix, n_tok):
    _, n_q, _, n_seq = q.ne
    for name, t, n in (("first", first, n_q * n_seq), ("prefix", prefix, n_seq), ("n_tok", n_tok, n_seq)):
        _i32(name, t)
        _size(name, t, n)
    return [_ptr(first), _ptr(prefix), _ptr(n_tok)]


def fa_chunk(q: DevTensor, cache: KvPages, dst: DevTensor, params: XqChunkParams, first=None, prefix=None, n_tok=None, lse=None,
             workspace=None, stream=None):
    """Attention of each sequence's chunk of new tokens over its cached rows and their own.
    Returns the workspace, for the next call of these shapes."""
    _, n_q, h, n_seq = q.ne
    masks = _chunk_masks(q, first, prefix, n_tok)
    _f32("lse", lse, n_q * h * n_seq)
    dq, c, dd = q.desc(), cache.struct(), dst.desc()
    n = fa_chunk_workspace(q, cache, dst)
    with _on(stream, q.t, dst.t, first, prefix, n_tok, lse, cache.table, cache.rows, cache.k.t, cache.v.t, workspace) as s:
        ws, wp, wn = _space(n, workspace, dst.t)
        _check(load().xq_fa_chunk(ctypes.byref(dq), ctypes.byref(c), ctypes.byref(params), *masks, ctypes.byref(dd), _ptr(lse),
                                  ctypes.c_void_p(wp), wn, s), "fa_chunk")
    return ws


def kv_weights_workspace(q, cache: KvPages) -> int:
    dq, c = q.desc(), cache.struct()
    n = ctypes.c_size_t(0)
    _check(load().xq_kv_weights_workspace(ctypes.byref(dq), ctypes.byref(c), ctypes.byref(n)), "kv_weights_workspace")
    return int(n.value)


def kv_weights(q: DevTensor, cache: KvPages, params: XqChunkParams, lse, scores, scores_out, first=None, prefix=None, n_tok=None,
               decay=1.0, fresh=True, workspace=None, stream=None):
    """The cached rows' attention weights of a chunk's tokens, added to `scores` [n_seq, cols] (None: zeros)."""
    _, n_q, h, n_seq = q.ne
    masks = _chunk_masks(q, first, prefix, n_tok)
    _f32("lse", lse, n_q * h * n_seq)
    if scores_out.dim() != 2 or scores_out.shape[0] != n_seq or (scores is not None and scores.shape != scores_out.shape):
        raise ValueError("scores and scores_out must be [n_seq, cols]")
    _f32("scores", scores, scores_out.numel())
    _f32("scores_out", scores_out, scores_out.numel())
    dq, c = q.desc(), cache.struct()
    n = kv_weights_workspace(q, cache)
    with _on(stream, q.t, first, prefix, n_tok, lse, scores, scores_out, cache.table, cache.rows, cache.k.t, workspace) as s:
        ws, wp, wn = _space(n, workspace, scores_out)
        _check(load().xq_kv_weights(ctypes.byref(dq), ctypes.byref(c), ctypes.byref(params), *masks, _ptr(lse), _ptr(scores), _ptr(scores_out),
                                    scores_out.shape[1], decay, int(fresh), ctypes.c_void_p(wp), wn, s), "kv_weights")
    return ws


def kv_pages_copy(pools, src, dst, stream=None):
    """Page dst[i] of every pool becomes page src[i]'s content."""
    _i32("src", src)
    _i32("dst", dst)
    _size("dst", dst, src.numel())
    arr, n = _pools(pools)
    with _on(stream, src, dst, *_memory(pools)) as s:
        _check(load().xq_kv_pages_copy(arr, n, _ptr(src), _ptr(dst), src.numel(), s), "kv_pages_copy")


def kv_pages_compact(pools, table, rows, path, n_path, rows_out, stream=None):
    """The accepted path's rows moved to the front of each sequence's new rows."""
    for name, t, dims in (("table", table, 2), ("rows", rows, 1), ("path", path, 2), ("n_path", n_path, 1), ("rows_out", rows_out, 1)):
        _i32(name, t, dims)
    for name, t in (("rows", rows), ("n_path", n_path), ("rows_out", rows_out)):
        _size(name, t, table.shape[0])
    if path.shape[0] != table.shape[0]:
        raise ValueError("path must have one row per sequence")
    arr, n = _pools(pools)
    with _on(stream, table, rows, path, n_path, rows_out, *_memory(pools)) as s:
        _check(load().xq_kv_pages_compact(arr, n, _ptr(table), _ptr(rows), *table.shape, _ptr(path), _ptr(n_path), path.shape[1],
                                          _ptr(rows_out), s), "kv_pages_compact")


def kv_pages_reserve(table, refs, page_rows, want, got, workspace=None, stream=None):
    """Free pages for rows [0, want[b]) of every sequence; got[b] rows then have pages."""
    for name, t, dims in (("table", table, 2), ("refs", refs, 1), ("want", want, 1), ("got", got, 1)):
        _i32(name, t, dims)
    for name, t in (("want", want), ("got", got)):
        _size(name, t, table.shape[0])
    n = ctypes.c_size_t(0)
    _check(load().xq_kv_pages_reserve_workspace(table.shape[0], refs.numel(), ctypes.byref(n)), "kv_pages_reserve_workspace")
    with _on(stream, table, refs, want, got, workspace) as s:
        ws, wp, wn = _space(n.value, workspace, table)
        _check(load().xq_kv_pages_reserve(_ptr(table), _ptr(refs), *table.shape, refs.numel(), page_rows, _ptr(want), _ptr(got),
                                          ctypes.c_void_p(wp), wn, s), "kv_pages_reserve")
    return ws


def kv_pages_fork(pools, table, rows, refs, parents, children, done, workspace=None, stream=None):
    """children[i] becomes a second holder of parents[i]'s rows; done[i] tells whether it did."""
    for name, t, dims in (("table", table, 2), ("rows", rows, 1), ("refs", refs, 1), ("parents", parents, 1), ("children", children, 1), ("done", done, 1)):
        _i32(name, t, dims)
    _size("rows", rows, table.shape[0])
    count = parents.numel()
    _size("children", children, count)
    _size("done", done, count)
    arr, m = _pools(pools)
    if arr[0].ne[3] != refs.numel():
        raise ValueError("refs must hold one number per page")
    n = ctypes.c_size_t(0)
    _check(load().xq_kv_pages_fork_workspace(count, ctypes.byref(n)), "kv_pages_fork_workspace")
    with _on(stream, table, rows, refs, parents, children, done, workspace, *_memory(pools)) as s:
        ws, wp, wn = _space(n.value, workspace, table)
        _check(load().xq_kv_pages_fork(arr, m, _ptr(table), _ptr(rows), _ptr(refs), *table.shape, _ptr(parents), _ptr(children), count,
                                       _ptr(done), ctypes.c_void_p(wp), wn, s), "kv_pages_fork")
    return ws


def kv_pages_release(table, rows, refs, seqs, stream=None):
    """The named sequences hold no page and no rows any more."""
    for name, t, dims in (("table", table, 2), ("rows", rows, 1), ("refs", refs, 1), ("seqs", seqs, 1)):
        _i32(name, t, dims)
    _size("rows", rows, table.shape[0])
    with _on(stream, table, rows, refs, seqs) as s:
        _check(load().xq_kv_pages_release(_ptr(table), _ptr(rows), _ptr(refs), *table.shape, refs.numel(), _ptr(seqs), seqs.numel(), s),
               "kv_pages_release")


def kv_pages_evict(pools, table, rows, refs, keep, scores, rows_out, first_rows=0, last_rows=0, positions=None, scores_out=None,
                   positions_out=None, workspace=None, stream=None):
    """Each sequence keeps keep[b] of its rows: protected ones, then those of most weight. refs
    (or None: no page is shared or given back)."""
    for name, t, dims in (("table", table, 2), ("rows", rows, 1), ("refs", refs, 1), ("keep", keep, 1), ("positions", positions, 2),
                          ("positions_out", positions_out, 2), ("rows_out", rows_out, 1)):
        _i32(name, t, dims)
    for name, t in (("rows", rows), ("keep", keep), ("rows_out", rows_out)):
        _size(name, t, table.shape[0])
    if scores.dim() != 2 or scores.shape[0] != table.shape[0]:
        raise ValueError("scores must have one row per sequence")
    for name, t in (("scores", scores), ("scores_out", scores_out)):
        _f32(name, t, scores.numel())
    for name, t in (("positions", positions), ("scores_out", scores_out), ("positions_out", positions_out)):
        if t is not None and t.shape != scores.shape:
            raise ValueError(f"{name} must have scores' shape")
    arr, m = _pools(pools)
    if refs is not None and arr[0].ne[3] != refs.numel():
        raise ValueError("refs must hold one number per page")
    n = ctypes.c_size_t(0)
    _check(load().xq_kv_pages_evict_workspace(table.shape[0], scores.shape[1], ctypes.byref(n)), "kv_pages_evict_workspace")
    with _on(stream, table, rows, refs, keep, scores, positions, scores_out, positions_out, rows_out, workspace, *_memory(pools)) as s:
        ws, wp, wn = _space(n.value, workspace, table)
        _check(load().xq_kv_pages_evict(arr, m, _ptr(table), _ptr(rows), _ptr(refs), *table.shape, _ptr(keep), first_rows, last_rows,
                                        _ptr(scores), _ptr(positions), scores.shape[1], _ptr(scores_out), _ptr(positions_out),
                                        _ptr(rows_out), ctypes.c_void_p(wp), wn, s), "kv_pages_evict")
    return ws


def verify_tokens_workspace(logits) -> int:
    d = logits.desc()
    n = ctypes.c_size_t(0)
    _check(load().xq_verify_tokens_workspace(ctypes.byref(d), ctypes.byref(n)), "verify_tokens_workspace")
    return int(n.value)


def verify_tokens(logits: DevTensor, tokens, path, n_path, next_token, uniform=None, draft: DevTensor = None, parents=None, n_tok=None,
                  temperature=None, logp=None, workspace=None, stream=None):
    """Which drafted tokens stand (path, n_path) and the token after them; uniform None: greedy."""
    _, n_q, n_seq, _ = logits.ne
    for name, t, n in (("tokens", tokens, n_q * n_seq), ("parents", parents, n_q * n_seq), ("n_tok", n_tok, n_seq), ("path", path, n_q * n_seq),
                       ("n_path", n_path, n_seq), ("next_token", next_token, n_seq)):
        _i32(name, t)
        _size(name, t, n)
    for name, t, n in (("temperature", temperature, n_seq), ("uniform", uniform, n_seq * (n_q + 1)), ("logp", logp, n_seq * (n_q + 1))):
        _f32(name, t, n)
    dl, dd = logits.desc(), None if draft is None else draft.desc()
    n = verify_tokens_workspace(logits)
    with _on(stream, logits.t, None if draft is None else draft.t, tokens, parents, n_tok, temperature, uniform, path, n_path, next_token,
             logp, workspace) as s:
        ws, wp, wn = _space(n, workspace, tokens)
        _check(load().xq_verify_tokens(ctypes.byref(dl), None if dd is None else ctypes.byref(dd), _ptr(tokens), _ptr(parents), _ptr(n_tok),
                                       _ptr(temperature), _ptr(uniform), _ptr(path), _ptr(n_path), _ptr(next_token), _ptr(logp),
                                       ctypes.c_void_p(wp), wn, s), "verify_tokens")
    return ws


def signatures():
    """ctypes argument types of this file's exports."""
    T, P, i32, f32, sz = ctypes.POINTER(XqTensor), ctypes.c_void_p, ctypes.c_int32, ctypes.c_float, ctypes.c_size_t
    C, R, S = ctypes.POINTER(XqKvPages), ctypes.POINTER(XqRopeParams), ctypes.POINTER(ctypes.c_size_t)
    K = ctypes.POINTER(XqChunkParams)
    return {
        "xq_supports_qk_norm_rope": (ctypes.c_int, [T, T, T, R, T, C]),
        "xq_qk_norm_rope": (i32, [T, T, T, P, P, P, P, P, R, T, C, P]),
        "xq_supports_fa_tree": (ctypes.c_int, [T, C, T]),
        "xq_fa_tree_workspace": (i32, [T, C, T, S]),
        "xq_fa_tree": (i32, [T, C, P, P, T, P, f32, P, sz, P]),
        "xq_supports_fa_chunk": (ctypes.c_int, [T, C, T]),
        "xq_fa_chunk_workspace": (i32, [T, C, T, S]),
        "xq_fa_chunk": (i32, [T, C, K, P, P, P, T, P, P, sz, P]),
        "xq_kv_weights_workspace": (i32, [T, C, S]),
        "xq_kv_weights": (i32, [T, C, K, P, P, P, P, P, P, i32, f32, i32, P, sz, P]),
        "xq_kv_pages_evict_workspace": (i32, [i32, i32, S]),
        "xq_kv_pages_evict": (i32, [T, i32, P, P, P, i32, i32, P, i32, i32, P, P, i32, P, P, P, P, sz, P]),
        "xq_verify_tokens_workspace": (i32, [T, S]),
        "xq_verify_tokens": (i32, [T, T, P, P, P, P, P, P, P, P, P, P, sz, P]),
        "xq_kv_pages_copy": (i32, [T, i32, P, P, i32, P]),
        "xq_kv_pages_compact": (i32, [T, i32, P, P, i32, i32, P, P, i32, P, P]),
        "xq_kv_pages_reserve_workspace": (i32, [i32, i32, S]),
        "xq_kv_pages_reserve": (i32, [P, P, i32, i32, i32, i32, P, P, P, sz, P]),
        "xq_kv_pages_fork_workspace": (i32, [i32, S]),
        "xq_kv_pages_fork": (i32, [T, i32, P, P, P, i32, i32, P, P, i32, P, P, sz, P]),
        "xq_kv_pages_release": (i32, [P, P, P, i32, i32, i32, P, i32, P]),
    }
