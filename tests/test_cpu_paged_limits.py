"""Refusals of the paged entry points and their binding at sizes and arguments of their own. No GPU:
every call is refused before a launch."""
import pytest

import xqattn
from test_cpu_paged import DATA, UNSUPPORTED, WORKSPACE, tensor
from xqattn import workloads as wl


def test_reserve_refuses_tables_whose_entries_pass_32_bits():
    lib = xqattn.load()
    X = DATA
    call = lambda n_seq, cols, ws_bytes: lib.xq_kv_pages_reserve(X, X, n_seq, cols, 100, 16, X, X, X, ws_bytes, None)  # noqa: E731
    for n_seq, cols in ((1 << 16, 1 << 16), (1 << 17, 1 << 15), ((1 << 31) - 1, (1 << 31) - 1), (3, (1 << 31) - 1)):
        assert call(n_seq, cols, 1 << 40) == UNSUPPORTED and lib.xq_last_error(), (n_seq, cols)
    assert call((1 << 16) - 1, 1 << 16, 0) == WORKSPACE  # below: the next check


def test_binding_takes_pools_by_descriptor_and_refuses_none():
    """Pools as plain descriptors go as far as the check of the other tensors' device; an empty list is
    refused."""
    import torch
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pool = tensor(wl.F16, (128, 16, 4, 3))
    with pytest.raises(ValueError, match="device"):
        xqattn.kv_pages_copy([pool], i32(2), i32(2))
    with pytest.raises(ValueError, match="device"):
        xqattn.kv_pages_compact([pool], i32(2, 3), i32(2), i32(2, 4), i32(2), i32(2))
    with pytest.raises(ValueError, match="device"):
        xqattn.kv_pages_fork([pool], i32(2, 3), i32(2), i32(3), i32(1), i32(1), i32(1))
    with pytest.raises(ValueError, match="pool"):
        xqattn.kv_pages_fork([], i32(2, 3), i32(2), i32(3), i32(1), i32(1), i32(1))
