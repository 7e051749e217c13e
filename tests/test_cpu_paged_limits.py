"""Refusals of the paged entry points and their binding at sizes and arguments of their own. No GPU:
every call is refused before a launch."""
import xqattn
from test_cpu_paged import DATA, UNSUPPORTED, WORKSPACE


def test_reserve_refuses_tables_whose_entries_pass_32_bits():
    lib = xqattn.load()
    X = DATA
    call = lambda n_seq, cols, ws_bytes: lib.xq_kv_pages_reserve(X, X, n_seq, cols, 100, 16, X, X, X, ws_bytes, None)  # noqa: E731
    for n_seq, cols in ((1 << 16, 1 << 16), (1 << 17, 1 << 15), ((1 << 31) - 1, (1 << 31) - 1), (3, (1 << 31) - 1)):
        assert call(n_seq, cols, 1 << 40) == UNSUPPORTED and lib.xq_last_error(), (n_seq, cols)
    assert call((1 << 16) - 1, 1 << 16, 0) == WORKSPACE  # below: the next check
