"""Edges of the paged K/V cache operators that the cases of test_paged_kv.py leave out; the cache, the reference in
float64 and its tolerance are that file's."""

import numpy as np
import pytest

from runtime import hb_lib
from test_paged_kv import Case, _torch, ints

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 6, 2 ** 40])
@pytest.mark.parametrize("heads,rows,lengths", [((14, 2, 64), [10, 3], [5, 70]), ((14, 2, 64), [300, 130], [200, 129]),
                                                ((16, 2, 128), [40, 300], [30, 500])])
def test_windows_wider_than_any_context(heads, rows, lengths, window):
    """They hide nothing, also in tiles whose first rows stand before the
    sequence (positions -5 .. -1 of the first case)."""
    torch = _torch()
    case = Case(heads, "bfloat16", rows, lengths, seed=41)
    plain, plain_lse = case.check()
    out, lse = case.check(window)
    assert torch.equal(out, plain) and torch.equal(lse, plain_lse)


def test_a_pool_in_host_memory_is_refused():
    """Before the library, or a device, is touched: the kernels would read host addresses."""
    torch = _torch()
    from runtime.paged_kv import PagedKVCache

    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache(1, 1, 64, 4, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache.wrap(torch.zeros((4, 1, 1, 2, 1, 64, 64), dtype=torch.bfloat16),
                          torch.zeros((2, 2), dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                          torch.zeros(2, dtype=torch.int32))


@gpu
@pytest.mark.parametrize("heads,rows", [((14, 2, 64), [2, 3, 1]), ((16, 2, 128), [200, 100, 50])])
def test_row_starts_that_descend_are_refused(heads, rows):
    """Entries would share rows, and their work could be any multiple of what
    the host has counted: the call gives zeros and says so, the next one runs."""
    torch = _torch()
    case = Case(heads, "bfloat16", rows, [250, 300, 270], seed=42)
    good, lse = case.check()
    a, b, c = np.cumsum(rows)
    right = case.row_start
    for bad in ([0, b, a, c], [0, a, c, b], [a, 0, b, c], [c, c, a, b]):
        case.row_start = ints(bad)
        out, none = case.attend(out=torch.full_like(case.q, 7.0))
        with pytest.raises(hb_lib.HbError, match="out of range"):
            case.cache.status()
        assert bool((out == 0).all()) and bool((none == -np.inf).all())
    case.row_start = right
    out, again = case.check()
    assert torch.equal(out, good) and torch.equal(again, lse)
