"""Which kernel an attention call over packed sequences takes, in how many workgroups, and what is refused as too large for one launch
(no GPU)."""
import ctypes as ct

import pytest

from laya_cuda import _lib
from test_attend import description

FEW_THREADS = 512  # of a workgroup of the kernel for few rows, at most


def workspace(**change):
    return _lib.load().laya_attend_workspace(ct.byref(description(**change)))


@pytest.mark.parametrize("n_seq,kv_heads", [(1, 7), (7, 1), (3, 5), (57, 1)])
def test_grids_of_whole_xcds_stay_below_a_launch(n_seq, kv_heads):
    """The kernel for few rows rounds its (sequence, key head) pairs up to a multiple of 8 where they spread evenly: with the
    rounding a launch has fewer than 2^32 threads, or the call is refused."""
    pairs, rounded, most = n_seq * kv_heads, (n_seq * kv_heads + 7) // 8 * 8, (1 << 32) // FEW_THREADS
    call = dict(n_seq=n_seq, heads=kv_heads, kv_heads=kv_heads, dim=64, max_k=10, kernel=_lib.ATTEND_FEW)
    for tiles, fits in (((most - 1) // pairs, False), ((most - 1) // rounded + 1, False), ((most - 1) // rounded, True)):
        assert workspace(max_q=32 * tiles, **call) == (0 if fits else -1)
