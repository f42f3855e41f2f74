"""Extents of 8-bit rows that a launch does not cover are refused before it (no GPU)."""
import pytest

from laya_cuda import _lib
from test_rows8 import P, refused

# Four pieces of 4 fp32 values a thread and 256 threads a workgroup: 4,096 codes each, and fewer than 2^32 threads in all.
MOST = (2 ** 32 // 256 - 1) * 4096


@pytest.mark.parametrize("rows,width", [(2 ** 29 - 1, 1), (2 ** 29 - 16, 128), ((MOST // 1024) + 1, 1000), (2 ** 6, 2 ** 30)])
def test_the_last_workgroup_s_threads_count(rows, width):
    """Codes of just under 2^36: their 2^24 workgroups would be 2^32 threads."""
    assert MOST < rows * -(-width // 128) * 128
    refused("laya_op_quantize8", P, _lib.F32, width, P, P, rows, width, None, match="2^36 codes less 4096")
    refused("laya_op_dequantize8", P, P, P, _lib.F32, width, rows, width, None, match="2^36 codes less 4096")
