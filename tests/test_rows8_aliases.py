"""A residual that is the output itself has its type (no GPU): read in another, each lane would take what others have written."""
import pytest

from laya_cuda import _lib
from test_rows8 import P, refused


@pytest.mark.parametrize("rtype,out", [(_lib.F32, _lib.F16), (_lib.BF16, _lib.F16), (_lib.F16, _lib.BF16), (_lib.BF16, _lib.F32), (_lib.F32, _lib.E4M3)])
def test_in_place_residuals_of_another_type_are_refused(rtype, out):
    refused("laya_op_linear8", P, P, P, P, None, P, rtype, P, P if out == _lib.E4M3 else None, out, 0, 3, 64, 100, -1, None, match="has its type")
