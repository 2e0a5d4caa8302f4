"""CPU tests of the output head's limits on sizes."""
import ctypes

import pytest

import mxs_sampler
from mxs_sampler import MXS_ERR_INVALID
from test_head_abi import A, bwd, lib  # noqa: F401  (lib is a fixture)


@pytest.mark.parametrize("rows", [2 ** 24 + 1, 2 ** 28, 2 ** 31 - 2000])
def test_backward_refuses_rows_beyond_its_waits(lib, rows):  # noqa: F811
    """What the gradients' kernels wait for, for a second at most, grows with the rows:
    2^24 take half of it."""
    n = ctypes.c_size_t()
    assert bwd(lib, rows=rows) == MXS_ERR_INVALID
    assert lib.mxs_ce_workspace_size(A, 64, rows, 64, 100, 1, ctypes.byref(n)) == MXS_ERR_INVALID
