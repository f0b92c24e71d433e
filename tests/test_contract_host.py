"""What the header says about workspaces, by the C entries alone (nothing is launched)."""
import ctypes as C

import pytest

A = 1 << 20          # an address aligned to anything, never read


@pytest.mark.parametrize("R", [1, 10, 16])
def test_few_rows_need_a_workspace_in_the_weight_gradient_only(R):
    from mole_b200 import _lib
    lib, n = _lib.lib, C.c_int64(-1)
    for elem, kn in ((4, 0), (4, 1), (2, 0), (2, 1), (1, 0)):
        assert lib.mole_grouped_mm_workspace_bytes(A, A, R, 33, 65, 3, kn, elem, C.byref(n)) == 0 and n.value == 0
    assert lib.mole_grouped_mm_wgrad_workspace_bytes(A, A, R, 64, 128, 3, 1, C.byref(n)) == 0 and n.value == 0
    # rows that do not start on 16 bytes are copied to rows that do: 33 columns of bf16 to 40
    assert lib.mole_grouped_mm_wgrad_workspace_bytes(A, A, R, 33, 64, 3, 1, C.byref(n)) == 0
    assert n.value == -(-R * 40 * 2 // 256) * 256
    assert lib.mole_grouped_mm_wgrad(A, A, A, R, 33, 64, 3, 1, A, None, 0, None) == -1
    assert b"workspace" in lib.mole_last_error_string()
