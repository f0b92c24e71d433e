"""What the header says about workspaces, and what arguments raise by themselves; nothing is launched."""
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


def test_an_argument_without_a_truth_value_raises_its_own_error():
    import torch
    import mole_b200
    from mole_b200 import ops
    x, w, o = torch.zeros(4, 8), torch.zeros(2, 6, 8), torch.tensor([0, 2, 4], dtype=torch.int32)
    both = torch.tensor([True, False])

    class Broken:
        def __bool__(self):
            raise KeyError("no truth in it")
        __float__ = __bool__
    for f in (ops.grouped_mm, mole_b200.grouped_mm):
        with pytest.raises(RuntimeError, match="more than one value"):
            f(x, w, o, w_kn=both)
        with pytest.raises(KeyError, match="no truth"):
            f(x, w, o, w_kn=Broken())
    t = [torch.zeros(4)]
    for kw in ({"adamw": Broken()}, {"lr": Broken()}):
        with pytest.raises(KeyError, match="no truth"):
            ops.adam_multi(t, t, t, t, **{"t": 1, "lr": 1e-3, **kw})
    with pytest.raises(RuntimeError, match="more than one value"):
        ops.adam_multi(t, t, t, t, t=1, lr=1e-3, adamw=both)
    with pytest.raises(TypeError):
        ops.adam_multi(t, t, t, t, t=1, lr=1e-3, seed="7")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adam_multi(t, t, t, t, t=1, lr=1e-3)
