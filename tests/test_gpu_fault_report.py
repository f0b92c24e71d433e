"""A kernel that gave up on a bounded wait is reported to the calls behind it: the products over packed rows and
the Adam step refuse to go on from results that were never written.  The fault is a barrier whose flag
nothing sets: it returns after its limit of 5 ms and leaves the context usable."""
import ctypes as C

import pytest
import torch

from test_gpu_ragged import F32, offs, rnd
from test_gpu_runtime import _flag_arrays, _free

pytestmark = pytest.mark.gpu
CODE = 42           # of the barrier: 40 and the first rank that is missing


@pytest.fixture
def fault():
    """Call it to have a wait run out; the code is cleared afterwards."""
    from mole_b200 import ops
    from mole_b200._lib import check, lib
    assert ops.device_fault() == 0
    ptrs, views, table = _flag_arrays(3)
    views[0][1] = 1
    torch.cuda.synchronize()

    def run_out():
        check(lib.mole_peer_barrier(table, 3, 0, 1, 5_000_000, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        torch.cuda.synchronize()
    yield run_out
    torch.cuda.synchronize()
    ops.device_fault()
    assert ops.device_fault() == 0 and ops.device_fault_peek() == 0
    _free(ptrs)


def test_products_and_steps_refuse_until_the_code_is_cleared(fault):
    from mole_b200 import ops
    from mole_b200._lib import MoleError
    o, x, w, big = offs([4, 6]), rnd(10, 16), rnd(2, 8, 16, seed=1), rnd(64, 16)
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(w)
    p, m, v = torch.ones(300, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    out = torch.full((10, 8), 7.0, device="cuda")
    calls = [lambda: ops.grouped_mm(x, w, o, out=out), lambda: ops.grouped_mm(big.bfloat16(), w.bfloat16(), offs([60, 4])),
             lambda: ops.grouped_mm_wgrad(x, x, o), lambda: ops.quantize_rows(x),
             lambda: ops.grouped_mm_int8(q, s, wq, ws, o, out_dtype=F32), lambda: ops.mm_int8(q, s, wq[0], ws[0]),
             lambda: ops.adam_multi([p], [p], [m], [v], t=1, lr=0.1)]
    for f in calls[1:-1]:
        f()
    torch.cuda.synchronize()
    fault()
    assert ops.device_fault_peek() == CODE                 # nobody has polled
    for f in calls:
        with pytest.raises(MoleError, match="a barrier that a rank did not reach gave up .*fault code 42") as e:
            f()
        assert e.value.status == -6
    torch.cuda.synchronize()
    assert (out == 7).all() and (p == 1).all() and not m.any() and p._version == 0 and out._version == 0
    assert ops.device_fault() == CODE and ops.device_fault_peek() == 0
    for f in calls:
        f()
    assert (p != 1).all() and not (out == 7).all()


def test_a_polled_code_counts_too(fault):
    """Other kernels' codes travel by the poll."""
    from mole_b200 import ops
    from mole_b200._lib import MoleError
    x, w, o = rnd(10, 16), rnd(2, 8, 16, seed=1), offs([4, 6])
    fault()
    ops.device_fault_poll()
    torch.cuda.synchronize()
    with pytest.raises(MoleError, match="fault code 42"):
        ops.grouped_mm(x, w, o)
    assert ops.device_fault_peek() == CODE
    assert ops.device_fault() == CODE
    ops.device_fault_poll()
    torch.cuda.synchronize()
    assert ops.device_fault_peek() == 0
    ops.grouped_mm(x, w, o)


def test_backward_and_optimizer_raise(fault):
    import mole_b200
    from mole_b200 import ops
    from mole_b200._lib import MoleError
    from mole_b200.optim import DeviceAdam
    x, o = rnd(10, 16).requires_grad_(), offs([4, 6])
    w = torch.nn.Parameter(rnd(2, 8, 16, seed=1))
    opt = DeviceAdam([w], lr=0.1)
    y = mole_b200.grouped_mm(x, w, o).sum()
    y.backward(retain_graph=True)
    grad, before = x.grad.clone(), w.detach().clone()
    fault()
    with pytest.raises(MoleError, match="fault code 42") as e:
        y.backward(retain_graph=True)
    assert e.value.status == -6
    with pytest.raises(MoleError, match="fault code 42"):
        opt.step()
    assert torch.equal(x.grad, grad) and torch.equal(w, before) and opt.state[w]["step"] == 0
    assert ops.device_fault() == CODE
    y.backward()
    opt.step()
    assert torch.equal(x.grad, 2 * grad) and not torch.equal(w, before) and opt.state[w]["step"] == 1


def test_the_layer_names_what_gave_up(fault):
    from mole_b200 import MOLEModule, ops
    m = MOLEModule(0, 4, 128, 128, -1, 2, 4, {"local_rank": 0, "world_size": 1, "rank": 0}, "gelu", 1, False, False, dtype=F32)
    x = rnd(64, 128)
    m(x, capacity_factor=2.0)
    fault()
    with pytest.raises(RuntimeError, match="a barrier that a rank did not reach gave up .*fault code 42"):
        m(x, capacity_factor=2.0)
    assert ops.device_fault() == CODE
    m(x, capacity_factor=2.0)
