"""``grouped_mm`` where a program has it in other hands: inference mode, activation checkpointing, saved-tensor hooks,
an expanded or empty gradient, no rows, several graphs alive at once, backward on another stream."""
import pytest
import torch
import torch.utils.checkpoint

from test_gpu_ragged import BF16, F32, offs, rnd

pytestmark = pytest.mark.gpu
COUNTS = [7, 0, 40, 17]


def operands(dtype, tail=5):
    x = rnd(sum(COUNTS) + tail, 48, dtype=dtype).requires_grad_()
    return x, rnd(4, 64, 48, seed=1, dtype=dtype).requires_grad_(), offs(COUNTS), rnd(sum(COUNTS) + tail, 64, seed=2, dtype=dtype)


def plain(x, w, o, dy):
    import mole_b200
    y = mole_b200.grouped_mm(x, w, o)
    return (y.detach(), *torch.autograd.grad(y, (x, w), dy))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_inference_mode(dtype):
    import mole_b200
    x, w, o, dy = operands(dtype)
    want = plain(x, w, o, dy)[0]
    with torch.inference_mode():
        y = mole_b200.grouped_mm(x, w, o)
        assert torch.equal(y, want) and not y.requires_grad
        fresh = [t.clone() for t in (x, w, o)]
        assert torch.equal(mole_b200.grouped_mm(*fresh), want)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_checkpointed(dtype, reentrant):
    import mole_b200
    x, w, o, dy = operands(dtype)
    want = plain(x, w, o, dy)
    y = torch.utils.checkpoint.checkpoint(lambda a: mole_b200.grouped_mm(a, w, o), x, use_reentrant=reentrant)
    y.backward(dy)
    assert all(torch.equal(a, b) for a, b in zip((y, x.grad, w.grad), want))


def test_saved_tensors_on_the_host():
    import mole_b200
    for dtype in (BF16, F32):
        x, w, o, dy = operands(dtype)
        want = plain(x, w, o, dy)
        with torch.autograd.graph.save_on_cpu():
            y = mole_b200.grouped_mm(x, w, o)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want[1:]))


def test_gradients_without_rows_and_of_part_of_the_output():
    import mole_b200
    for dtype in (BF16, F32):
        x = torch.empty(0, 48, dtype=dtype, device="cuda", requires_grad=True)
        w = rnd(4, 64, 48, dtype=dtype).requires_grad_()
        y = mole_b200.grouped_mm(x, w, offs([0, 0, 0, 0]))
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == (0, 48) and dw.shape == w.shape and not dw.any()
        x, w, o, dy = operands(dtype)
        y = mole_b200.grouped_mm(x, w, o)
        (dx,) = torch.autograd.grad(y[7:30, 3], x, torch.ones(23, dtype=dtype, device="cuda"))
        full = torch.zeros_like(dy)
        full[7:30, 3] = 1
        assert torch.equal(dx, plain(x, w, o, full)[1])


def test_graphs_alive_at_once_and_backward_on_another_stream():
    import mole_b200
    x, w, o, dy = operands(BF16)
    want = plain(x, w, o, dy)
    graphs = [mole_b200.grouped_mm(x, w, o) for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                     # the engine runs each node on its forward's stream
        got = [torch.autograd.grad(y, (x, w), dy) for y in reversed(graphs)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want[1:]))
    del graphs[1:3]
    again = torch.autograd.grad(mole_b200.grouped_mm(x, w, o), (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(again, want[1:]))


@pytest.mark.filterwarnings("ignore")
def test_anomaly_mode_and_hooks_see_the_gradients():
    import mole_b200
    x, w, o, dy = operands(F32)
    seen = []
    x.register_hook(lambda g: seen.append(g.clone()))
    with torch.autograd.detect_anomaly(check_nan=True):
        mole_b200.grouped_mm(x, w, o).backward(dy)
    assert torch.equal(seen[0], x.grad)
    bad = dy.clone()
    bad[0, 0] = float("nan")
    with pytest.raises(RuntimeError, match="nan"), torch.autograd.detect_anomaly(check_nan=True):
        mole_b200.grouped_mm(x, w, o).backward(bad)
