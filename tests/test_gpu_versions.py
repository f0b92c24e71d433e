"""What the products and the Adam step over many tensors write counts the tensors' versions up, as torch's own
operations in place do: a backward that still needs the old values raises instead of using the new ones."""
import pytest
import torch

from test_gpu_ragged import F32, offs, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("optimizer", ["torch", 32, 8])
def test_a_step_between_forward_and_backward_is_told(optimizer):
    import mole_b200
    from mole_b200.optim import DeviceAdam
    o, w = offs([4, 6]), torch.nn.Parameter(rnd(2, 8, 16, seed=1))
    opt = torch.optim.AdamW([w], lr=0.1) if optimizer == "torch" else DeviceAdam([w], lr=0.1, state_bits=optimizer)
    x = rnd(10, 16).requires_grad_()
    mole_b200.grouped_mm(x, w, o).sum().backward()
    late = mole_b200.grouped_mm(x, w, o)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.sum().backward()
    # in the right order nothing is in the way
    for _ in range(2):
        opt.zero_grad()
        mole_b200.grouped_mm(x, w, o).sum().backward()
        opt.step()


def test_every_tensor_that_is_written_counts_up():
    from mole_b200 import ops
    n = 300
    p, g = torch.ones(n, device="cuda"), torch.ones(n, device="cuda")
    zeros8 = lambda: torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # noqa: E731
    m, v, ms, vs = zeros8(), zeros8(), torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")
    before = [t._version for t in (p, m, v, ms, vs)] + [g._version]
    ops.adam_multi([p], [g], [m], [v], [ms], [vs], t=1, lr=1e-3)
    assert [t._version for t in (p, m, v, ms, vs)] + [g._version] == [b + 1 for b in before[:5]] + before[5:]
    with pytest.raises(RuntimeError, match="step count"):
        ops.adam_multi([p], [g], [m], [v], [ms], [vs], t=0, lr=1e-3)
    assert p._version == before[0] + 1                    # a refused call has written nothing


def test_a_given_output_counts_up():
    import mole_b200
    from mole_b200 import ops
    o, w = offs([4, 6]), rnd(2, 16, 16, seed=1).requires_grad_()
    q, s = ops.quantize_rows(rnd(10, 16, seed=2))
    wq, ws = ops.quantize_rows(rnd(2, 16, 16, seed=3))
    a = rnd(10, 16, seed=4)
    for write in (lambda out: ops.grouped_mm(a, w.detach(), o, out=out),
                  lambda out: ops.grouped_mm_int8(q, s, wq, ws, o, out_dtype=F32, out=out),
                  lambda out: ops.mm_int8(q, s, wq[0], ws[0], out_dtype=F32, out=out)):
        x = rnd(10, 16)
        y = mole_b200.grouped_mm(x, w, o)
        write(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    x = rnd(10, 16).requires_grad_()
    y = mole_b200.grouped_mm(x, w, o)
    ops.grouped_mm_wgrad(a, a, o, out=w.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_inference_tensors_are_written_too():
    from mole_b200 import ops
    from mole_b200.optim import DeviceAdam
    with torch.inference_mode():
        o, x, w, out = offs([4, 6]), rnd(10, 16), rnd(2, 8, 16, seed=1), torch.zeros(10, 8, device="cuda")
        ops.grouped_mm(x, w, o, out=out)
        assert torch.equal(out, ops.grouped_mm(x, w, o)) and out.any()
        p = torch.ones(10, device="cuda")
        z = [torch.zeros(10, device="cuda") for _ in range(2)]
        ops.adam_multi([p], [torch.ones_like(p)], [z[0]], [z[1]], t=1, lr=0.5)
        assert (p < 1).all()
    # parameters made outside, stepped inside
    q = torch.nn.Parameter(torch.ones(10, device="cuda"))
    q.grad = torch.ones_like(q)
    with torch.inference_mode():
        DeviceAdam([q], lr=0.5).step()
    assert (q < 1).all()


def test_an_operand_that_no_gradient_takes_may_be_overwritten():
    """As in torch's own products: dw takes x, dx takes w."""
    import mole_b200
    o, x, w = offs([4, 6]), rnd(10, 16), rnd(2, 8, 16, seed=1)
    for one, other in ((0, 1), (1, 0)):
        t = [x.clone(), w.clone()]
        t[one].requires_grad_()
        y = mole_b200.grouped_mm(*t, o)
        (want,) = torch.autograd.grad(y.sum(), t[one], retain_graph=True)
        with torch.no_grad():
            t[one].mul_(2)
        (got,) = torch.autograd.grad(y.sum(), t[one], retain_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(y.sum(), t[one], create_graph=True)
        t[other].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
