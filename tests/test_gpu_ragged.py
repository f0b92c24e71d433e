"""Products over rows packed by expert: ``ops.grouped_mm`` / ``grouped_mm_wgrad``, the differentiable
``mole_b200.grouped_mm``, ``quantize_rows`` and the products of 8-bit integers.

Tolerance of the products, against 64 bits on the same inputs: the stored value is rounded once, half
a step of its type (2^-8 bf16, 2^-24 fp32 relative), and the sum of L products is held in 32 bits,
whose every addition is off by at most a unit of 2^-23 (the tensor cores cut; the CUDA cores round,
half of that) of the partial sum, itself at most sum |a b|: (L + 2) 2^-23 sum |a b| in all.  Integer
products are exact, their scaling is restated operation by operation: equal bits."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def close(got, want, mag, length, what):
    """``mag``: the same sum over magnitudes."""
    err = (got.double() - want).abs()
    bound = HALF[got.dtype] * want.abs() + (length + 2) * 2.0 ** -23 * mag * 1.01 + 1e-37
    ok = err <= bound
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.numel()} off, worst {(err / bound).max().item():.3g} of the bound"


def spans(offsets):
    o = offsets.tolist()
    return list(zip(o[:-1], o[1:]))


def want_rows(x, w, offsets, kn):
    y = torch.zeros(x.shape[0], w.shape[2 if kn else 1], dtype=torch.float64, device=x.device)
    m = y.clone()
    for e, (a, b) in enumerate(spans(offsets)):
        if b > a:
            we = w[e].double() if kn else w[e].double().t()
            y[a:b], m[a:b] = x[a:b].double() @ we, x[a:b].double().abs() @ we.abs()
    return y, m


def want_wgrad(a, b, offsets):
    out = torch.zeros(len(offsets) - 1, a.shape[1], b.shape[1], dtype=torch.float64, device=a.device)
    m = out.clone()
    for e, (i, j) in enumerate(spans(offsets)):
        out[e], m[e] = a[i:j].double().t() @ b[i:j].double(), a[i:j].double().abs().t() @ b[i:j].double().abs()
    return out, m


def rnd(*shape, seed=0, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def offs(counts, head=0):
    return torch.tensor([head] + list(itertools.accumulate(counts, initial=head))[1:], dtype=torch.int32, device="cuda")


# rows per expert, rows before the first expert, rows behind the last
GROUPS = {
    "one row": ([1], 0, 0),
    "one expert": ([300], 0, 0),
    "nobody": ([0, 0, 0], 0, 9),
    "ragged": ([5, 0, 17, 1, 0, 130, 64, 3], 0, 0),
    "head and tail": ([0, 31, 16, 0], 3, 70),
    "many small": ([(i * 7) % 4 for i in range(64)], 0, 1),
    "large": ([513, 0, 255, 256, 257, 1000], 0, 5),
}
WIDTHS = [(1, 1), (7, 5), (8, 8), (24, 40), (64, 64), (72, 104), (128, 256), (200, 136), (256, 1001), (333, 96),
          (640, 520), (1024, 512)]


@pytest.mark.parametrize("groups", GROUPS)
@pytest.mark.parametrize("k,n", WIDTHS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_products_against_64_bits(dtype, k, n, groups):
    from mole_b200 import ops
    counts, head, tail = GROUPS[groups]
    o = offs(counts, head)
    R, E = head + sum(counts) + tail, len(counts)
    x = rnd(R, k, seed=1, dtype=dtype)
    for kn in (False, True):
        w = rnd(E, *((k, n) if kn else (n, k)), seed=2, dtype=dtype)
        y = ops.grouped_mm(x, w, o, w_kn=kn)
        close(y, *want_rows(x, w, o, kn), k, f"kn={kn}")
        assert not y[:head].any() and not y[R - tail:].any()
    b = rnd(R, n, seed=3, dtype=dtype)
    longest = max(counts)
    close(ops.grouped_mm_wgrad(x, b, o), *want_wgrad(x, b, o), longest, "wgrad")


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 15, 16, 17, 33, 100])
@pytest.mark.parametrize("k,n", [(2048, 512), (520, 2056), (4096, 136)])
def test_few_rows_long_reductions(rows, k, n):
    from mole_b200 import ops
    counts = [rows // 2, 0, rows - rows // 2, 0, 0]
    o = offs(counts)
    for dtype, kn in itertools.product((BF16, F32), (False, True)):
        x, w = rnd(rows, k, seed=1, dtype=dtype), rnd(5, *((k, n) if kn else (n, k)), seed=2, dtype=dtype)
        close(ops.grouped_mm(x, w, o, w_kn=kn), *want_rows(x, w, o, kn), k, f"{dtype} kn={kn}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("counts,head,tail,k,n", [
    ([40], 0, 0, 2048, 64), ([1, 16, 17, 0, 33], 2, 90, 1000, 100), ([15], 0, 300, 4100, 72), ([0, 3], 1, 60, 8192, 33),
    ([5000], 0, 7, 97, 146), ([0, 3001, 12], 5, 0, 64, 64), ([4096, 130], 0, 0, 264, 8), ([100], 0, 0, 1, 7)])
def test_few_tiles_and_long_reductions(dtype, counts, head, tail, k, n):
    """Too few tiles for the SMs: the reductions are cut into parts, over the width in the products, over
    the rows in the weight gradient; tiles of at most 16 rows have a form of their own."""
    from mole_b200 import ops
    o, R, E = offs(counts, head), head + sum(counts) + tail, len(counts)
    x, b = rnd(R, k, seed=1, dtype=dtype), rnd(R, n, seed=2, dtype=dtype)
    x[:head], b[:head], x[R - tail:], b[R - tail:] = (float("nan"),) * 4
    for kn in (False, True):
        w = rnd(E, *((k, n) if kn else (n, k)), seed=3, dtype=dtype)
        y = ops.grouped_mm(x, w, o, w_kn=kn)
        assert not y[:head].any() and not y[R - tail:].any()
        own = slice(head, R - tail)
        want, mag = want_rows(x, w, o, kn)
        close(y[own], want[own], mag[own], k, f"kn={kn}")
        assert torch.equal(y, ops.grouped_mm(x, w, o, w_kn=kn))
    dw = ops.grouped_mm_wgrad(x, b, o)
    close(dw, *want_wgrad(x, b, o), max(counts), "wgrad")
    assert torch.equal(dw, ops.grouped_mm_wgrad(x, b, o))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k,n", [(136, 264), (72, 33)])
def test_rows_of_others_do_not_leak(dtype, k, n):
    """NaN and infinities in the rows of one expert and of nobody stay there, also where a tile of the
    neighbour reaches over them."""
    from mole_b200 import ops
    counts, head, tail = [37, 16, 5, 130, 1, 200], 3, 40
    o, E = offs(counts, head), len(counts)
    R = head + sum(counts) + tail
    x, b, w = rnd(R, k, seed=1, dtype=dtype), rnd(R, n, seed=2, dtype=dtype), rnd(E, n, k, seed=3, dtype=dtype)
    lo, hi = o[2].item(), o[3].item()
    for t in (x, b):
        t[:head] = float("nan")
        t[R - tail:] = float("inf")
        t[lo:hi] = float("nan")
    y, dw = ops.grouped_mm(x, w, o), ops.grouped_mm_wgrad(b, x, o)
    own = torch.ones(R, dtype=torch.bool)
    own[lo:hi] = False
    assert torch.isfinite(y[own]).all() and torch.isnan(y[lo:hi]).all()
    assert not y[:head].any() and not y[R - tail:].any()
    keep = [0, 1, 3, 4, 5]
    assert torch.isfinite(dw[keep]).all() and torch.isnan(dw[2]).all()
    x0, b0 = x.clone(), b.clone()
    for t in (x0, b0):
        t[~torch.isfinite(t)] = 0
    want, mag = want_wgrad(b0, x0, o)
    close(dw[keep], want[keep], mag[keep], max(counts), "wgrad")
    want, mag = want_rows(x0, w, o, False)
    close(y[own], want[own.cuda()], mag[own.cuda()], k, "rows")


def test_weights_of_others_do_not_leak():
    from mole_b200 import ops
    for dtype, (k, n), kn in itertools.product((BF16, F32), ((136, 264), (33, 40)), (False, True)):
        x, w = rnd(64, k, dtype=dtype), rnd(4, *((k, n) if kn else (n, k)), seed=1, dtype=dtype)
        w[1], w[3] = float("nan"), float("inf")
        o = offs([30, 0, 34, 0])
        y = ops.grouped_mm(x, w, o, w_kn=kn)
        w[1], w[3] = 0, 0
        close(y, *want_rows(x, w, o, kn), k, f"{dtype} {k} {n} {kn}")


def test_offsets_out_of_order_or_range_are_clamped():
    from mole_b200 import ops
    for dtype, k in ((BF16, 64), (BF16, 33), (F32, 20)):
        x, w = rnd(50, k, dtype=dtype), rnd(3, 40, k, seed=1, dtype=dtype)
        bad = torch.tensor([5, 2, 40, 100000], dtype=torch.int32, device="cuda")
        meant = torch.tensor([5, 5, 40, 50], dtype=torch.int32, device="cuda")
        assert torch.equal(ops.grouped_mm(x, w, bad), ops.grouped_mm(x, w, meant))
        assert torch.equal(ops.grouped_mm_wgrad(x, x, bad), ops.grouped_mm_wgrad(x, x, meant))
        below = torch.tensor([-7, -1, 3, -5], dtype=torch.int32, device="cuda")
        meant = torch.tensor([0, 0, 3, 3], dtype=torch.int32, device="cuda")
        assert torch.equal(ops.grouped_mm(x, w, below), ops.grouped_mm(x, w, meant))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [1, 4])
def test_pointers_off_their_alignment(dtype, shift):
    from mole_b200 import ops

    def put(t):
        big = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")
        big[shift:] = t.flatten()
        return big[shift:].view(t.shape)
    x, w, b = rnd(70, 128, dtype=dtype), rnd(3, 64, 128, seed=1, dtype=dtype), rnd(70, 64, seed=2, dtype=dtype)
    o = offs([20, 0, 50])
    y, m = want_rows(x, w, o, False)
    out = put(torch.zeros(70, 64, dtype=dtype, device="cuda"))
    for args in ((put(x), w), (x, put(w)), (put(x), put(w))):
        close(ops.grouped_mm(*args, o), y, m, 128, "rows")
    close(ops.grouped_mm(x, w, o, out=out), y, m, 128, "out")
    want, mag = want_wgrad(b, x, o)
    close(ops.grouped_mm_wgrad(put(b), x, o), want, mag, 50, "wgrad")
    close(ops.grouped_mm_wgrad(b, put(x), o, out=put(torch.zeros(3, 64, 128, dtype=dtype, device="cuda"))), want, mag,
          50, "wgrad out")


def test_same_bits_every_time():
    from mole_b200 import ops
    o = offs([1000, 3, 0, 700])
    x, b, w = rnd(1703, 512, dtype=BF16), rnd(1703, 256, seed=1, dtype=BF16), rnd(4, 256, 512, seed=2, dtype=BF16)
    ys = [ops.grouped_mm(x, w, o) for _ in range(3)]
    gs = [ops.grouped_mm_wgrad(b, x, o) for _ in range(3)]
    assert all(torch.equal(ys[0], y) for y in ys) and all(torch.equal(gs[0], g) for g in gs)


# ---- gradients ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kn", [False, True])
@pytest.mark.parametrize("dtype,k,n", [(BF16, 128, 264), (BF16, 33, 20), (F32, 48, 40)])
def test_gradients(dtype, k, n, kn):
    import mole_b200
    counts, tail = [7, 0, 64, 129], 11
    o = offs(counts)
    R = sum(counts) + tail
    x = rnd(R, k, dtype=dtype).requires_grad_()
    w = rnd(4, *((k, n) if kn else (n, k)), seed=1, dtype=dtype).requires_grad_()
    dy = rnd(R, n, seed=2, dtype=dtype)
    y = mole_b200.grouped_mm(x, w, o, w_kn=kn)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    close(dx, *want_rows(dy, w.detach(), o, not kn), n, "dx")
    close(dw, *(want_wgrad(x.detach(), dy, o) if kn else want_wgrad(dy, x.detach(), o)), max(counts), "dw")
    assert not dx[R - tail:].any()
    # one gradient alone, an expanded dy, and dy that is not contiguous
    assert torch.equal(torch.autograd.grad(y, w, dy, retain_graph=True)[0], dw)
    assert torch.equal(torch.autograd.grad(y, x, dy.t().contiguous().t(), retain_graph=True)[0], dx)
    (g1,) = torch.autograd.grad(y.sum(), x)
    close(g1, *want_rows(torch.ones_like(dy), w.detach(), o, not kn), n, "dx of a sum")


def test_second_derivatives_are_refused():
    import mole_b200
    x, w, o = rnd(10, 16).requires_grad_(), rnd(2, 8, 16, seed=1).requires_grad_(), offs([4, 6])
    y = mole_b200.grouped_mm(x, w, o)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    y = mole_b200.grouped_mm(x, w, o)
    with torch.no_grad():
        w.mul_(2)                                     # what backward needs has been changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert not mole_b200.grouped_mm(x.detach(), w.detach(), o).requires_grad
    with torch.no_grad():
        assert not mole_b200.grouped_mm(x, w, o).requires_grad


def test_gradients_against_differences():
    """fp32: the product is bilinear, so a central difference along a direction is its derivative up to
    the rounding of two values: each is off by (K + 2) 2^-24 sum |x w| |dy|, over a step of 2^-3."""
    import mole_b200
    o = offs([9, 0, 30])
    x, w, dy = rnd(39, 24), rnd(3, 16, 24, seed=1), rnd(39, 16, seed=2)
    ux, uw = rnd(39, 24, seed=3), rnd(3, 16, 24, seed=4)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(mole_b200.grouped_mm(xr, wr, o), (xr, wr), dy)
    f = lambda a, b: (mole_b200.grouped_mm(a, b, o).double() * dy.double()).sum()  # noqa: E731
    h = 0.125
    mag = (want_rows(x.abs() + ux.abs(), w.abs() + uw.abs(), o, False)[1] * dy.double().abs()).sum()
    tol = 2 * 26 * 2.0 ** -24 * mag / h
    assert abs((f(x + h * ux, w) - f(x - h * ux, w)) / (2 * h) - (dx.double() * ux.double()).sum()) < tol
    assert abs((f(x, w + h * uw) - f(x, w - h * uw)) / (2 * h) - (dw.double() * uw.double()).sum()) < tol


# ---- 8-bit integers --------------------------------------------------------------------------------------
def want_quantized(x):
    top = x.float().abs().amax(-1)
    scale = (top.double() / 127).float()
    q = torch.where(scale[..., None] > 0, torch.round(x.double() / scale[..., None].double()), 0.0)
    return q.clamp(-127, 127).to(torch.int8), scale


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (1, 2048), (300, 264), (17, 1000), (4, 33, 72), (2, 8200),
                                   (70000, 16)])
def test_quantize_rows_is_the_nearest_integer(dtype, shape):
    from mole_b200 import ops
    x = rnd(*shape, dtype=dtype) * torch.exp(rnd(*shape[:-1], 1, seed=1)).to(dtype)
    x.view(-1)[:5] = 0
    q, s = ops.quantize_rows(x)
    wq, ws = want_quantized(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)


def test_quantize_rows_ties_and_extremes():
    from mole_b200 import ops
    # scale 1 exactly (127 in the row): every half is a tie and goes to the even integer
    x = torch.arange(-254, 255, device="cuda").float()[None] / 2
    q, s = ops.quantize_rows(x)
    assert s.item() == 1 and torch.equal(q, torch.round(x).to(torch.int8))
    # next to ties by one unit of fp32, for scales that are no power of two
    for seed in range(20):
        s0 = torch.rand(1, device="cuda") + 0.3
        n = torch.arange(0, 126, device="cuda").float() + 0.5
        near = (n.double() * s0.double()).float()
        row = torch.cat([near, torch.nextafter(near, near * 2), torch.nextafter(near, near * 0), -near, s0 * 127])[None]
        q, s = ops.quantize_rows(row)
        wq, ws = want_quantized(row)
        assert torch.equal(q, wq) and torch.equal(s, ws)
    big = torch.finfo(F32).max
    x = torch.stack([torch.full((64,), v, device="cuda") for v in (0.0, big, -big, 1e-38, 1e-30, 3e-43)])
    x[:, ::2] *= 0.3
    q, s = ops.quantize_rows(x)
    wq, ws = want_quantized(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)
    x = rnd(4, 64)
    x[1, 3], x[2, 5], x[3, 60] = float("nan"), float("inf"), float("-inf")
    q, s = ops.quantize_rows(x)
    assert torch.isfinite(s).tolist() == [True, False, False, False] and not q[1:].any()
    y = ops.mm_int8(q, s, *ops.quantize_rows(rnd(10, 64, seed=1)), out_dtype=F32)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1:]).all()


def want_int8(q, qs, w, ws, offsets, dtype):
    y = torch.zeros(q.shape[0], w.shape[1], dtype=F32, device=q.device)
    for e, (a, b) in enumerate(spans(offsets)):
        if b > a:
            acc = (q[a:b].double() @ w[e].double().t()).float()           # exact in 64 bits, rounded once
            y[a:b] = (acc * qs[a:b, None]) * ws[e]
    return y.to(dtype)


def int8s(*shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).cuda()


@pytest.mark.parametrize("groups", GROUPS)
@pytest.mark.parametrize("k,n", [(1, 1), (7, 5), (16, 16), (48, 40), (64, 1001), (144, 264), (272, 136), (1024, 512)])
def test_int8_products_are_exact(k, n, groups):
    from mole_b200 import ops
    counts, head, tail = GROUPS[groups]
    o, R, E = offs(counts, head), head + sum(counts) + tail, len(counts)
    q, w = int8s(R, k, seed=1), int8s(E, n, k, seed=2)
    qs, ws = torch.rand(R, device="cuda") + 0.1, torch.rand(E, n, device="cuda") + 0.1
    if head:
        qs[:head] = float("nan")                       # rows of nobody: zeros whatever their scale
    for dtype in (BF16, F32):
        y = ops.grouped_mm_int8(q, qs, w, ws, o, out_dtype=dtype)
        assert torch.equal(y, want_int8(q, qs, w, ws, o, dtype))


@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 129])
@pytest.mark.parametrize("k,n", [(2048, 1024), (8192, 104), (4112, 33)])
def test_int8_dense_and_few_rows(rows, k, n):
    from mole_b200 import ops
    q, w = int8s(rows, k, seed=1), int8s(n, k, seed=2)
    qs, ws = torch.rand(rows, device="cuda"), torch.rand(n, device="cuda")
    o = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    want = want_int8(q, qs, w[None], ws[None], o, F32)
    assert torch.equal(ops.mm_int8(q, qs, w, ws, out_dtype=F32), want)
    assert torch.equal(ops.grouped_mm_int8(q, qs, w[None], ws[None], o, out_dtype=F32), want)


def test_int8_sums_use_all_32_bits():
    """All products at their largest: 131071 times -128 times -128 is 2^31 - 2^14."""
    from mole_b200 import ops
    for k, rows in itertools.product((131071, 131056), (3, 20)):
        q, w = (torch.full((n, k), -128, dtype=torch.int8, device="cuda") for n in (rows, 5))
        ones = torch.ones(20, device="cuda")
        y = ops.mm_int8(q, ones[:rows], w, ones[:5], out_dtype=F32)
        assert (y == torch.tensor(k * 16384.0)).all()
        y = ops.mm_int8(q, ones[:rows], torch.full_like(w, 127), ones[:5], out_dtype=F32)
        assert (y == torch.tensor(float(-k * 128 * 127))).all()


# ---- together, as they are used ----------------------------------------------------------------------------
def _dropless(x, gate_w, w1, w2, k):
    """A layer without capacity: route, pack, both products, combine; returns also what packs the rows."""
    import mole_b200
    from mole_b200 import ops
    T, E = x.shape[0], gate_w.shape[0]
    plan = ops.gate_route(x.detach(), gate_w, k, T)               # capacity T: nothing is dropped
    rows = plan.perm.long() // k
    h = torch.nn.functional.gelu(mole_b200.grouped_mm(x[rows], w1, plan.offsets))
    y = mole_b200.grouped_mm(h, w2, plan.offsets, w_kn=True)
    g = plan.gates.flatten()[plan.perm.long()].to(y.dtype)
    return torch.zeros_like(x).index_add_(0, rows, y * g[:, None]), plan, rows


def test_a_layer_without_capacity_trains_and_serves():
    from mole_b200 import MOLEModule, ops
    from mole_b200.optim import DeviceAdam
    T, M, F, E, k = 600, 128, 256, 8, 2
    x, gate_w = rnd(T, M), rnd(E, M, seed=1, std=0.1)
    w1 = torch.nn.Parameter(rnd(E, F, M, seed=2, std=0.05))
    w2 = torch.nn.Parameter(rnd(E, F, M, seed=3, std=0.05))
    gy = rnd(T, M, seed=4)
    xr = x.clone().requires_grad_()
    y, plan, rows = _dropless(xr, gate_w, w1, w2, k)
    y.backward(gy)
    # the framework's layer with room for every token computes the same function
    m = MOLEModule(0, E, M, F, -1, k, E, {"local_rank": 0, "world_size": 1, "rank": 0}, "gelu", 1, False, False, dtype=F32)
    zero = lambda n: torch.zeros(n)  # noqa: E731
    m.set_layer_state({"gate": [gate_w.cpu(), None],
                       "experts": [[w1[e].detach().cpu(), zero(F), w2[e].detach().cpu(), zero(M)] for e in range(E)]}, False)
    xl = x.clone().requires_grad_()
    yl = m(xl, capacity_factor=float(E))
    yl.backward(gy)
    for a, b in ((y, yl), (w1.grad, m.FC1_W_GPU.grad_tensors), (w2.grad, m.FC2_W_GPU.grad_tensors)):
        # both are fp32 sums of up to T + F + M products in their own order
        assert (a - b).abs().max() <= (T + F + M) * 2.0 ** -23 * 4 * b.abs().max()
    # a step of the optimizer with 8-bit moments moves the weights by about lr each
    before = w1.detach().clone()
    DeviceAdam([w1, w2], lr=1e-3, weight_decay=0.0, state_bits=8).step()
    moved = (w1.detach() - before).abs()
    live = w1.grad.abs() > 1e-4
    assert live.any() and ((moved[live] - 1e-3).abs() < 2e-5).all()
    # serving from 8 bits: first product against the same product of the unrounded operands; |q s - x| is
    # at most half a scale, for tokens and for weights
    q1, s1 = ops.quantize_rows(w1.detach())
    xp = x[rows]
    qx, sx = ops.quantize_rows(xp)
    h8 = ops.grouped_mm_int8(qx, sx, q1, s1, plan.offsets, out_dtype=F32)
    h = ops.grouped_mm(xp, w1.detach(), plan.offsets)
    o = plan.offsets.tolist()
    for e in range(E):
        a, b = o[e], o[e + 1]
        bound = 0.5 * xp[a:b].abs().sum(1)[:, None] * s1[e] + 0.5 * sx[a:b, None] * (w1[e].detach().abs().sum(1) + M * s1[e] / 2)
        assert ((h8[a:b] - h[a:b]).abs() <= bound * 1.001).all()


def test_on_another_stream_and_two_at_once():
    from mole_b200 import ops
    o = offs([100, 0, 412])
    x, w = rnd(512, 256, dtype=BF16), rnd(3, 512, 256, seed=1, dtype=BF16)
    want = ops.grouped_mm(x, w, o)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([ops.grouped_mm(x, w, o) for _ in range(5)] + [ops.grouped_mm_wgrad(want, x, o)])
    torch.cuda.synchronize()
    assert all(torch.equal(want, y) for ys in outs for y in ys[:5]) and torch.equal(outs[0][5], outs[1][5])


@pytest.mark.parametrize("rows", [9, 700, 5000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_calls_back_to_back_see_what_the_one_before_wrote(dtype, rows):
    """Inputs rewritten and outputs consumed right before and behind each call, without a pause, give the bits
    that the same calls give one at a time."""
    from mole_b200 import ops
    E, K, N = 5, 256, 512
    w1, w2 = rnd(E, N, K, seed=1, dtype=dtype, std=0.06), rnd(E, K, N, seed=2, dtype=dtype, std=0.06)
    q1, s1 = ops.quantize_rows(w1)
    news = [rnd(rows, K, seed=10 + i, dtype=dtype) for i in range(8)]
    cuts = [offs([(rows * c) // 40 for c in (i, 8, 2 * i, 0, 16 - i)], head=i) for i in range(8)]

    def chain(pause):
        x, o = torch.empty_like(news[0]), torch.empty_like(cuts[0])
        outs = []
        for xi, oi in zip(news, cuts):
            x.copy_(xi)
            o.copy_(oi)
            for f in (lambda: ops.grouped_mm(x, w1, o), lambda: ops.grouped_mm(outs[-1], w2, o),
                      lambda: ops.grouped_mm(outs[-1], w2, o, w_kn=True), lambda: ops.grouped_mm_wgrad(outs[-1], x, o),
                      lambda: ops.grouped_mm(outs[-4], outs[-1], o, w_kn=True),
                      lambda: ops.quantize_rows(outs[-4])):
                if pause:
                    torch.cuda.synchronize()
                got = f()
                outs += got if isinstance(got, tuple) else [got]
            if pause:
                torch.cuda.synchronize()
            outs.append(ops.grouped_mm_int8(outs[-2], outs[-1], q1, s1, o, out_dtype=dtype))
            if pause:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs
    chain(False)
    want, got = chain(True), chain(False)
    assert len(got) == 8 * 8 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed_with_new_rows_and_offsets():
    import mole_b200
    from mole_b200 import ops
    from mole_b200.utils.Ugraph import GraphedStep
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = offs([100, 28, 0, 50])
        x = rnd(200, 128, dtype=BF16).requires_grad_()
        w = rnd(4, 256, 128, seed=1, dtype=BF16).requires_grad_()
        dy = rnd(200, 256, seed=2, dtype=BF16)
        wq, ws = ops.quantize_rows(w.detach())

    def step():
        y = mole_b200.grouped_mm(x, w, o)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        return y.detach(), dx, dw, ops.grouped_mm_int8(*ops.quantize_rows(x.detach()), wq, ws, o)
    graph = GraphedStep(step, side)
    with torch.no_grad():
        x.copy_(rnd(200, 128, seed=7, dtype=BF16))
        o.copy_(offs([0, 3, 190, 7]))
    got = [t.clone() for t in graph()]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows():
    from mole_b200 import ops
    o = offs([0, 0])
    x, w = torch.empty(0, 64, dtype=BF16, device="cuda"), rnd(2, 32, 64, dtype=BF16)
    assert ops.grouped_mm(x, w, o).shape == (0, 32)
    dw = ops.grouped_mm_wgrad(torch.empty(0, 32, dtype=BF16, device="cuda"), x, o)
    assert dw.shape == (2, 32, 64) and not dw.any()
    q, s = ops.quantize_rows(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    assert ops.grouped_mm_int8(q, s, *ops.quantize_rows(w), o).shape == (0, 32)


def test_refusals():
    from mole_b200 import ops
    x, w, o = rnd(10, 16), rnd(2, 8, 16), offs([4, 6])
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(w)
    for exc, match, call in (
            (ValueError, "offsets must be int32", lambda: ops.grouped_mm(x, w, o.long())),
            (ValueError, "offsets must be int32", lambda: ops.grouped_mm(x, w, o[:2])),
            (ValueError, "width", lambda: ops.grouped_mm(x, w, o, w_kn=True)),
            (TypeError, "one dtype", lambda: ops.grouped_mm(x, w.bfloat16(), o)),
            (TypeError, "unsupported dtype", lambda: ops.grouped_mm(x.half(), w.half(), o)),
            (ValueError, "takes x", lambda: ops.grouped_mm(x, w[0], o)),
            (RuntimeError, "contiguous", lambda: ops.grouped_mm(x.t().contiguous().t(), w, o)),
            (ValueError, "different devices", lambda: ops.grouped_mm(x, w, o.cpu())),
            (RuntimeError, "CUDA tensors", lambda: ops.grouped_mm(x.cpu(), w.cpu(), o.cpu())),
            (ValueError, "out must be", lambda: ops.grouped_mm(x, w, o, out=x)),
            (ValueError, "overlaps", lambda: ops.grouped_mm(x, rnd(2, 16, 16), o, out=x)),
            (ValueError, "takes a", lambda: ops.grouped_mm_wgrad(x, x[:5], o)),
            (ValueError, "out must be", lambda: ops.grouped_mm_wgrad(x, x, o, out=w)),
            (TypeError, "int8", lambda: ops.grouped_mm_int8(x, s, wq, ws, o)),
            (ValueError, "q_scale", lambda: ops.grouped_mm_int8(q, s[:3], wq, ws, o)),
            (ValueError, "w_scale", lambda: ops.grouped_mm_int8(q, s, wq, ws[0], o)),
            (TypeError, "unsupported dtype", lambda: ops.mm_int8(q, s, wq[0], ws[0], out_dtype=torch.float16)),
            (ValueError, "at least one element", lambda: ops.quantize_rows(x[:, :0])),
            (TypeError, "unsupported dtype", lambda: ops.quantize_rows(q)),
            (RuntimeError, "E=300", lambda: ops.grouped_mm(x, rnd(300, 8, 16), offs([0] * 300)))):
        with pytest.raises(exc, match=match):
            call()
