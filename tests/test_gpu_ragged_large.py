"""Products over packed rows at sizes where a pair of SMs takes 512 features with two accumulators: many
experts, wide outputs, row counts on both sides of half a panel, so that a pair's items use one
accumulator, both, and one again.  Tolerances as in ``test_gpu_ragged.py``: against 64 bits on the same
inputs a sum of L products is off by at most (L + 2) 2^-23 sum |a b|, the stored value by half a step more;
integer products are exact."""
import pytest
import torch

from test_gpu_ragged import BF16, F32, close, int8s, offs, rnd, spans, want_int8, want_rows, want_wgrad

pytestmark = pytest.mark.gpu

# rows per expert: none, one, less than half a panel, a step more than half, a panel, two panels of which the
# second is below half (257, 270), more than two
MIXED = [(0, 1, 100, 129, 200, 300, 257, 16, 128, 270)[i % 10] for i in range(39)] + [1100]
SMALL = [(0, 1, 2, 5, 17, 31)[i % 6] for i in range(60)]


def takes_512_features(counts, head, tail, n):
    """The rule by which the kernel with 512 features per pair is chosen (panels of 256 rows)."""
    R, E = head + sum(counts) + tail, len(counts)
    panels = R // 256 + min(E, R)
    return panels * (-(-n // 512)) >= torch.cuda.get_device_properties(0).multi_processor_count and (n % 512 == 0 or n > 1024)


CASES = [(MIXED, 3, 70, 192, 2048), (MIXED, 0, 0, 1000, 2048), (MIXED, 0, 5, 64, 1544), (MIXED, 37, 0, 2048, 2056),
         (SMALL, 0, 1, 1096, 2048), (SMALL, 5, 90, 328, 1536), (MIXED, 0, 9, 33, 2048)]


def poisoned(x, head, tail, o, e):
    """NaN into the rows of expert e, infinities into those of nobody."""
    R = x.shape[0]
    x[:head], x[R - tail:] = float("inf"), float("nan")
    x[o[e]:o[e + 1]] = float("nan")
    own = torch.ones(R, dtype=torch.bool, device="cuda")
    own[:head] = own[R - tail:] = False
    own[o[e]:o[e + 1]] = False
    return own


@pytest.mark.parametrize("counts,head,tail,k,n", CASES)
@pytest.mark.parametrize("kn", [False, True])
def test_products_of_512_features(kn, counts, head, tail, k, n):
    from mole_b200 import ops
    assert takes_512_features(counts, head, tail, n)
    o, R, E = offs(counts, head), head + sum(counts) + tail, len(counts)
    x, w = rnd(R, k, seed=1, dtype=BF16), rnd(E, *((k, n) if kn else (n, k)), seed=2, dtype=BF16)
    bad = counts.index(max(counts))
    own = poisoned(x, head, tail, o.tolist(), bad)
    w[[i for i, c in enumerate(counts) if c == 0]] = float("nan")     # experts without rows
    y = ops.grouped_mm(x, w, o, w_kn=kn)
    assert not y[:head].any() and not y[R - tail:].any()
    assert torch.isnan(y[o[bad]:o[bad + 1]]).all()
    want, mag = want_rows(x, w, o, kn)
    close(y[own], want[own], mag[own], k, f"kn={kn}")
    for _ in range(3):
        assert torch.equal(y[own], ops.grouped_mm(x, w, o, w_kn=kn)[own])
    # an output whose rows do not start on 16 bytes is stored another way
    if n % 8 == 0:
        out = torch.empty(R * n + 1, dtype=BF16, device="cuda")[1:].view(R, n)
        assert torch.equal(y[own], ops.grouped_mm(x, w, o, w_kn=kn, out=out)[own])


@pytest.mark.parametrize("k,n", [(192, 2048), (1024, 2056)])
def test_gradients_of_512_features(k, n):
    """dx runs over n with k outputs: 512 features there too where k allows it; dw over the rows."""
    import mole_b200
    for kn in (False, True):
        o, R, E = offs(MIXED, 2), 2 + sum(MIXED) + 40, len(MIXED)
        x = rnd(R, k, seed=1, dtype=BF16).requires_grad_()
        w = rnd(E, *((k, n) if kn else (n, k)), seed=2, dtype=BF16).requires_grad_()
        dy = rnd(R, n, seed=3, dtype=BF16)
        dx, dw = torch.autograd.grad(mole_b200.grouped_mm(x, w, o, w_kn=kn), (x, w), dy)
        close(dx, *want_rows(dy, w.detach(), o, not kn), n, "dx")
        close(dw, *(want_wgrad(x.detach(), dy, o) if kn else want_wgrad(dy, x.detach(), o)), max(MIXED), "dw")
        assert not dx[:2].any() and not dx[R - 40:].any()


@pytest.mark.parametrize("counts,head,tail,k,n", CASES)
def test_int8_products_of_512_features(counts, head, tail, k, n):
    from mole_b200 import ops
    assert takes_512_features(counts, head, tail, n)
    o, R, E = offs(counts, head), head + sum(counts) + tail, len(counts)
    q, w = int8s(R, k, seed=1), int8s(E, n, k, seed=2)
    qs, ws = torch.rand(R, device="cuda") + 0.1, torch.rand(E, n, device="cuda") + 0.1
    qs[:head], qs[R - tail:] = float("nan"), float("inf")
    for dtype in (BF16, F32):
        assert torch.equal(ops.grouped_mm_int8(q, qs, w, ws, o, out_dtype=dtype), want_int8(q, qs, w, ws, o, dtype))


def test_captured_and_replayed_with_other_offsets():
    """The grid stays, the panels move: from MIXED to one expert with everything, to many small ones."""
    from mole_b200 import ops
    R, E, k, n = sum(MIXED) + 11, len(MIXED), 320, 2048
    x, w = rnd(R, k, seed=1, dtype=BF16), rnd(E, n, k, seed=2, dtype=BF16)
    q, w8 = int8s(R, k, seed=3), int8s(E, n, k, seed=4)
    qs, ws = torch.rand(R, device="cuda") + 0.1, torch.rand(E, n, device="cuda") + 0.1
    o = offs(MIXED, 0)
    step = lambda: (ops.grouped_mm(x, w, o), ops.grouped_mm_int8(q, qs, w8, ws, o), ops.grouped_mm_wgrad(x, x, o))  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    layouts = [[0] * 7 + [R] + [0] * (E - 8), [i % 5 for i in range(E)], MIXED[::-1], [0] * E, MIXED]
    for counts in layouts:
        o.copy_(offs(counts, 0))
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        want, mag = want_rows(x, w, o, False)
        close(got[0], want, mag, k, "replayed")
        assert [b - a for a, b in spans(o)] == counts
    torch.cuda.synchronize()
    assert ops.device_fault() == 0
