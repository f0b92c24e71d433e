"""A given output that shares memory with anything the product reads is refused: tiles are written while others
are still to be computed."""
import pytest
import torch

from test_gpu_ragged import F32, offs, rnd

pytestmark = pytest.mark.gpu
R, E, N, K = 40, 3, 24, 32


def test_outputs_over_offsets_and_scales():
    from mole_b200 import ops
    o = offs([10, 0, 30])
    x, w = rnd(R, K), rnd(E, N, K, seed=1)
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(w)
    buf = torch.zeros(4000, device="cuda")

    def there(t, at):
        """The same values inside the buffer."""
        view = buf[at:at + t.numel()].view(t.dtype).view(t.shape)
        view.copy_(t)
        return view
    out = buf[100:100 + R * N].view(R, N)
    dw = buf[100:100 + E * N * K].view(E, N, K)
    for at in (100, 99, 100 + R * N - 1):               # inside, across the first element, the last one
        for call in (lambda: ops.grouped_mm(x, w, there(o, at), out=out),
                     lambda: ops.grouped_mm_int8(q, s, wq, ws, there(o, at), out_dtype=F32, out=out),
                     lambda: ops.grouped_mm_int8(q, there(s, at), wq, ws, o, out_dtype=F32, out=out),
                     lambda: ops.grouped_mm_int8(q, s, wq, there(ws, at), o, out_dtype=F32, out=out),
                     lambda: ops.mm_int8(q, there(s, at), wq[0], ws[0], out_dtype=F32, out=out),
                     lambda: ops.mm_int8(q, s, wq[0], there(ws[0], at), out_dtype=F32, out=out)):
            with pytest.raises(ValueError, match="overlaps an operand"):
                call()
    for at in (100, 99, 100 + E * N * K - 1):
        with pytest.raises(ValueError, match="overlaps an operand"):
            ops.grouped_mm_wgrad(rnd(R, N), x, there(o, at), out=dw)
    # right behind the output, and right before it
    want = ops.grouped_mm_int8(q, s, wq, ws, o, out_dtype=F32)
    end = 100 + R * N
    got = ops.grouped_mm_int8(q, there(s, 100 - R), wq, there(ws, end), there(o, end + E * N), out_dtype=F32, out=out)
    assert torch.equal(got, want)
