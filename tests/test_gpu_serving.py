"""Both products of an expert from 8-bit weights, as the documentation writes them down."""
import pytest
import torch

from test_gpu_ragged import BF16, F32, offs, rnd, want_int8, want_quantized

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("counts", [[1, 0, 2, 1], [40, 0, 7, 300]])
def test_both_products_from_8_bits(dtype, counts):
    from mole_b200 import ops
    E, M, F = len(counts), 72, 200
    o, x = offs(counts), rnd(sum(counts) + 3, M, dtype=dtype)
    w1, w2 = rnd(E, F, M, seed=1, dtype=dtype, std=0.1), rnd(E, F, M, seed=2, dtype=dtype, std=0.1)
    q1, s1 = ops.quantize_rows(w1)
    q2, s2 = ops.quantize_rows(w2.transpose(1, 2).contiguous())
    assert q2.shape == (E, M, F) and s2.shape == (E, M)
    h = torch.nn.functional.gelu(ops.grouped_mm_int8(*ops.quantize_rows(x), q1, s1, o, out_dtype=dtype))
    y = ops.grouped_mm_int8(*ops.quantize_rows(h), q2, s2, o, out_dtype=dtype)
    # integers and scales restated: the same bits
    want_h = torch.nn.functional.gelu(want_int8(*want_quantized(x), *want_quantized(w1), o, dtype))
    want = want_int8(*want_quantized(want_h), *want_quantized(w2.transpose(1, 2)), o, dtype)
    assert torch.equal(h, want_h) and torch.equal(y, want)
    assert not y[sum(counts):].any()
