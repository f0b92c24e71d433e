"""Argument checks of the operators on packed rows and on lists of tensors, which come before any
device work: the C entries are called with addresses that are never read."""
import ctypes as C

import pytest
import torch

A = 1 << 20          # an address aligned to anything; nothing is launched


def status(rc):
    from mole_b200 import _lib
    return rc, _lib.lib.mole_last_error_string().decode()


@pytest.mark.parametrize("R,N,K,E,dtype,code", [
    (10, 0, 8, 2, 1, -1), (10, 8, 0, 2, 1, -1), (10, 8, 8, 0, 1, -1), (10, 8, 8, 257, 1, -1),
    (-1, 8, 8, 2, 1, -1), (1 << 31, 8, 8, 2, 1, -1), (10, 8, 8, 2, 7, -1), (0, 8, 8, 2, 1, 0)])
def test_grouped_mm_sizes(R, N, K, E, dtype, code):
    from mole_b200 import _lib
    assert _lib.lib.mole_grouped_mm(A, A, A, R, N, K, E, 0, dtype, A, None, 0, None) == code
    if code:
        assert _lib.lib.mole_grouped_mm_wgrad(A, A, A, R, N, K, E, dtype, A, None, 0, None) == code


def test_null_and_misaligned_pointers():
    from mole_b200 import _lib
    lib = _lib.lib
    for bad in range(4):
        p = [A] * 4
        p[bad] = None
        assert status(lib.mole_grouped_mm(p[0], p[1], p[2], 4, 8, 8, 2, 0, 1, p[3], None, 0, None)) == (-1, "null pointer argument")
        p[bad] = A + 1
        rc, text = status(lib.mole_grouped_mm(p[0], p[1], p[2], 4, 8, 8, 2, 0, 1, p[3], None, 0, None))
        assert rc == -1 and "aligned" in text
    assert lib.mole_grouped_mm_wgrad(A, A, None, 0, 8, 8, 2, 1, A, None, 0, None) == -1
    assert lib.mole_quantize_rows(None, 3, 8, 1, A, A, None) == -1
    assert lib.mole_quantize_rows(A, 3, 0, 1, A, A, None) == -1
    assert lib.mole_quantize_rows(A, 0, 8, 1, A, A, None) == 0


def test_workspace_of_rows_that_do_not_start_on_16_bytes():
    from mole_b200 import _lib
    lib = _lib.lib
    n = C.c_int64()

    def size(x, w, R, N, K, E, kn, elem):
        assert lib.mole_grouped_mm_workspace_bytes(x, w, R, N, K, E, kn, elem, C.byref(n)) == 0
        return n.value
    up = lambda b: -(-b // 256) * 256  # noqa: E731
    assert size(A, A, 100, 33, 64, 3, 0, 2) == 0                 # only the reduction has to fit
    assert size(A, A, 100, 33, 64, 3, 1, 2) == up(3 * 64 * 40 * 2)
    assert size(A, A, 100, 64, 33, 3, 1, 2) == up(100 * 40 * 2)
    assert size(A, A, 100, 64, 33, 3, 0, 2) == up(100 * 40 * 2) + up(3 * 64 * 40 * 2)
    assert size(A + 2, A, 100, 64, 64, 3, 0, 2) == up(100 * 64 * 2)
    assert size(A, A, 100, 64, 24, 3, 0, 1) == up(100 * 32) + up(3 * 64 * 32)
    assert size(A, A, 16, 64, 33, 3, 0, 2) == 0 and size(A, A, 100, 64, 33, 3, 0, 4) == 0
    assert lib.mole_grouped_mm_workspace_bytes(A, A, 100, 64, 33, 3, 0, 3, C.byref(n)) == -1
    assert lib.mole_grouped_mm_wgrad_workspace_bytes(A, A, 100, 64, 33, 3, 1, C.byref(n)) == 0
    assert n.value == up(100 * 40 * 2)
    # too little of it
    rc, text = status(lib.mole_grouped_mm(A, A, A, 100, 64, 33, 3, 0, 1, A, None, 0, None))
    assert rc == -1 and "workspace" in text
    rc, text = status(lib.mole_grouped_mm_wgrad(A, A, A, 100, 64, 33, 3, 1, A, A, 100, None))
    assert rc == -1 and "workspace" in text
    rc, text = status(lib.mole_grouped_mm_i8(A, A, A, A, A, 100, 64, 24, 3, 0, A, A, 100, None))
    assert rc == -1 and "workspace" in text


def test_integer_products():
    from mole_b200 import _lib
    lib = _lib.lib
    rc, text = status(lib.mole_grouped_mm_i8(A, A, A, A, A, 4, 8, 1 << 17, 1, 0, A, None, 0, None))
    assert rc == -1 and "32 bits" in text
    rc, text = status(lib.mole_grouped_mm_i8(A, A, A, A, None, 4, 8, 16, 2, 0, A, None, 0, None))
    assert rc == -1 and "one expert" in text
    assert lib.mole_grouped_mm_i8(A, None, A, A, A, 4, 8, 16, 2, 0, A, None, 0, None) == -1
    assert lib.mole_grouped_mm_i8(A, A, A, A, None, 0, 8, 16, 1, 0, A, None, 0, None) == 0


def test_adam_list():
    from mole_b200 import _lib
    lib = _lib.lib

    def call(n=1, dtype=0, bits=32, b1=0.9, t=1, lr=1e-3, lam=0.0, eps=1e-8, **entry):
        e = {"p": A, "g": A, "m": A, "v": A, "m_scale": A, "v_scale": A, "n": 10, **entry}
        table = (_lib.AdamTensor * 1)(_lib.AdamTensor(**e))
        return status(lib.mole_adam_multi(table, n, dtype, bits, b1, 0.999, t, lr, lam, eps, 1, 0, None))
    for kw, word in (({"t": 0}, "step count"), ({"bits": 16}, "32 or 8"), ({"dtype": 3}, "dtype"), ({"b1": 1.0}, "beta1"),
                     ({"lr": float("nan")}, "lr="), ({"eps": -1.0}, "eps="), ({"n": -1}, "list"), ({"p": None}, "null"),
                     ({"bits": 8, "m_scale": None}, "scales"), ({"p": A + 2}, "aligned"), ({"m": A + 2}, "aligned")):
        if "n" in kw:
            rc, text = status(lib.mole_adam_multi(None, -1, 0, 32, 0.9, 0.999, 1, 1e-3, 0.0, 1e-8, 1, 0, None))
        else:
            rc, text = call(**kw)
        assert rc == -1 and word in text, (kw, text)
    e = (_lib.AdamTensor * 1)(_lib.AdamTensor(A, A, A, A, None, None, 1 << 34))
    assert lib.mole_adam_multi(e, 1, 0, 32, 0.9, 0.999, 1, 1e-3, 0.0, 1e-8, 1, 0, None) == -1


def test_python_checks_come_before_the_device():
    from mole_b200 import ops
    x, w = torch.zeros(4, 8), torch.zeros(2, 6, 8)
    o = torch.tensor([0, 2, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.grouped_mm(x, w, o)
    with pytest.raises(ValueError, match="offsets"):
        ops.grouped_mm(x, w, o.float())
    with pytest.raises(ValueError, match="rows of at least"):
        ops.quantize_rows(x[:, :0])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.quantize_rows(x)


def test_moments_survive_packing():
    """Codes and scales of values that are codes times a scale come back: the pair is what a checkpoint of
    fp32 moments turns into."""
    from mole_b200.optim.device_adam import pack_moment, unpack_moment
    g = torch.Generator().manual_seed(0)
    for n in (1, 255, 256, 1000):
        codes = (torch.randn(n, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        codes[::256] = torch.tensor(448.0).to(torch.float8_e4m3fn)
        scale = torch.rand(-(-n // 256), generator=g) + 0.1
        for square in (False, True):
            c = codes.float().abs().to(torch.float8_e4m3fn) if square else codes
            again, s2 = pack_moment(unpack_moment(c, scale, square), square)
            assert torch.equal(again.float(), c.float())
            assert ((s2 - scale).abs() <= 2.0 ** -22 * scale).all()
    c, s = pack_moment(torch.zeros(300), False)
    assert not c.float().any() and not s.any()
    c, s = pack_moment(torch.tensor([1.0, 1e-20, 0.0]), True)          # never zero unless it is
    assert c.float()[1] > 0 and c.float()[2] == 0
