"""A step's own codes for moments that are not finite are those that ``pack_moment`` makes of them on load."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_step_and_a_load_hold_lost_elements_alike():
    """A fresh state, so that m = (1 - beta1) g and sqrt(v) = sqrt(1 - beta2) |g|: block 0 has other values, block 1
    is zeros but for one infinity, block 2 has a NaN as well."""
    from mole_b200 import ops
    from mole_b200.optim.device_adam import pack_moment, unpack_moment
    n, inf, nan = 768, float("inf"), float("nan")
    g = torch.randn(n, generator=torch.Generator().manual_seed(3)).cuda()
    g[256:512] = 0
    g[5], g[300], g[520], g[530] = -inf, inf, nan, inf
    p, zeros = torch.ones(n, device="cuda"), lambda: torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    m, v, ms, vs = zeros(), zeros(), torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    ops.adam_multi([p], [g], [m], [v], [ms], [vs], t=1, lr=1e-3)
    lost = ~g.isfinite()
    for codes, scale, square, value in ((m, ms, False, 0.1 * g), (v, vs, True, 0.001 * g.square())):
        want, want_scale = pack_moment(value, square)
        assert ((scale - want_scale).abs() <= 2.0 ** -20 * want_scale).all() and scale[1] == 0
        assert torch.equal(codes.float()[lost].nan_to_num(nan=999), want.float()[lost].nan_to_num(nan=999))
        assert codes.float()[300].isnan() and codes.float()[520].isnan()
        got = unpack_moment(codes, scale, square)
        assert got[~lost].isfinite().all() and not got[256:300].any() and not got[301:512].any()
        # one step of a code up or down: 2^-3 of the value (2^-2 and its square in v), 2^-9 of 448ths of the top
        top = want_scale.repeat_interleave(256) * 448
        top = top.square() if square else top
        near = (0.27 if square else 0.126) * value.abs() + (2.0 ** -9 / 448) * 1.01 * top
        assert ((got - value).abs() <= near)[~lost].all()
    assert p[~lost].isfinite().all()
