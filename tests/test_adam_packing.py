"""Packing of fp32 moments into 8-bit codes on load: values that are not finite stay with their element."""
import pytest
import torch


@pytest.mark.parametrize("square", [False, True])
def test_values_that_are_not_finite_stay_with_their_element(square):
    """One NaN and one infinity in every block; the other 254 pack as without them (to zeros in the block of
    zeros), so that a checkpoint or torch's own state loses no more than the element that was lost."""
    from mole_b200.optim.device_adam import pack_moment, unpack_moment
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1000, generator=g)
    x[512:768] = 0
    if square:
        x = x.square()
    inf = float("inf")
    bad = x.clone()
    for b in range(4):
        bad[256 * b + 7], bad[256 * b + 100] = float("nan"), inf if square or b % 2 == 0 else -inf
        x[256 * b + 7] = x[256 * b + 100] = 0
    want, want_scale = pack_moment(x, square)
    got, scale = pack_moment(bad, square)
    assert torch.equal(scale, want_scale)
    hurt = ~bad.isfinite()
    assert torch.equal(got.float()[~hurt], want.float()[~hurt])
    values = unpack_moment(got, scale, square)
    assert values[bad.isnan()].isnan().all() and values[~hurt].isfinite().all()
    for b in (0, 1, 3):
        i = 256 * b + 100
        assert got.float()[i] == (448.0 if bad[i] > 0 else -448.0)
        top = x[256 * b:256 * (b + 1)].abs().max()       # held as the largest value of its block, within the scale's rounding
        assert abs(values[i].abs() / top - 1) < 2.0 ** -20
    assert values[612].isnan()                             # a block of zeros has no largest code to hold it as


def test_a_block_of_nothing_finite():
    from mole_b200.optim.device_adam import pack_moment
    codes, scale = pack_moment(torch.full((300,), float("nan")), False)
    assert codes.float().isnan().all() and not scale.any()
    codes, scale = pack_moment(torch.tensor([1e-35, float("inf"), 1e-36]), False)       # below 2^-100: held as zeros
    assert not codes.float()[[0, 2]].any() and codes.float()[1].isnan() and not scale.any()


def test_a_state_with_a_lost_element_loads_into_either_width():
    from mole_b200.optim import DeviceAdam
    p = torch.nn.Parameter(torch.zeros(600))
    ref = torch.optim.Adam([p])
    p.grad = torch.randn(600, generator=torch.Generator().manual_seed(2))
    ref.step()
    ref.state[p]["exp_avg"][3] = float("nan")
    ref.state[p]["exp_avg_sq"][300] = float("inf")
    from mole_b200.optim.device_adam import unpack_moment
    narrow = DeviceAdam([torch.nn.Parameter(torch.zeros(600))], state_bits=8)
    narrow.load_state_dict(ref.state_dict())
    st = narrow.state[narrow.param_groups[0]["params"][0]]
    for name, square, at in (("exp_avg", False, 3), ("exp_avg_sq", True, 300)):
        v, want = unpack_moment(st[name], st[name + "_scale"], square), ref.state[p][name]
        others = torch.ones(600, dtype=torch.bool)
        others[at] = False
        # half a step of a code, 2^-4 (twice that in a square), or half of the smallest, 2^-10 of 448ths of the top
        top = want[others].max()
        assert ((v - want).abs()[others] <= (2 ** -3 if square else 2 ** -4) * 1.1 * want.abs()[others] + 1e-5 * top).all()
    assert st["exp_avg"].float()[3].isnan() and st["exp_avg_sq"].float()[300] == 448
