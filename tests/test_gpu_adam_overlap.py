"""``ops.adam_multi`` refuses lists in which two of the tensors it writes share memory: thread blocks would race
on them.  Gradients are only read and may be shared."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
N = 600


def lists(bits, count=3):
    code = lambda: torch.zeros(N, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # noqa: E731
    flat = lambda n=N: torch.zeros(n, device="cuda")  # noqa: E731
    out = {"p": [flat() + 1 for _ in range(count)], "g": [flat() + 1 for _ in range(count)]}
    for k in ("m", "v"):
        out[k] = [flat() if bits == 32 else code() for _ in range(count)]
    for k in ("ms", "vs"):
        out[k] = [flat(3) for _ in range(count)] if bits == 8 else None
    return out


def go(s):
    from mole_b200 import ops
    ops.adam_multi(s["p"], s["g"], s["m"], s["v"], s["ms"], s["vs"], t=1, lr=0.1)


@pytest.mark.parametrize("bits", [32, 8])
def test_shared_moments_and_scales_are_refused(bits):
    names = ["p", "m", "v"] + (["ms", "vs"] if bits == 8 else [])
    for k in names:                                     # the same tensor for two parameters
        s = lists(bits)
        s[k][2] = s[k][0]
        before = s["p"][1].clone()
        with pytest.raises(ValueError, match="tensors [02] and [02].*twice"):
            go(s)
        assert torch.equal(s["p"][1], before)
    for a, b in itertools.combinations(names, 2):       # one list's tensor in another's place, where the types agree
        s = lists(bits)
        if s[a][0].dtype == s[b][1].dtype and s[a][0].numel() == s[b][1].numel():
            s[a][0] = s[b][1]
            with pytest.raises(ValueError, match="twice"):
                go(s)
            s = lists(bits)
            s[a][1] = s[b][1]
            with pytest.raises(ValueError, match="tensors 1 and 1.*twice"):
                go(s)


@pytest.mark.parametrize("order", list(itertools.permutations(range(3))))
def test_parts_of_one_buffer(order):
    """Views that touch are fine in any order; views that overlap by one element are not."""
    from mole_b200 import ops
    big, s = torch.ones(3 * N, device="cuda"), lists(32)
    s["p"] = [big[N * i:N * (i + 1)] for i in order]
    go(s)
    alone = lists(32)
    go(alone)
    assert torch.equal(big[:N], alone["p"][0]) and torch.equal(big[2 * N:], alone["p"][0])
    s["p"][order.index(1)] = big[N - 1:2 * N - 1]
    with pytest.raises(ValueError, match="twice"):
        go(s)
    empty = torch.zeros(0, device="cuda")               # tensors without elements share nothing
    ops.adam_multi([empty, empty], [empty, empty], [empty, empty], [empty, empty], t=1, lr=0.1)


def test_a_shared_gradient_is_only_read():
    s, want = lists(32), lists(32)
    s["g"] = [s["g"][0]] * 3
    go(s)
    go(want)
    assert all(torch.equal(a, b) for a, b in zip(s["p"], want["p"]))
