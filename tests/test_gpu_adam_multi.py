"""One Adam step over many tensors (``ops.adam_multi``) and the optimizer over it (``DeviceAdam``,
``MOLEMixedAdam(state_bits=...)``).

The 32-bit form is compared with the formula in 64 bits, and every state and parameter with the same
operations in numpy's float32, each rounded by itself: the rounding of an 8-bit state up or down
depends on every bit, so nothing less says whether a code is right.  All bits have to be equal, but
for one value in a thousand that may be one unit of fp32 off (the kernel's root and quotient are
correctly rounded but for about one in 2^20) and, where that moves a value across its random
threshold, one code."""
import copy
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK, TOP = 256, np.float32(448)
HP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
f32 = np.float32


def mix(h):
    h = (h * 0x9E3779B1) & 0xffffffff
    h = ((h ^ (h >> 15)) * 0x85157AF5) & 0xffffffff
    return h ^ (h >> 13)


def random_words(n, seed, t, place):
    """Element i: step i % 8 + 1 of the congruential sequence that starts at the hash of i // 8."""
    key = mix((mix((mix(seed) + t) & 0xffffffff) + place) & 0xffffffff)
    out = np.empty(n, np.int64)
    for i in range(n):
        if i % 8 == 0:
            r = mix((i // 8 + key) & 0xffffffff)
        r = (r * 1664525 + 1013904223) & 0xffffffff
        out[i] = r
    return out


def round_codes(x, u, floor):
    """Values of one moment onto e4m3 codes by 16 random bits each; returns (values of the codes, scales)."""
    codes, scales = np.zeros_like(x), np.zeros(-(-len(x) // BLOCK), f32)
    for b in range(len(scales)):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        fin = np.abs(x[at][np.isfinite(x[at])])
        top = fin.max() if len(fin) else f32(0)
        if top < 2.0 ** -100:
            continue
        scales[b] = top * f32(1 / 448)
        y = x[at] * (TOP / top)
        a = np.abs(y)
        lift = np.where(a < f32(2 ** -6), f32(2 ** -6), f32(0))
        with np.errstate(invalid="ignore"):
            bits = (a + lift).view(np.uint32) + (u[at].astype(np.uint32) << np.uint32(4))
        r = (bits & np.uint32(0xFFF00000)).view(f32) - lift
        r = np.where(np.isnan(y), f32(np.nan), np.minimum(r, TOP))
        if floor:
            r = np.where((x[at] > 0) & (r < f32(2 ** -9)), f32(2 ** -9), r)
        codes[at] = np.copysign(r, y)
    return codes, scales


def step_f32(p, g, m, v, t, place, adamw, seed, bits, ms=None, vs=None):
    """One step in float32, operation by operation; m and v are code values with their scales for 8 bits."""
    n = len(p)
    b1, b2 = HP["betas"]
    lr, lam, eps = HP["lr"], HP["weight_decay"], HP["eps"]
    if bits == 8:
        rep = lambda s: np.repeat(s, BLOCK)[:n]  # noqa: E731
        m = m * rep(ms)
        v = v * rep(vs)
        v = v * v
    if not adamw:
        g = g + f32(lam) * p
    m = f32(b1) * m + f32(1 - b1) * g
    v = f32(b2) * v + (f32(1 - b2) * g) * g
    s = np.sqrt(v)
    if adamw:
        p = p * f32(1 - lr * lam)
    p = p - (f32(lr / (1 - b1 ** t)) * m) / (s * f32(1 / math.sqrt(1 - b2 ** t)) + f32(eps))
    if bits == 32:
        return p, m, v, None, None
    w = random_words(n, seed, t, place)
    m, ms = round_codes(m, w >> 16, False)
    v, vs = round_codes(s, w & 0xffff, True)
    return p, m, v, ms, vs


def make(sizes, dtype, bits, fresh=False, seed=0, offset=0):
    """Tensors of the given sizes; ``offset``: elements in front of each, to move it off its alignment."""
    g = torch.Generator().manual_seed(seed)
    out = {k: [] for k in ("p", "g", "m", "v", "ms", "vs")}
    put = lambda x: torch.cat([torch.zeros(offset, dtype=x.dtype), x]).cuda()[offset:]  # noqa: E731
    for n in sizes:
        out["p"].append(put(torch.randn(n, generator=g).to(dtype)))
        out["g"].append(put((torch.randn(n, generator=g) * 10 ** (2 * torch.randn(n, generator=g))).to(dtype)))
        m, v = torch.randn(n, generator=g), torch.rand(n, generator=g) * 2
        if bits == 32:
            out["m"].append(put(m * (not fresh)))
            out["v"].append(put(v * (not fresh)))
            continue
        code = lambda x: put(x.to(torch.float8_e4m3fn).view(torch.uint8)).view(torch.float8_e4m3fn)  # noqa: E731
        out["m"].append(code((m * 150 * (not fresh)).clamp(-448, 448)))
        out["v"].append(code(v * 200 * (not fresh)))
        nb = -(-n // BLOCK)
        out["ms"].append((torch.rand(nb, generator=g) * 1e-2 * (not fresh)).cuda())
        out["vs"].append((torch.rand(nb, generator=g) * 1e-2 * (not fresh)).cuda())
    return out


def call(s, bits, t, adamw, seed=5, **kw):
    from mole_b200 import ops
    scales = (s["ms"], s["vs"]) if bits == 8 else ()
    ops.adam_multi(s["p"], s["g"], s["m"], s["v"], *scales, t=t, adamw=adamw, seed=seed, **HP, **kw)


def host(s):
    to = lambda x: (x.float() if x.dtype != torch.float32 else x).cpu().numpy().copy()  # noqa: E731
    return {k: [to(x) for x in xs] for k, xs in s.items()}


def same_bits(got, want, what, kind=None):
    """``kind``: what one value in a thousand may be off by, a unit of "f32" or "bf16" or a "code"."""
    got = got.astype(np.float32)
    assert got.shape == want.shape
    bad = ~((got.view(np.uint32) == want.view(np.uint32)) | (np.isnan(got) & np.isnan(want)))
    if kind == "code":
        near = np.abs(got - want) <= np.maximum(np.abs(want) / 8, 2.0 ** -9)
    else:
        unit = {None: 0, "f32": 1, "bf16": 1 << 16}[kind]
        near = np.abs(got.view(np.int32).astype(np.int64) - want.view(np.int32)) <= unit
    if kind is not None and bad.sum() <= 1 + bad.size // 1000 and near[bad].all():
        return
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} differ, first at {np.argmax(bad)}: " \
                          f"{got[bad][0]!r} {want[bad][0]!r}"


def kind_of(name, bits, dtype=torch.float32):
    if name == "p":
        return "f32" if dtype == torch.float32 else "bf16"
    return "code" if bits == 8 and name in ("m", "v") else "f32"


SIZES = [1, 7, 8, 255, 256, 257, 0, 1000, 8192, 8193, 20001]


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("adamw", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_step_is_the_formula_operation_by_operation(bits, dtype, adamw, offset):
    s = make(SIZES, dtype, bits, seed=bits + offset, offset=offset)
    for t in (3, 4):
        h = host(s)
        call(s, bits, t, adamw)
        got = host(s)
        for i in range(len(SIZES)):
            extra = (h["ms"][i], h["vs"][i]) if bits == 8 else ()
            want = step_f32(h["p"][i], h["g"][i], h["m"][i], h["v"][i], t, i, adamw, 5, bits, *extra)
            p = torch.from_numpy(want[0]).to(dtype).float().numpy()
            for name, a, b in zip(("p", "m", "v", "ms", "vs"),
                                  [got[k][i] for k in ("p", "m", "v")] + ([got["ms"][i], got["vs"][i]] if bits == 8 else []),
                                  (p,) + want[1:]):
                same_bits(a, b, f"tensor {i} ({SIZES[i]}) {name} at t={t}", kind_of(name, bits, dtype))


@pytest.mark.parametrize("n_tensors", [17, 501, 1003])
def test_many_tensors_take_several_launches(n_tensors):
    sizes = [(7 * i) % 700 for i in range(n_tensors)]
    s = make(sizes, torch.float32, 8, seed=2)
    h = host(s)
    call(s, 8, 9, True)
    got = host(s)
    for i in list(range(0, n_tensors, 97)) + [n_tensors - 1]:
        want = step_f32(h["p"][i], h["g"][i], h["m"][i], h["v"][i], 9, i, True, 5, 8, h["ms"][i], h["vs"][i])
        for name, w in zip(("p", "m", "v", "ms", "vs"), want):
            same_bits(got[name][i], w, f"tensor {i} {name}", kind_of(name, 8))


def test_against_torch_adamw_in_64_bits():
    """Twenty steps against ``torch.optim.AdamW`` in fp64.  Each step rounds about ten operations at
    half a unit of 2^-24 relative to its terms; |p| <= ~5 and moves by at most ~lr a step, so after 20
    steps an element is off by less than 20 * 10 * 2^-24 * 5 = 6e-5 (in practice far less); a wrong
    bias correction or decay is off by lr * 1e-1 = 1e-3."""
    torch.manual_seed(0)
    ps = [torch.randn(n, device="cuda") for n in (1000, 37)]
    ref = [p.double().clone().requires_grad_() for p in ps]
    from mole_b200.optim import DeviceAdam
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    opt, want = DeviceAdam(params, **HP), torch.optim.AdamW(ref, **HP)
    for i in range(20):
        for p, r in zip(params, ref):
            p.grad = torch.randn_like(p)
            r.grad = p.grad.double()
        opt.step()
        want.step()
    for p, r in zip(params, ref):
        assert (p.double() - r).abs().max() < 6e-5


def test_fresh_zero_and_tiny_states():
    """Zero gradients leave zero states and move nothing; gradients of 1e-35 (blocks below 2^-100) are
    held as zeros; nothing becomes NaN."""
    s = make([600, 600], torch.float32, 8, fresh=True)
    s["g"][0].zero_()
    s["g"][1].fill_(1e-35)
    before = s["p"][0].clone()
    call(s, 8, 1, False)
    h = host(s)
    call(s, 8, 2, False)
    for k in ("p", "m", "v", "ms", "vs"):
        for x in host(s)[k]:
            assert np.isfinite(x).all()
    # weight decay in the gradient is what moves tensor 0
    assert not torch.equal(before, s["p"][0])
    t = make([300], torch.float32, 8, fresh=True)
    t["g"][0].zero_()
    p0 = t["p"][0].clone()
    from mole_b200 import ops
    ops.adam_multi(t["p"], t["g"], t["m"], t["v"], t["ms"], t["vs"], t=1, lr=1e-2)
    assert torch.equal(p0, t["p"][0]) and not t["m"][0].float().any() and not t["ms"][0].any()
    assert h["p"][0].shape == (600,)


def test_values_that_are_not_finite_stay_with_their_element():
    s = make([1024], torch.float32, 8, seed=3)
    clean = {k: [x.clone() for x in v] for k, v in s.items()}
    s["g"][0][5] = float("nan")
    s["g"][0][300] = float("inf")
    call(s, 8, 2, True)
    call(clean, 8, 2, True)
    a, b = host(s), host(clean)
    assert np.isnan(a["p"][0][5]) and np.isnan(a["m"][0][5])
    # block 1's infinite element is held as the largest code, blocks 2 and 3 do not notice
    assert np.abs(a["m"][0][300]) == 448 and a["v"][0][300] == 448
    assert np.isfinite(a["ms"][0]).all() and np.isfinite(a["vs"][0]).all()
    for k in ("p", "m", "v"):
        same_bits(a[k][0][512:], b[k][0][512:], k)
    others = np.ones(1024, bool)
    others[[5, 300]] = False
    assert np.isfinite(a["p"][0][others]).all() and np.isfinite(a["m"][0][others]).all()


def test_second_moment_moves_by_less_than_a_code():
    """beta2 = 0.999 moves v by 0.1 % a step, a hundredth of a code.  From v = 1 with g^2 = 4 the mean of
    sqrt(v) over 16384 elements has to follow 2000 steps of the exact recursion.  The rounding has mean
    zero in sqrt(v) and its spread, about a fifth of the value, averages to 0.2 %; its square adds half
    the variance, 2 to 4 %, to the recursion of v (sqrt is concave): 8 % covers both.  A rounding to
    nearest stays at 1, half of what is right."""
    n = 64 * BLOCK
    s = make([n], torch.float32, 8, fresh=True)
    s["g"][0].fill_(2.0)
    s["v"][0].copy_(torch.full((n,), 224.0))
    s["v"][0][::BLOCK] = 448.0                          # one element per block that holds the scale
    s["vs"][0].fill_(1 / 224)
    s["g"][0][::BLOCK] = 4.0
    for t in range(1, 2001):
        call(s, 8, t, True)
    rv = s["v"][0].float().view(-1, BLOCK)[:, 1:] * s["vs"][0][:, None]
    want = math.sqrt(4 + (1 - 4) * 0.999 ** 2000)
    assert abs(rv.mean().item() / want - 1) < 0.08


def test_same_seed_same_bits_other_seed_other_bits():
    a, b, c = (make([5000], torch.bfloat16, 8, seed=1) for _ in range(3))
    call(a, 8, 7, True, seed=1)
    call(b, 8, 7, True, seed=1)
    call(c, 8, 7, True, seed=2)
    for k in ("p", "m", "v", "ms", "vs"):
        assert torch.equal(a[k][0].float(), b[k][0].float())
    assert not torch.equal(a["m"][0].float(), c["m"][0].float())
    assert torch.equal(a["p"][0], c["p"][0])


def test_on_another_stream():
    s, ref = make([100000], torch.float32, 8, seed=1), make([100000], torch.float32, 8, seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s["g"][0].mul_(2)
        call(s, 8, 1, True)
    side.synchronize()
    ref["g"][0].mul_(2)
    call(ref, 8, 1, True)
    assert torch.equal(s["p"][0], ref["p"][0]) and torch.equal(s["m"][0].float(), ref["m"][0].float())


def test_capture_is_refused():
    s = make([1000], torch.float32, 32)
    from mole_b200 import _lib
    call(s, 32, 1, True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s["p"][0].add_(0)
        with pytest.raises(_lib.MoleError, match="MOLE_ERR_STATE"):
            call(s, 32, 2, True)
    g.replay()
    torch.cuda.synchronize()


def test_refusals():
    s = make([100, 50], torch.float32, 8)
    from mole_b200 import ops
    args = lambda **kw: {**{k: list(v) for k, v in s.items()}, **kw}  # noqa: E731

    def go(a, **kw):
        ops.adam_multi(a["p"], a["g"], a["m"], a["v"], a["ms"], a["vs"], **{"t": 1, "lr": 1e-3, **kw})
    before = s["p"][0].clone()
    with pytest.raises(ValueError, match="scales must be"):
        go(args(ms=[s["ms"][0], s["ms"][0][:0]]))
    with pytest.raises(ValueError, match="differ in size"):
        go(args(g=[s["g"][0], s["g"][0]]))
    with pytest.raises(TypeError, match="gradients must all be"):
        go(args(g=[s["g"][0], s["g"][1].bfloat16()]))
    with pytest.raises(TypeError, match="moments must all be"):
        go(args(v=[s["v"][0], s["v"][1].float()]))
    with pytest.raises(ValueError, match="one gradient"):
        go(args(g=s["g"][:1]))
    with pytest.raises(ValueError, match="twice"):
        go(args(p=[s["p"][0][:50], s["p"][0][:50]], g=[s["g"][1]] * 2, m=[s["m"][1]] * 2, v=[s["v"][1]] * 2,
                ms=[s["ms"][1]] * 2, vs=[s["vs"][1]] * 2))
    with pytest.raises(ValueError, match="8-bit moments need"):
        ops.adam_multi(s["p"], s["g"], s["m"], s["v"], t=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="contiguous"):
        go(args(p=[s["p"][0], torch.zeros(100, device="cuda")[::2]]))
    with pytest.raises(RuntimeError, match="step count"):
        go(args(), t=0)
    assert torch.equal(before, s["p"][0])


# ---- the optimizer ---------------------------------------------------------------------------------------
def _params(dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(*n, generator=g).to(dtype).cuda()) for n in ((40, 30), (7,), (3, 5, 11))]


def _grads(params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = torch.randn(*p.shape, generator=g).to(p.dtype).cuda()


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_checkpoint_continues_bit_for_bit(bits):
    from mole_b200.optim import DeviceAdam
    a, b = _params(), _params()
    oa, ob = DeviceAdam(a, state_bits=bits, seed=3, **HP), DeviceAdam(b, state_bits=bits, seed=3, **HP)
    for i in range(3):
        _grads(a, i)
        oa.step()
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    oc = copy.deepcopy(oa)                        # carries its width and seed along
    assert (oc.state_bits, oc.seed) == (bits, 3)
    for i in range(3, 6):
        _grads(a, i)
        _grads(b, i)
        oa.step()
        ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_optimizer_parameters_without_gradients_and_new_widths():
    from mole_b200.optim import DeviceAdam
    a = _params()
    opt = DeviceAdam(a, state_bits=8)
    _grads(a, 0)
    a[1].grad = None
    keep = a[1].detach().clone()
    opt.step()
    assert torch.equal(keep, a[1]) and not opt.state[a[1]]
    _grads(a, 1)
    opt.step()
    assert [opt.state[p]["step"] for p in a] == [2, 1, 2]
    # torch's own state comes in, at either width; a state goes over to 32 bits and back unchanged
    b = _params()
    tor = torch.optim.AdamW(b, lr=1e-3)
    _grads(b, 5)
    tor.step()
    wide, narrow = DeviceAdam(_params(), state_bits=32), DeviceAdam(_params(), state_bits=8)
    wide.load_state_dict(tor.state_dict())
    narrow.load_state_dict(tor.state_dict())
    for x, y, z in zip(b, wide.param_groups[0]["params"], narrow.param_groups[0]["params"]):
        assert torch.equal(tor.state[x]["exp_avg"], wide.state[y]["exp_avg"])
        from mole_b200.optim.device_adam import pack_moment, unpack_moment
        for name, sq in (("exp_avg", False), ("exp_avg_sq", True)):
            st = narrow.state[z]
            v = unpack_moment(st[name], st[name + "_scale"], sq)
            # nearest code: half a step, 2^-4 of the value (2^-3 in the square), or half of the smallest
            # code, 2^-10 of 448ths of the block's top
            top = tor.state[x][name].abs().max()
            off = (v - tor.state[x][name]).abs()
            assert (off <= (2 ** -3 if sq else 2 ** -4) * 1.1 * tor.state[x][name].abs() + 1e-5 * top).all()
            again = pack_moment(v, sq)
            assert torch.equal(again[0].float(), st[name].float())


def test_optimizer_steps_a_pickled_copy_and_refuses_what_it_lacks():
    from mole_b200.optim import DeviceAdam
    with pytest.raises(ValueError, match="8 or 32"):
        DeviceAdam(_params(), state_bits=16)
    with pytest.raises(ValueError, match="betas"):
        DeviceAdam(_params(), betas=(1.0, 0.9))
    p = _params()
    o = torch.optim.Adam(p, amsgrad=True)
    with pytest.raises(ValueError, match="amsgrad"):
        DeviceAdam(_params()).load_state_dict(o.state_dict())
    cpu = [torch.nn.Parameter(torch.zeros(4))]
    cpu[0].grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        DeviceAdam(cpu).step()


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_optimizer_takes_it_for_resident_experts(bits, tmp_path):
    """A layer stepped by ``MOLEMixedAdam(state_bits=...)`` through ``UniScheduler.build_optimizer``:
    with 32 bits as ``torch.optim.AdamW`` steps it (fp32: the order of the update's operations differs,
    a few units of 2^-24 of lr-sized steps), with 8 bits it trains and its checkpoint restores."""
    from mole_b200 import MOLEModule
    from mole_b200.utils.Uscheduler import UniScheduler
    from oracle import moe_ref as O
    T, M, E, F, k = 256, 128, 4, 128, 2
    inp = O.make_inputs(T, M, E, F, seed=4)

    def run(state_bits):
        MOLEModule._instance.clear()
        UniScheduler._instance = UniScheduler._optimizer = None
        UniScheduler(local_rank=0, disable_overlap=False, gate_control_by_MOLE=True)
        m = MOLEModule(0, E, M, F, -1, k, E, {"local_rank": 0, "world_size": 1, "rank": 0}, "gelu", 1,
                       False, False, dtype=torch.float32)
        m.set_layer_state({"gate": [inp["wg"], None],
                           "experts": [[inp["w1"][e], inp["b1"][e], inp["w2"][e], inp["b2"][e]]
                                       for e in range(E)]}, grad=False)
        opt = UniScheduler.build_optimizer(lr=1e-3, adamW=True, state_bits=state_bits)
        for i in range(2):
            x = inp["x"].cuda()
            y = m(x, capacity_factor=2.0)
            (y * inp["gy"].cuda()).sum().backward()
            opt.step()
            opt.zero_grad()
        return m, opt
    want = [p.detach().clone() for p in run(None)[0].s_experts_param()]
    m, opt = run(bits)
    got = [p.detach().clone() for p in m.s_experts_param()]
    if bits == 32:
        for a, b in zip(got, want):
            # second steps see gradients of parameters that differ in their last bits: 5e-4 of the 2 lr that
            # an element can move, as for the instant step
            assert (a - b).abs().max() <= 5e-4 * 2e-3 + 1e-6
    state = opt.get_optim_state()
    assert state[0][0]["exp_avg"].dtype == torch.float32 and state[0][0]["exp_avg"].device.type == "cpu"
    UniScheduler.save_states(str(tmp_path / "ckpt"))
    m2, opt2 = run(bits)
    UniScheduler.load_states(str(tmp_path / "ckpt"))
    for (a, b) in zip(opt.gpu_optimizer.state.values(), opt2.gpu_optimizer.state.values()):
        assert a["step"] == b["step"] and torch.equal(a["exp_avg"].float(), b["exp_avg"].float())
        assert torch.equal(a["exp_avg_sq"].float(), b["exp_avg_sq"].float())
    for a, b in zip(m2.s_experts_param(), got):
        assert torch.equal(a, b)
    UniScheduler._instance = UniScheduler._optimizer = None
