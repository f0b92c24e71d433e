"""``ops.adam_multi`` where every thread block walks many chunks: the stages of its ring are used again and
again, up to the bound of a block's walk, over tensors that begin and end inside it, with blocks among
them that the whole blocks' form leaves to the general one.

The formula is restated on the device in float32 by separate torch operations, each of which rounds by
itself (products, sums, quotients and roots correctly).  As in ``test_gpu_adam_multi.py`` one value in a
thousand may be one unit off (root and quotient of the whole blocks' form) and, where that moves a value
across its random threshold, one code."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK, M32 = 256, 0xFFFFFFFF
HP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def f32(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def mix(h):
    h = h * 0x9E3779B1 & M32
    h = (h ^ (h >> 15)) * 0x85157AF5 & M32
    return h ^ (h >> 13)


def random_words(n, seed, t, place):
    """Element i: step i % 8 + 1 of the congruential sequence that starts at the hash of i // 8."""
    key = mix(mix(mix(seed) + t & M32) + place & M32)
    r = mix(torch.arange(-(-n // 8), device="cuda") + key & M32)
    out = torch.empty(len(r), 8, dtype=torch.int64, device="cuda")
    for i in range(8):
        r = r * 1664525 + 1013904223 & M32
        out[:, i] = r
    return out.flatten()[:n]


def blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def round_codes(x, u, floor):
    b = blocks(x)
    top = torch.where(b.isfinite(), b.abs(), 0).amax(1, keepdim=True)
    live = top >= 2.0 ** -100
    y = b * torch.where(live, f32(448.0) / top, f32(0.0))
    a = y.abs()
    lift = torch.where(a < 2.0 ** -6, f32(2.0 ** -6), f32(0.0))
    bits = (a + lift).view(torch.int32).long() + (blocks(u) << 4)
    r = (bits & 0xFFF00000).int().view(torch.float32) - lift
    r = torch.where(y.isnan(), y, r.clamp(max=448.0))
    if floor:
        r = torch.where((b > 0) & live & (r < 2.0 ** -9), f32(2.0 ** -9), r)
    r = torch.where(live, r.copysign(y), 0.0)
    return r.flatten()[:x.numel()], torch.where(live, top * f32(1 / 448), f32(0.0)).flatten()


def step_f32(p, g, m, v, t, place, adamw, seed, bits, ms, vs):
    n, (b1, b2) = len(p), HP["betas"]
    p, g, m, v = p.float(), g.float(), m.float(), v.float()
    if bits == 8:
        m = m * ms.repeat_interleave(BLOCK)[:n]
        v = v * vs.repeat_interleave(BLOCK)[:n]
        v = v * v
    if not adamw:
        g = g + f32(HP["weight_decay"]) * p
    m = f32(b1) * m + f32(1 - b1) * g
    v = f32(b2) * v + (f32(1 - b2) * g) * g
    s = v.sqrt()
    if adamw:
        p = p * f32(1 - HP["lr"] * HP["weight_decay"])
    q = (f32(HP["lr"] / (1 - b1 ** t)) * m) / (s * f32(1 / math.sqrt(1 - b2 ** t)) + f32(HP["eps"]))
    p = p - q
    if bits == 32:
        return p, q, m, v, None, None
    w = random_words(n, seed, t, place)
    return (p, q, *(lambda a, b: (a[0], b[0], a[1], b[1]))(round_codes(m, w >> 16, False), round_codes(s, w & 0xffff, True)))


def make(sizes, dtype, bits, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    out = {k: [] for k in ("p", "g", "m", "v", "ms", "vs")}
    for n in sizes:
        out["p"].append(rand(n).to(dtype))
        grad, m, v = rand(n) * torch.exp(2 * rand(n)), rand(n), rand(n).abs() + 1e-3
        if n > 4000:        # blocks for the general form: no gradient yet, and a value that is not finite
            for at in range(1000, n - 1000, 70000):
                grad[at:at + 700] = 0
                m[at:at + 700] = 0
                v[at:at + 700] = 0
            grad[n // 2] = float("nan")
            grad[n // 3] = float("inf")
        out["g"].append(grad.to(dtype))
        if bits == 32:
            out["m"].append(m)
            out["v"].append(v)
            continue
        nb = -(-n // BLOCK)
        out["m"].append((m * 120).clamp(-448, 448).to(torch.float8_e4m3fn))
        out["v"].append((v * 120).clamp(max=448).to(torch.float8_e4m3fn))
        out["ms"].append(rand(nb).abs() * 1e-2 + 1e-4)
        out["vs"].append(rand(nb).abs() * 1e-2 + 1e-4)
    return out


def same(got, want, what, kind, step=None):
    """``step``: what was subtracted; a unit of it is more than one of a difference that nearly cancels."""
    got, want = got.float(), want.float()
    bad = ~((got.view(torch.int32) == want.view(torch.int32)) | (got.isnan() & want.isnan()))
    if kind == "code":
        near = (got - want).abs() <= torch.maximum(want.abs() / 8, f32(2.0 ** -9))
    else:
        near = (got.view(torch.int32).long() - want.view(torch.int32)).abs() <= {"f32": 1, "bf16": 1 << 16}[kind]
    if step is not None:
        near |= (got - want).abs() <= 2.0 ** -23 * step.abs()
    assert int(bad.sum()) <= 1 + bad.numel() // 1000 and bool(near[bad].all()), \
        f"{what}: {int(bad.sum())} of {bad.numel()} differ, {int((bad & ~near).sum())} by more than a unit, " \
        f"first at {int(bad.int().argmax())}"


# 32 million fp32 elements are 15,700 chunks of 2048: more than 32 for each of 444 resident blocks
SIZES = {"one tensor": [6_000_001], "mixed": [300, 2_500_000, 1, 0, 4096, 3_333_333, 70, 255, 1_000_000, 8192],
         "longest walk": [32_000_000]}


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_chunks_per_block(bits, dtype, sizes):
    from mole_b200 import ops
    s = make(SIZES[sizes], dtype, bits, seed=bits)
    adamw = sizes != "mixed"
    for t in (3, 4):
        before = {k: [x.clone() for x in xs] for k, xs in s.items()}
        ops.adam_multi(s["p"], s["g"], s["m"], s["v"], *((s["ms"], s["vs"]) if bits == 8 else ()), t=t, adamw=adamw,
                       seed=9, **HP)
        for i, n in enumerate(SIZES[sizes]):
            if n == 0:
                continue
            b = {k: xs[i] if xs else None for k, xs in before.items()}
            p, q, m, v, ms, vs = step_f32(b["p"], b["g"], b["m"], b["v"], t, i, adamw, 9, bits, b["ms"], b["vs"])
            what = f"tensor {i} ({n}) at t={t}"
            same(s["p"][i], p.to(dtype), what + " p", "f32" if dtype == torch.float32 else "bf16", q)
            code = "code" if bits == 8 else "f32"
            same(s["m"][i], m, what + " m", code)
            same(s["v"][i], v, what + " v", code)
            if bits == 8:
                same(s["ms"][i], ms, what + " ms", "f32")
                same(s["vs"][i], vs, what + " vs", "f32")
            assert torch.equal(s["g"][i].nan_to_num(), b["g"].nan_to_num())
    assert ops.device_fault() == 0
