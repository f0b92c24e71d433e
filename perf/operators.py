"""Cases by which the operators on an expert's weights are measured: their ragged grouped products in
training, their products from 8-bit integers when serving, and the Adam step over many tensors with
states in 32 or 8 bits.  With ``own`` false every operator runs in its plain form, elementary torch
operations in 32 bits; with ``own`` true through this package's public calls."""
import math

import numpy as np
import torch

own = False

BLOCK = 256          # elements of a tensor that share one scale of an 8-bit state
E4M3_MAX = 448.0
MASK32 = 0xFFFFFFFF


def listed():
    return [
        # one token through top-2 of 64 experts (d_model 2048, d_ffn 8192): a decode step's first product
        {"name": "gmm decode 1 token", "op": "gmm", "rows": 2, "experts": 64, "k": 2048, "n": 8192, "kn": False,
         "spread": "even", "tail": 0, "grad": False, "dtype": "bf16"},
        # a serving batch of 48 tokens, top-2, through the second product ([F, M] weights, long reduction)
        {"name": "gmm batch 48 kn", "op": "gmm", "rows": 96, "experts": 64, "k": 8192, "n": 2048, "kn": True,
         "spread": "even", "tail": 0, "grad": False, "dtype": "bf16"},
        # the 64-expert layer's first product under Zipf routing, nothing dropped: forward and both gradients
        {"name": "gmm train zipf", "op": "gmm", "rows": 32768, "experts": 64, "k": 1024, "n": 4096, "kn": False,
         "spread": "zipf", "tail": 0, "grad": True, "dtype": "bf16"},
        # the GPT-MoE block's second product: forward and both gradients, 2 GB of weights
        {"name": "gmm train 8192x2048 kn", "op": "gmm", "rows": 16384, "experts": 64, "k": 8192, "n": 2048, "kn": True,
         "spread": "even", "tail": 0, "grad": True, "dtype": "bf16"},
        # the fp32 layer (d_model 512, 8 experts) with its gradients
        {"name": "gmm train fp32", "op": "gmm", "rows": 8192, "experts": 8, "k": 512, "n": 2048, "kn": False,
         "spread": "even", "tail": 0, "grad": True, "dtype": "fp32"},
        # odd sizes: experts without rows, rows behind the last expert, widths that are no multiple of a tile
        {"name": "gmm odd", "op": "gmm", "rows": 1237, "experts": 13, "k": 328, "n": 1001, "kn": False,
         "spread": "sparse", "tail": 37, "grad": True, "dtype": "bf16"},
        # one token through top-1 of the 128-expert layer held in 8 bits
        {"name": "int8 decode 1 token", "op": "int8", "rows": 1, "experts": 128, "k": 2048, "n": 8192,
         "spread": "even", "tail": 0, "dtype": "bf16"},
        # the same layer's batch of 32768 tokens, top-1
        {"name": "int8 experts 32768", "op": "int8", "rows": 32768, "experts": 128, "k": 2048, "n": 8192,
         "spread": "even", "tail": 0, "dtype": "bf16"},
        # one dense product (a shared expert or a projection) of a ragged token count, fp32 in and out
        {"name": "int8 dense 1000", "op": "int8", "rows": 1000, "experts": 0, "k": 2048, "n": 2000,
         "spread": "even", "tail": 0, "dtype": "fp32"},
        # the gate and the biases of a few small layers: latency
        {"name": "adam32 small fp32", "op": "adam", "tensors": 12, "elements": 60000, "bits": 32, "dtype": "fp32",
         "adamw": False, "step": 0},
        # many tensors of widely differing sizes, 32-bit states
        {"name": "adam32 400 tensors", "op": "adam", "tensors": 400, "elements": 60000000, "bits": 32, "dtype": "bf16",
         "adamw": True, "step": 100},
        # the two weights of 64 experts (d_model 1024, d_ffn 4096), 8-bit states
        {"name": "adam8 experts", "op": "adam", "tensors": 2, "elements": 536870912, "bits": 8, "dtype": "bf16",
         "adamw": True, "step": 1000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gmm", "gmm", "int8", "adam"])
    if op == "adam":
        tensors = _log(rng, 1, 400)
        return {"op": op, "tensors": tensors, "elements": max(tensors, _log(rng, 1000, 200000000)),
                "bits": rng.choice([8, 8, 32]), "dtype": rng.choice(["bf16", "bf16", "fp32"]),
                "adamw": rng.random() < 0.7, "step": _log(rng, 1, 100000) - 1}
    experts = rng.choice([0, 1, 128, _log(rng, 2, 128)]) if op == "int8" else _log(rng, 1, 128)
    step = rng.choice([1, 8, 16, 64])          # widths: any, or multiples of what wide loads and tiles want
    k = max(step, _log(rng, 64, 8192) // step * step)
    n = max(step, _log(rng, 64, 8192) // step * step)
    rows = _log(rng, 1, 32768)
    while experts * k * n > 2 ** (31 if op == "int8" else 30):      # as many weights as the largest listed layer
        experts = max(1, experts // 2)
    case = {"op": op, "experts": experts, "k": k, "n": n, "rows": rows,
            "spread": rng.choice(["even", "zipf", "sparse"]), "tail": rng.choice([0, 0, rng.randrange(1, 100)])}
    case["dtype"] = rng.choice(["bf16", "bf16", "fp32"])
    if op == "gmm":
        case["kn"] = rng.random() < 0.5
        case["grad"] = rng.random() < 0.6
    if op == "int8" and experts == 0:
        case["tail"] = 0
    # products in fp32, and widths that no wide load divides, stay small enough for a training step
    slow = case["dtype"] == "fp32" and op == "gmm" or step == 1
    while rows * k * n > (2 ** 34 if slow else 2 ** 38):
        rows = max(1, rows // 2)
        case["rows"] = rows
    return case


# ---- inputs ------------------------------------------------------------------------------------------
def _dtype(case):
    return {"bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]


def _bounds(case, seed):
    """Row ranges of the experts: [0, b1, ..., bE], the rows from bE on belong to nobody."""
    experts, rows = max(1, case["experts"]), case["rows"]
    r = np.random.RandomState(seed % (1 << 31))
    if case["spread"] == "zipf":
        share = r.permutation(1.0 / np.arange(1, experts + 1) ** 1.2)
    elif case["spread"] == "sparse":
        share = r.random_sample(experts) * (r.random_sample(experts) < 0.4)
        share[r.randint(experts)] += 0.5
    else:
        share = np.ones(experts)
    counts = r.multinomial(rows, share / share.sum())
    return [0] + np.cumsum(counts).tolist()


def _prepare_products(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, experts = _dtype(case), max(1, case["experts"])
    total = case["rows"] + case["tail"]
    k, n = case["k"], case["n"]
    bounds = _bounds(case, seed)
    rand = lambda *s, std=1.0: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32).mul_(std)  # noqa: E731
    st = {"case": case, "bounds": bounds, "x": rand(total, k).to(dt),
          "offsets": torch.tensor(bounds, dtype=torch.int32, device="cuda")}
    if case["op"] == "int8":
        # weights as a program holds them after it has quantised them once, a scale per expert and channel
        st["wq"] = torch.randint(-127, 128, (experts, n, k), generator=g, device="cuda", dtype=torch.int8)
        st["ws"] = torch.rand(experts, n, generator=g, device="cuda").mul_(0.0004).add_(0.0002)
        if case["experts"] == 0:
            st["wq"], st["ws"] = st["wq"][0], st["ws"][0]
        return st
    shape = (k, n) if case["kn"] else (n, k)
    st["w"] = torch.empty(experts, *shape, dtype=dt, device="cuda").normal_(0, 0.02, generator=g)
    if case["grad"]:
        st["dy"] = rand(total, n).to(dt)
    return st


def _sizes(case):
    """Sizes of the tensors of one optimizer: they add up to about the case's elements, spread over decades."""
    n, total = case["tensors"], case["elements"]
    if n == 2:
        return [total // 2, total - total // 2]
    share = np.exp(np.random.RandomState(n + total).uniform(0, 7, n))
    sizes = np.maximum(1, (share / share.sum() * total).astype(np.int64))
    return sizes.tolist()


def _prepare_adam(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(case)
    sizes = _sizes(case)
    starts, at, blocks = [], 0, []
    for s in sizes:                        # each tensor starts on a block of the flat buffers
        starts.append(at)
        blocks.append(at // BLOCK)
        at += -(-s // BLOCK) * BLOCK
    nb = at // BLOCK
    rand = lambda std: torch.randn(at, generator=g, device="cuda").mul_(std)  # noqa: E731
    flat = {"p": rand(0.02).to(dt)}
    # gradients of blocks differ in size, as those of layers and experts do
    size = torch.exp(torch.randn(nb, 1, generator=g, device="cuda"))
    grad = rand(1e-3)
    grad.view(nb, BLOCK).mul_(size)
    flat["g"] = grad.to(dt)
    del grad
    if case["bits"] == 32:
        flat["m"], flat["v"] = rand(3e-4), rand(1e-3).square_()
        if case["step"] == 0:
            flat["m"].zero_(), flat["v"].zero_()
    else:
        flat["m"] = rand(120.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        flat["v"] = rand(120.0).abs_().add_(2 ** -9).clamp_(max=E4M3_MAX).to(torch.float8_e4m3fn)
        flat["ms"] = size.flatten() * (1e-3 / E4M3_MAX)
        flat["vs"] = size.flatten() * (3e-3 / E4M3_MAX)
        if case["step"] == 0:
            for name in ("m", "v", "ms", "vs"):
                flat[name].zero_()
    st = {"case": case, "flat": flat, "t": case["step"], "seed": seed & MASK32,
          "sizes": sizes, "starts": starts}
    for name in ("p", "g", "m", "v"):
        st[name] = [flat[name][a:a + s] for a, s in zip(starts, sizes)]
    if case["bits"] == 8:
        for name in ("ms", "vs"):
            st[name] = [flat[name][b:b + -(-s // BLOCK)] for b, s in zip(blocks, sizes)]
    return st


def prepare(case, seed):
    return _prepare_adam(case, seed) if case["op"] == "adam" else _prepare_products(case, seed)


HYPER = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01}


# ---- plain forms ---------------------------------------------------------------------------------------
def _plain_gmm(st):
    case, bounds, x, w = st["case"], st["bounds"], st["x"], st["w"]
    y = torch.zeros(x.shape[0], case["n"], device="cuda")
    if case["grad"]:
        dx, dw = torch.zeros(x.shape, device="cuda"), torch.zeros_like(w)
    for e in range(len(bounds) - 1):
        rows = slice(bounds[e], bounds[e + 1])
        if bounds[e] == bounds[e + 1]:
            continue
        xe, we = x[rows].float(), w[e].float()
        y[rows] = xe @ (we if case["kn"] else we.t())
        if case["grad"]:
            de = st["dy"][rows].float()
            dx[rows] = de @ (we.t() if case["kn"] else we)
            dw[e] = xe.t() @ de if case["kn"] else de.t() @ xe
    if not case["grad"]:
        return {"y": y.to(x.dtype)}
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw}


def _plain_int8(st):
    # scale = amax / 127 of each token, rounded once; q = the integer nearest to x / scale (ties to even),
    # the quotient in 64 bits because a quotient next to a tie must not be rounded onto it
    case, bounds, x = st["case"], st["bounds"], st["x"].float()
    wq, ws = (st["wq"], st["ws"]) if case["experts"] else (st["wq"][None], st["ws"][None])
    scale = x.abs().amax(1)
    scale = scale / torch.full_like(scale, 127.0)          # (a division by a Python number multiplies by its inverse)
    q = torch.where(scale[:, None] > 0, torch.round(x.double() / scale[:, None].double()), 0.0).clamp_(-127, 127).float()
    y = torch.zeros(x.shape[0], case["n"], device="cuda")
    for e in range(len(bounds) - 1):
        rows = slice(bounds[e], bounds[e + 1])
        if bounds[e] != bounds[e + 1]:
            y[rows] = (q[rows] @ wq[e].float().t()) * scale[rows, None] * ws[e]
    return {"y": y.to(st["x"].dtype), "scale": scale}


# Random bits of the 8-bit states' rounding: element i takes step i % 8 of a linear congruential
# sequence that starts from a hash of i // 8, the tensor's place and the step's key.
LCG_A, LCG_C = 1664525, 1013904223
STEP_A = [pow(LCG_A, j + 1, 1 << 32) for j in range(8)]
STEP_C = [sum(pow(LCG_A, i, 1 << 32) for i in range(j + 1)) * LCG_C & MASK32 for j in range(8)]


def _mix(h):
    h = h * 0x9E3779B1 & MASK32
    h = (h ^ (h >> 15)) * 0x85157AF5 & MASK32
    return h ^ (h >> 13)


def _random_bits(n, seed, t, place):
    """32 bits for each of n elements."""
    key = _mix(_mix(_mix(seed) + t & MASK32) + place & MASK32)
    h = _mix(torch.arange(-(-n // 8), device="cuda") + key & MASK32)
    r = h[:, None] * torch.tensor(STEP_A, device="cuda") + torch.tensor(STEP_C, device="cuda") & MASK32
    return r.flatten()[:n]


def _blocks(x):
    """A flat tensor as [blocks, BLOCK], the last one filled with zeros."""
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _to_e4m3(x, random16):
    """(codes, scales) of a flat fp32 tensor: magnitudes above the code below are rounded up with the
    probability of their distance to it."""
    b = _blocks(x)
    top = b.abs().amax(1, keepdim=True)
    live = top >= 2.0 ** -100
    y = b * torch.where(live, torch.full_like(top, E4M3_MAX) / top, 0.0)
    a = y.abs()
    lift = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)          # below 2^-6 the codes are 2^-9 apart
    bits = (a + lift).view(torch.int32) + (_blocks(random16) << 4).int()
    r = (bits & -(1 << 20)).view(torch.float32) - lift
    r = r.clamp_(max=E4M3_MAX).copysign(y)
    return r.flatten()[:x.numel()], torch.where(live, top * (1.0 / E4M3_MAX), 0.0).flatten()


def _adam_scalars(case, t):
    h = HYPER
    return {"decay": float(np.float32(1.0 - h["lr"] * h["weight_decay"])), "lam": float(np.float32(h["weight_decay"])),
            "b1": float(np.float32(h["beta1"])), "c1": float(np.float32(1.0 - h["beta1"])),
            "b2": float(np.float32(h["beta2"])), "c2": float(np.float32(1.0 - h["beta2"])),
            "step": float(np.float32(h["lr"] / (1.0 - h["beta1"] ** t))),
            "r2": float(np.float32(1.0 / math.sqrt(1.0 - h["beta2"] ** t))), "eps": float(np.float32(h["eps"]))}


def _plain_adam(st):
    case, t = st["case"], st["t"]
    c = _adam_scalars(case, t)
    for i in range(len(st["sizes"])):
        n = st["sizes"][i]
        p, g, m, v = st["p"][i].float(), st["g"][i].float(), st["m"][i].float(), st["v"][i].float()
        if case["bits"] == 8:
            m = m * st["ms"][i].repeat_interleave(BLOCK)[:n]
            v = (v * st["vs"][i].repeat_interleave(BLOCK)[:n]).square()
        if not case["adamw"]:
            g = g + c["lam"] * p
        m = c["b1"] * m + c["c1"] * g
        v = c["b2"] * v + (c["c2"] * g) * g
        s = v.sqrt()
        if case["adamw"]:
            p = p * c["decay"]
        st["p"][i].copy_(p - (c["step"] * m) / (s * c["r2"] + c["eps"]))
        if case["bits"] == 32:
            st["m"][i].copy_(m)
            st["v"][i].copy_(v)
            continue
        r = _random_bits(n, st["seed"], t, i)
        mq, ms = _to_e4m3(m, r >> 16)
        vq, vs = _to_e4m3(s, r & 0xFFFF)
        # a second moment that is not zero is never held as zero: the step divides by it
        vq = torch.where((s > 0) & (vs.repeat_interleave(BLOCK)[:n] > 0), vq.clamp(min=2.0 ** -9), vq)
        for name, x in (("m", mq), ("v", vq), ("ms", ms), ("vs", vs)):
            st[name][i].copy_(x)


# ---- one pass ----------------------------------------------------------------------------------------
def _run_adam(st):
    st["t"] += 1
    if own:
        from mole_b200 import ops
        ops.adam_multi(st["p"], st["g"], st["m"], st["v"], st.get("ms"), st.get("vs"), t=st["t"], lr=HYPER["lr"],
                       betas=(HYPER["beta1"], HYPER["beta2"]), eps=HYPER["eps"], weight_decay=HYPER["weight_decay"],
                       adamw=st["case"]["adamw"], seed=st["seed"])
    else:
        _plain_adam(st)
    return {name: st["flat"][name] for name in ("p", "m", "v", "ms", "vs") if name in st["flat"]}


def _run_gmm(st):
    if not own:
        return _plain_gmm(st)
    import mole_b200
    case = st["case"]
    if not case["grad"]:
        return {"y": mole_b200.grouped_mm(st["x"], st["w"], st["offsets"], w_kn=case["kn"])}
    x, w = st["x"].detach().requires_grad_(), st["w"].detach().requires_grad_()
    y = mole_b200.grouped_mm(x, w, st["offsets"], w_kn=case["kn"])
    dx, dw = torch.autograd.grad(y, (x, w), st["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def _run_int8(st):
    if not own:
        return _plain_int8(st)
    from mole_b200 import ops
    q, scale = ops.quantize_rows(st["x"])
    if st["case"]["experts"]:
        y = ops.grouped_mm_int8(q, scale, st["wq"], st["ws"], st["offsets"], out_dtype=st["x"].dtype)
    else:
        y = ops.mm_int8(q, scale, st["wq"], st["ws"], out_dtype=st["x"].dtype)
    return {"y": y, "scale": scale}


def run(state):
    return {"adam": _run_adam, "gmm": _run_gmm, "int8": _run_int8}[state["case"]["op"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "adam":
        n = case["elements"]
        # p, m and v read and written, g read; the scales of the 8-bit states with them
        return {"bytes": n * 3 * size + n * (16 if case["bits"] == 32 else 4 + 16 / BLOCK), "flops": 14 * n}
    k, n, rows, experts = case["k"], case["n"], case["rows"], max(1, case["experts"])
    total = rows + case["tail"]
    # experts that have rows (about): only their weights have to be read
    live = min(experts, rows) * (0.45 if case["spread"] == "sparse" and experts > 2 else 1.0)
    if case["op"] == "int8":
        return {"bytes": total * (k * size + 4 + n * size) + live * n * (k + 4), "flops": 2 * rows * k * n}
    if not case["grad"]:
        return {"bytes": size * (total * (k + n) + live * k * n), "flops": 2 * rows * k * n}
    # forward, then both gradients: x, w and dy read, y, dx and dw written (dw of every expert)
    return {"bytes": size * (2 * total * (k + n) + (live + experts) * k * n), "flops": 6 * rows * k * n}


# ---- the definitions in 64 bits --------------------------------------------------------------------------
def _exact_products(case, seed):
    st = _prepare_products(case, seed)
    x, off = st["x"].double(), st["bounds"]
    out = {"y": torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device="cuda")}
    if case["op"] == "int8":
        # the token's scale is a 32-bit number by definition
        scale = (x.abs().max(1).values / 127.0).float().double()
        x = torch.round(x / torch.where(scale == 0, 1.0, scale)[:, None]).clamp(-127, 127)
        wq, ws = st["wq"].view(-1, case["n"], case["k"]), st["ws"].view(-1, case["n"]).double()
        for e, (a, b) in enumerate(zip(off[:-1], off[1:])):
            if b > a:
                out["y"][a:b] = torch.einsum("rk,nk->rn", x[a:b], wq[e].double()) * ws[e] * scale[a:b].unsqueeze(1)
        out["scale"] = scale
        return out
    if case["grad"]:
        out["dx"] = torch.zeros_like(x)
        out["dw"] = torch.zeros(st["w"].shape, dtype=torch.float64, device="cuda")
    for e, (a, b) in enumerate(zip(off[:-1], off[1:])):
        if b == a:
            continue
        w = st["w"][e].double()
        w = w.t() if case["kn"] else w                       # [N, K]
        out["y"][a:b] = torch.einsum("rk,nk->rn", x[a:b], w)
        if case["grad"]:
            d = st["dy"][a:b].double()
            out["dx"][a:b] = torch.einsum("rn,nk->rk", d, w)
            grad = torch.einsum("rn,rk->nk", d, x[a:b])
            out["dw"][e] = grad.t() if case["kn"] else grad
    return out


def _exact_rounded(x, u):
    """Magnitudes onto the grid of e4m3 by u in [0, 1): the floor of (position between codes + u)."""
    a = x.abs()
    power = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
    gap = torch.exp2(power - 3)
    return (torch.floor(a / gap + u) * gap).clamp(max=E4M3_MAX) * torch.sign(x)


def _exact_adam(case, seed):
    st = _prepare_adam(case, seed)
    t = st["t"] + 1
    f = st["flat"]
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    out = {k: f[k].double() for k in ("p", "m", "v", "ms", "vs") if k in f}
    for i, (a, n) in enumerate(zip(st["starts"], st["sizes"])):
        at = slice(a, a + n)
        p, g = f["p"][at].double(), f["g"][at].double()
        m, v = f["m"][at].double(), f["v"][at].double()
        if case["bits"] == 8:
            block = torch.arange(n, device="cuda") // BLOCK
            m, v = m * st["ms"][i].double()[block], (v * st["vs"][i].double()[block]) ** 2
        if not case["adamw"]:
            g = g + HYPER["weight_decay"] * p
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        if case["adamw"]:
            p = p - HYPER["lr"] * HYPER["weight_decay"] * p
        out["p"][at] = p - HYPER["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + HYPER["eps"])
        if case["bits"] == 32:
            out["m"][at], out["v"][at] = m, v
            continue
        bits = _random_bits(n, st["seed"], t, i)
        for name, x, u in (("m", m, bits >> 16), ("v", torch.sqrt(v), bits & 0xFFFF)):
            top = torch.zeros(st[name + "s"][i].numel(), dtype=torch.float64, device="cuda")
            top.scatter_reduce_(0, block, x.abs(), "amax")
            top = torch.where(top >= 2.0 ** -100, top, 0.0)
            y = torch.where(top[block] > 0, x * E4M3_MAX / top[block], 0.0)
            q = _exact_rounded(y, u / 65536.0)
            if name == "v":
                q = torch.where((x > 0) & (top[block] > 0), q.clamp(min=2.0 ** -9), q)
            out[name][at] = q
            out[name + "s"][a // BLOCK:a // BLOCK + top.numel()] = top / E4M3_MAX
    return out


def exact(case, seed):
    return _exact_adam(case, seed) if case["op"] == "adam" else _exact_products(case, seed)
