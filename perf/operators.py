"""Timed operators of a training step: the layer norm (``molix.F.layer_norm``, forward, backward and the second order
that force matching takes) and the AdamW step over many tensors (``molix.F.adamw_step`` with 32-bit states and
``molix.F.adamw8_step`` with 8-bit states, with the clipping of the gradients' norm).

``own`` false: the plain forms, elementary torch operations in float32, rounded once at the end; true: the package's
kernels.  ``exact`` restates the definitions in float64.

The 8-bit states, by their definition: blocks of 256 elements of a tensor share two bases (int16).  A code c stands for
the float32 whose bits are (base + c) << 20 (exponent and 3 bits), 0 for zero; a first moment's code has the sign in its
top bit and 7 bits of magnitude, a second moment's 8 bits of magnitude.  The base puts the block's largest magnitude,
rounded up, at the largest code.  Rounding adds a dither below bit 20 (16 random bits, centred) and cuts; a first moment
below the smallest code becomes that code with the probability that keeps its mean, a second moment is rounded up to it.
The dither of element i of tensor t at step s is a hash of (seed, t, s, i): the low half for the first moment, the high
half for the second.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 256
LOW32 = 0xFFFFFFFF


def listed():
    return [
        # the norm between the interactions of one small molecule's energy: latency
        {"name": "ln_infer_molecule", "kind": "norm", "direction": "forward", "rows": 96, "width": 128,
         "dtype": "float32"},
        # features of a mid-sized box in half precision (64 channels, l <= 2), an odd number of atoms
        {"name": "ln_infer_bf16", "kind": "norm", "direction": "forward", "rows": 20_001, "width": 576,
         "dtype": "bfloat16"},
        # a training batch of small molecules, 32 channels, l <= 1
        {"name": "ln_train_batch", "kind": "norm", "direction": "backward", "rows": 700, "width": 128,
         "dtype": "float32"},
        # the 50k-atom box, 128 channels, l <= 3, forward and every gradient
        {"name": "ln_train_50k", "kind": "norm", "direction": "backward", "rows": 50_000, "width": 2048,
         "dtype": "float32"},
        # a width that is no multiple of anything, half precision with gradients
        {"name": "ln_train_odd_f16", "kind": "norm", "direction": "backward", "rows": 12_345, "width": 333,
         "dtype": "float16"},
        # force matching on a box: the norm, its input gradient, and the gradients of a loss of both
        {"name": "ln_force_20k", "kind": "norm", "direction": "force", "rows": 20_000, "width": 512,
         "dtype": "float32"},
        # a small encoder's parameters: latency
        {"name": "adamw_small", "kind": "adamw", "bits": 32, "tensors": 24, "elements": 60_000, "clip": True,
         "dtype": "float32"},
        # the parameters of a 128-channel model
        {"name": "adamw_model", "kind": "adamw", "bits": 32, "tensors": 60, "elements": 3_200_001, "clip": True,
         "dtype": "float32"},
        # a model of 128 M parameters
        {"name": "adamw_128m", "kind": "adamw", "bits": 32, "tensors": 150, "elements": 128_000_003, "clip": True,
         "dtype": "float32"},
        # half-precision parameters, no clipping
        {"name": "adamw_bf16", "kind": "adamw", "bits": 32, "tensors": 90, "elements": 24_000_007, "clip": False,
         "dtype": "bfloat16"},
        # 8-bit states, a 128-channel model, read back as float32 (a checkpoint's export)
        {"name": "adamw8_model", "kind": "adamw", "bits": 8, "tensors": 60, "elements": 3_200_001, "clip": False,
         "dtype": "float32"},
        # 8-bit states, a large model
        {"name": "adamw8_64m", "kind": "adamw", "bits": 8, "tensors": 120, "elements": 64_000_001, "clip": False,
         "dtype": "float32"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if rng.random() < 0.5:
        direction = rng.choice(["forward", "backward", "force"])
        width = log(16, 6000)
        rows = log(1, min(60_000, 40_000_000 // width))
        # forces are matched in float32 alone: their accuracy does not survive 16 bits
        return {"kind": "norm", "direction": direction, "rows": rows, "width": width,
                "dtype": "float32" if direction == "force" else rng.choice(["float32", "float32", "bfloat16", "float16"])}
    bits = rng.choice([8, 32])
    tensors = log(1, 200)
    return {"kind": "adamw", "bits": bits, "tensors": tensors,
            "elements": tensors + log(2000, 100_000_000 if bits == 32 else 60_000_000),
            "clip": bits == 32 and rng.random() < 0.6, "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"])}


def _sizes(case):
    """Elements of each tensor: from biases to weight matrices, spread over a factor of 3000."""
    rng = random.Random("%d of %d" % (case["tensors"], case["elements"]))
    parts = [3000.0 ** rng.random() for _ in range(case["tensors"])]
    rest = case["elements"] - case["tensors"]
    got = [1 + int(rest * p / sum(parts)) for p in parts]
    got[rng.randrange(len(got))] += case["elements"] - sum(got)
    return got


def work(case):
    s = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "norm":
        n, d = case["rows"] * case["width"], case["width"]
        # forward: x read, y written; backward: x and the gradient read, y and grad_x written, and the weights'
        # gradients; force matching: x, the gradient and two seeds read, y, grad_x and three gradients written
        arrays, flops, vectors = {"forward": (2, 8, 2), "backward": (4, 22, 4), "force": (8, 60, 4)}[case["direction"]]
        return {"bytes": arrays * n * s + vectors * d * s, "flops": flops * n}
    n = case["elements"]
    if case["bits"] == 32:
        return {"bytes": n * (3 * s + 16), "flops": 16 * n}
    # the codes and bases in and out, the moments read back in float32
    return {"bytes": n * (3 * s + 4 + 8) + 8 * (n // BLOCK), "flops": 60 * n}


def _views(flat, sizes, starts):
    return [flat[a:a + n] for a, n in zip(starts, sizes)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["kind"] == "norm":
        R, D = case["rows"], case["width"]
        # features grow with the number of neighbours, so rows differ in scale, and have an offset
        x = normal(R, D) * torch.exp(0.5 * normal(R, 1)) + 0.5 * normal(R, 1)
        st = {"case": case, "x": x.to(dt), "w": (1 + 0.1 * normal(D)).to(dt), "b": (0.1 * normal(D)).to(dt)}
        if case["direction"] != "forward":
            st["g"] = (normal(R, D) * torch.exp(normal(R, 1))).to(dt)
        if case["direction"] == "force":
            st["seed_y"], st["seed_x"] = normal(R, D).to(dt), normal(R, D).to(dt)
        if case["direction"] != "forward":
            for k in ("x", "w", "b") + (("g",) if case["direction"] == "force" else ()):
                st[k].requires_grad_(True)
        return st

    # Parameters, gradients and states lie in one buffer each, every tensor at a multiple of 256 elements, so that
    # what a pass returns is whole and few.
    sizes = _sizes(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    inside = torch.zeros(total, dtype=torch.bool, device=DEV)
    scale = torch.ones(total, device=DEV)
    for a, n in zip(starts, sizes):
        inside[a:a + n] = True
        scale[a:a + n] = math.exp(random.Random(n).gauss(0, 1.5))  # tensors' gradients differ by orders of magnitude
    quiet = (torch.rand(total // BLOCK, generator=gen, device=DEV) < 0.05).repeat_interleave(BLOCK)  # no gradient yet
    p = torch.where(inside, 0.1 * normal(total), 0).to(dt)
    g = torch.where(inside & ~quiet, 0.01 * scale * normal(total) * torch.exp(normal(total)), 0).to(dt)
    m = torch.where(inside & ~quiet, 0.003 * scale * normal(total) * torch.exp(0.5 * normal(total)), 0)
    v = torch.where(inside & ~quiet, 2e-4 * scale * scale * torch.exp(normal(total)), 0)
    steps = torch.randint(1, 2000, (len(sizes),), generator=gen, device=DEV).float()
    st = {"case": case, "sizes": sizes, "flat_p": p, "flat_steps": steps,
          "params": _views(p, sizes, starts), "grads": _views(g, sizes, starts), "steps": list(steps.unbind()),
          "lengths": torch.tensor(sizes, device=DEV), "padded": torch.tensor([-(-n // BLOCK) * BLOCK for n in sizes], device=DEV),
          "hyper": {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}}
    if case["bits"] == 32:
        st.update(flat_m=m, flat_v=v, exp_avgs=_views(m, sizes, starts), exp_avg_sqs=_views(v, sizes, starts),
                  max_norm=1.0 if case["clip"] else None)
        return st
    # a state as an earlier step left it: codes and bases of these moments
    one = torch.full_like(m, 0.5)
    cm, cv, bases = _encode(m, v, one * 65536 - 0.5, one * 65536 - 0.5)
    back = torch.zeros(2, total, device=DEV)
    blocks = [slice(a // BLOCK, a // BLOCK + -(-n // BLOCK)) for a, n in zip(starts, sizes)]
    st.update(flat_cm=cm, flat_cv=cv, flat_bases=bases, back=back, seed=int(seed) % 1000,
              exp_avgs=_views(cm, sizes, starts), exp_avg_sqs=_views(cv, sizes, starts),
              bases=[bases[s] for s in blocks],
              out=(_views(back[0], sizes, starts), _views(back[1], sizes, starts)))
    return st


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _norm_parts(x, eps=1e-5):
    xc = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((xc * xc).mean(1, keepdim=True) + eps)
    return xc * r, r


def _project(a, xh, r):
    """The derivative of the normalised row applied to a (it is symmetric)."""
    return r * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))


def _plain_norm(st):
    dt, way = DTYPES[st["case"]["dtype"]], st["case"]["direction"]
    x, w, b = st["x"].detach().float(), st["w"].detach().float(), st["b"].detach().float()
    xh, r = _norm_parts(x)
    y = xh * w + b
    if way == "forward":
        return {"y": y.to(dt)}
    g = st["g"].detach().float()
    gx = _project(g * w, xh, r)
    if way == "backward":
        return {"y": y.to(dt), "gx": gx.to(dt), "gw": (g * xh).sum(0).to(dt), "gb": g.sum(0).to(dt)}
    # loss = <seed_y, y> + <seed_x, gx>
    s, u = st["seed_y"].float(), st["seed_x"].float()
    a, ju = g * w, _project(u, xh, r)
    alpha, ups = (a * xh).mean(1, keepdim=True), (u * xh).mean(1, keepdim=True)
    dx = _project(s * w, xh, r) - r * (alpha * ju + ups * gx) - r * xh * (ju * a).mean(1, keepdim=True)
    return {"y": y.to(dt), "gx": gx.to(dt), "dx": dx.to(dt), "dw": (s * xh + g * ju).sum(0).to(dt),
            "db": s.sum(0).to(dt), "dg": (w * ju).to(dt)}


def _mix(x):
    """A hash of 32-bit integers (held in int64): multiplications and shifted exclusive ors."""
    x = x & LOW32
    x = ((x ^ (x >> 15)) * 0x6A09E667) & LOW32
    x = ((x ^ (x >> 13)) * 0xBB67AE85) & LOW32
    return x ^ (x >> 16)


def _dither(seed, steps, lengths):
    """(low, high): 16 bits each for every element, tensors padded to blocks."""
    t = torch.arange(len(steps), device=DEV)
    key = _mix(_mix(seed * 0x3C6EF373 + t * 0xA54FF53B) + steps.long() * 0x510E527F)
    starts = torch.cumsum(lengths, 0) - lengths
    first = torch.repeat_interleave(key - starts * 0x9E3779B1, lengths)
    h = _mix(first + torch.arange(first.numel(), device=DEV) * 0x9E3779B1)
    return h & 0xFFFF, h >> 16


def _encode(m, v, dm, dv):
    """Codes of the moments and the blocks' bases; dm, dv: the dithers, 0 to 65535."""
    bm, bv = m.view(torch.int32).long(), v.view(torch.int32).long()
    sign, bm = (bm < 0).long() * 128, bm & 0x7FFFFFFF
    top = lambda b, most: ((b.view(-1, BLOCK).amax(1) >> 20) + 1 - most).clamp(min=0)  # noqa: E731
    em, ev = top(bm, 127), top(bv, 255)
    um, uv = dm.long(), dv.long()
    em_, ev_ = em.repeat_interleave(BLOCK), ev.repeat_interleave(BLOCK)
    qm = ((bm + (um << 4) + 8) >> 20) - em_
    least = ((em_ + 1) << 20).int().view(torch.float32)
    small = (m.abs() * 65536 > (um.float() + 0.5) * least).long()
    # a magnitude under the smallest code's is a matter of chance, also where the dither would lift it
    qm = torch.where((bm >> 20) <= em_, small, qm)
    qv = torch.where(bv == 0, 0, (((bv + (uv << 4) + 8) >> 20) - ev_).clamp(1, 255))
    return (torch.where(qm > 0, qm + sign, 0)).to(torch.uint8), qv.to(torch.uint8), torch.stack([em, ev], 1).to(torch.int16)


def _decode(cm, cv, bases):
    e = bases.long().repeat_interleave(BLOCK, 0)
    c, d = cm.long() & 127, cv.long()
    m = torch.where(c > 0, (e[:, 0] + c) << 20, 0).int().view(torch.float32)
    v = torch.where(d > 0, (e[:, 1] + d) << 20, 0).int().view(torch.float32)
    return torch.where(cm >= 128, -m, m), v


def _step_scalars(st, steps):
    h = st["hyper"]
    b1, b2 = h["betas"]
    t = steps.double()  # 1 - b^t of a few numbers, as a program has them on the host
    return (h["lr"] / (1 - b1 ** t)).float(), (1 - b2 ** t).sqrt().float()


def _plain_adamw(st):
    h = st["hyper"]
    b1, b2 = h["betas"]
    p = torch.cat(st["params"]).float()
    g = torch.cat(st["grads"]).float()
    m, v = torch.cat(st["exp_avgs"]), torch.cat(st["exp_avg_sqs"])
    out = {}
    if st["max_norm"] is not None:
        out["norm"] = g.square().sum().sqrt()
        g = g * (st["max_norm"] / (out["norm"] + 1e-6)).clamp(max=1.0)
    st["flat_steps"] += 1
    size, root = _step_scalars(st, st["flat_steps"])
    size, root = (torch.repeat_interleave(s, st["lengths"], output_size=p.numel()) for s in (size, root))
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = p * (1 - h["lr"] * h["weight_decay"]) - size * m / (v.sqrt() / root + h["eps"])
    torch._foreach_copy_(st["params"], list(p.split(st["sizes"])))
    torch._foreach_copy_(st["exp_avgs"], list(m.split(st["sizes"])))
    torch._foreach_copy_(st["exp_avg_sqs"], list(v.split(st["sizes"])))
    return out | {"p": st["flat_p"], "m": st["flat_m"], "v": st["flat_v"], "steps": st["flat_steps"]}


def _plain_adamw8(st):
    h = st["hyper"]
    b1, b2 = h["betas"]
    pad = lambda ts: torch.cat([torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)) for t in ts])  # noqa: E731
    whole = lambda flat: [t[:n] for t, n in zip(flat.split(st["padded_list"]), st["sizes"])]  # noqa: E731
    st.setdefault("padded_list", [-(-n // BLOCK) * BLOCK for n in st["sizes"]])
    p, g = pad(st["params"]).float(), pad(st["grads"]).float()
    m, v = _decode(pad(st["exp_avgs"]), pad(st["exp_avg_sqs"]), torch.cat(st["bases"]))
    st["flat_steps"] += 1
    size, root = _step_scalars(st, st["flat_steps"])
    size, root = (torch.repeat_interleave(s, st["padded"], output_size=p.numel()) for s in (size, root))
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = p * (1 - h["lr"] * h["weight_decay"]) - size * m / (v.sqrt() / root + h["eps"])
    cm, cv, bases = _encode(m, v, *_dither(st["seed"], st["flat_steps"], st["padded"]))
    torch._foreach_copy_(st["params"], whole(p))
    torch._foreach_copy_(st["exp_avgs"], whole(cm))
    torch._foreach_copy_(st["exp_avg_sqs"], whole(cv))
    torch._foreach_copy_(st["bases"], list(bases.split([n // BLOCK for n in st["padded_list"]])))
    m, v = _decode(cm, cv, bases)
    torch._foreach_copy_(st["out"][0], whole(m))
    torch._foreach_copy_(st["out"][1], whole(v))
    return {"p": st["flat_p"], "moments": st["back"], "steps": st["flat_steps"]}


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------


def _own_norm(st):
    from molnex_amd.molix import F

    way, x, w, b = st["case"]["direction"], st["x"], st["w"], st["b"]
    y = F.layer_norm(x, (x.shape[1],), w, b)
    if way == "forward":
        return {"y": y}
    if way == "backward":
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), st["g"])
        return {"y": y.detach(), "gx": gx, "gw": gw, "gb": gb}
    (gx,) = torch.autograd.grad(y, x, st["g"], create_graph=True)
    dx, dw, db, dg = torch.autograd.grad((y, gx), (x, w, b, st["g"]), (st["seed_y"], st["seed_x"]))
    return {"y": y.detach(), "gx": gx.detach(), "dx": dx, "dw": dw, "db": db, "dg": dg}


def _own_adamw(st):
    from molnex_amd.molix import F

    norm = F.adamw_step(st["params"], st["grads"], st["exp_avgs"], st["exp_avg_sqs"], st["steps"],
                        max_norm=st["max_norm"], **st["hyper"])
    out = {"p": st["flat_p"], "m": st["flat_m"], "v": st["flat_v"], "steps": st["flat_steps"]}
    return out if norm is None else out | {"norm": norm}


def _own_adamw8(st):
    from molnex_amd.molix import F

    F.adamw8_step(st["params"], st["grads"], st["exp_avgs"], st["exp_avg_sqs"], st["bases"], st["steps"],
                  seed=st["seed"], **st["hyper"])
    F.adamw8_moments(st["exp_avgs"], st["exp_avg_sqs"], st["bases"], out=st["out"])
    return {"p": st["flat_p"], "moments": st["back"], "steps": st["flat_steps"]}


def run(state):
    case = state["case"]
    if case["kind"] == "norm":
        return (_own_norm if own else _plain_norm)(state)
    if case["bits"] == 32:
        return (_own_adamw if own else _plain_adamw)(state)
    return (_own_adamw8 if own else _plain_adamw8)(state)


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------


def _exact_norm(st):
    """Autograd of the written-out definition in float64."""
    way = st["case"]["direction"]
    x, w, b = (st[k].detach().double().requires_grad_(True) for k in ("x", "w", "b"))
    mu = x.mean(1, keepdim=True)
    y = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + 1e-5) * w + b
    if way == "forward":
        return {"y": y.detach()}
    g = st["g"].detach().double().requires_grad_(True)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g, create_graph=way == "force")
    if way == "backward":
        return {"y": y.detach(), "gx": gx, "gw": gw, "gb": gb}
    dx, dw, db, dg = torch.autograd.grad((y, gx), (x, w, b, g), (st["seed_y"].double(), st["seed_x"].double()))
    return {"y": y.detach(), "gx": gx.detach(), "dx": dx, "dw": dw, "db": db, "dg": dg}


def _exact_hash(x):
    x = x.astype(np.uint64) & np.uint64(LOW32)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x6A09E667)) & np.uint64(LOW32)
    x = ((x ^ (x >> np.uint64(13))) * np.uint64(0xBB67AE85)) & np.uint64(LOW32)
    return x ^ (x >> np.uint64(16))


def _value(k):
    """What base + code = k stands for, with no use of float32's bits: eight values to the power of two from 2^-126
    on, and their spacing below it."""
    octave = np.maximum(k >> 3, 1)
    return np.ldexp((k - 8 * (octave - 1)) / 8.0, octave - 127)


def _key(z):
    """The largest k with _value(k) <= z."""
    part, e = np.frexp(z)
    e = np.where(z > 0, e, -126)
    return np.where(e < -125, np.floor(np.ldexp(z, 129)), np.floor((2 * part - 1) * 8) + 8 * (e + 126)).astype(np.int64)


def _exact_codes(x, draw16, most, up):
    """The values that the 8-bit codes of one tensor's float64 moments stand for."""
    pad = lambda v: np.pad(v, (0, -len(v) % BLOCK)).reshape(-1, BLOCK)  # noqa: E731
    z, chance = pad(np.abs(x)), (pad(draw16).astype(np.float64) + 0.5) / 65536
    k = _key(z)
    base = np.maximum(k.max(1, keepdims=True) + 1 - most, 0)
    low = np.where(k > base, _value(k), 0.0)  # under the smallest code there is zero
    high = _value(np.maximum(k, base) + 1)
    share = (z - low) / (high - low)
    if up:
        lifted = np.where(k > base, share >= 1 - chance, z > 0)
    else:
        lifted = np.where(k > base, share >= 1 - chance, share > chance)
    return np.sign(x) * np.where(lifted, high, low).reshape(-1)[:len(x)]


def _exact_moments(codes, bases, n, signed):
    c = codes.cpu().numpy().astype(np.int64)
    base = np.repeat(bases.cpu().numpy().astype(np.int64), BLOCK)[:n]
    size = c & 127 if signed else c
    got = np.where(size > 0, _value(base + size), 0.0)
    return torch.from_numpy(np.where(c > 127, -got, got) if signed else got).to(DEV)


def _exact_adamw(st):
    h, case = st["hyper"], st["case"]
    b1, b2 = h["betas"]
    eight = case["bits"] == 8
    flat = {"p": st["flat_p"].double(), "m": torch.zeros_like(st["flat_p"], dtype=torch.float64)}
    flat["v"] = flat["m"].clone()
    out, factor = {}, 1.0
    if not eight and st["max_norm"] is not None:
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in st["grads"]))
        out["norm"] = torch.tensor(norm, dtype=torch.float64)
        factor = min(1.0, st["max_norm"] / (norm + 1e-6))
    at = 0
    for i, (n, g) in enumerate(zip(st["sizes"], st["grads"])):
        t = float(st["flat_steps"][i]) + 1
        s = slice(at, at + n)
        g = g.double() * factor
        if eight:
            m = _exact_moments(st["exp_avgs"][i], st["bases"][i][:, 0], n, True)
            v = _exact_moments(st["exp_avg_sqs"][i], st["bases"][i][:, 1], n, False)
        else:
            m, v = st["exp_avgs"][i].double(), st["exp_avg_sqs"][i].double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        root = torch.sqrt(v / (1 - b2 ** t)) + h["eps"]
        flat["p"][s] = flat["p"][s] * (1 - h["lr"] * h["weight_decay"]) - h["lr"] * (m / (1 - b1 ** t)) / root
        if eight:
            key = _exact_hash(np.array([st["seed"] * 0x3C6EF373 + i * 0xA54FF53B]))
            key = _exact_hash(key + np.uint64(int(t) * 0x510E527F))
            r = _exact_hash(key + (np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B1) & np.uint64(LOW32)))
            m = torch.from_numpy(_exact_codes(m.cpu().numpy(), r & np.uint64(0xFFFF), 127, False)).to(DEV)
            v = torch.from_numpy(_exact_codes(v.cpu().numpy(), r >> np.uint64(16), 255, True)).to(DEV)
        flat["m"][s], flat["v"][s] = m, v
        at += -(-n // BLOCK) * BLOCK
    out["steps"] = st["flat_steps"] + 1
    if eight:
        return out | {"p": flat["p"], "moments": torch.stack([flat["m"], flat["v"]])}
    return out | flat


def exact(case, seed):
    if case["kind"] == "adamw" and case["bits"] == 8 and case["elements"] > 20_000_000:
        return None  # its codes are formed on the host: too slow there
    st = prepare(case, seed)
    return (_exact_norm if case["kind"] == "norm" else _exact_adamw)(st)
