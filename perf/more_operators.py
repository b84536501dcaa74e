"""Timed operators of models with weights per element: the linear map whose weights each row's class selects
(``molix.F.indexed_linear``, forward and both gradients), and the training of its stacks of matrices and of a model's
other matrices by orthogonalised updates (``molix.F.orthogonalize``, ``molix.F.muon_step``).

``own`` false: the plain forms, elementary torch operations in float32, rounded once at the end; true: the package's
kernels.  ``exact`` restates the definitions in float64.

Indexed linear: y[i] = x[i] W[z[i]], rows of a class outside [0, classes) give zeros.

Orthogonalisation of an m x n matrix G: X = G / max(|G|, 1e-7) with the Frobenius norm, transposed if m > n, then five
times X <- a X + (b A + c A A) X with A = X X^T and (a, b, c) = (3.4445, -4.775, 2.0315).

Muon step: M <- 0.95 M + 0.05 G, U = 0.05 G + 0.95 M, O the orthogonalised U,
P <- (1 - lr decay) P - lr sqrt(max(1, m / n)) O.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LR, DECAY, MU = 0.02, 0.1, 0.95
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


def listed():
    return [
        # one small molecule's atoms through per-element weights, without a plan: latency
        {"name": "indexed_infer_molecule", "kind": "indexed", "direction": "forward", "rows": 96, "classes": 5,
         "width": 64, "out": 64, "plan": False, "skew": 1.0, "dtype": "float32"},
        # features of a mid-sized box in half precision, an odd number of atoms, the elements' plan at hand
        {"name": "indexed_infer_bf16", "kind": "indexed", "direction": "forward", "rows": 20_001, "classes": 10,
         "width": 512, "out": 512, "plan": True, "skew": 1.0, "dtype": "bfloat16"},
        # 50k atoms, 128 channels, ten elements, both gradients
        {"name": "indexed_train_50k", "kind": "indexed", "direction": "backward", "rows": 50_000, "classes": 10,
         "width": 128, "out": 128, "plan": True, "skew": 1.0, "dtype": "float32"},
        # widths that are multiples of nothing, as many classes as a periodic table has, batches without a plan
        {"name": "indexed_train_odd_f16", "kind": "indexed", "direction": "backward", "rows": 12_345, "classes": 89,
         "width": 333, "out": 77, "plan": False, "skew": 2.0, "dtype": "float16"},
        # most rows of one element, padding rows behind the atoms
        {"name": "indexed_train_skew", "kind": "indexed", "direction": "backward", "rows": 200_003, "classes": 4,
         "width": 256, "out": 64, "plan": True, "skew": 3.0, "dtype": "float32"},
        # wide experts of a large training batch
        {"name": "indexed_train_wide_bf16", "kind": "indexed", "direction": "backward", "rows": 100_001,
         "classes": 64, "width": 1024, "out": 2048, "plan": True, "skew": 0.5, "dtype": "bfloat16"},
        # one small matrix: latency
        {"name": "ortho_small", "kind": "ortho", "batch": 1, "rows": 64, "width": 64, "dtype": "float32"},
        # a matrix of odd sizes in half precision
        {"name": "ortho_odd_f16", "kind": "ortho", "batch": 1, "rows": 333, "width": 1234, "dtype": "float16"},
        # a large tall matrix
        {"name": "ortho_large_bf16", "kind": "ortho", "batch": 1, "rows": 8192, "width": 4096, "dtype": "bfloat16"},
        # a small encoder's matrices
        {"name": "muon_encoder", "kind": "muon", "tensors": 24, "low": 16, "high": 128, "batch": 1,
         "dtype": "float32"},
        # the matrices of a larger model
        {"name": "muon_model", "kind": "muon", "tensors": 60, "low": 128, "high": 1024, "batch": 1,
         "dtype": "float32"},
        # stacks of experts' matrices in half precision
        {"name": "muon_experts_bf16", "kind": "muon", "tensors": 2, "low": 512, "high": 1024, "batch": 32,
         "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["indexed", "indexed", "ortho", "muon"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    if kind == "indexed":
        width, out = _log(rng, 16, 2048), _log(rng, 16, 2048)
        rows = _log(rng, 1, max(2, min(200_000, 100_000_000 // (width + out))))
        return {"kind": kind, "direction": rng.choice(["forward", "backward"]), "rows": rows,
                "classes": _log(rng, 1, 100), "width": width, "out": out, "plan": rng.random() < 0.5,
                "skew": round(rng.uniform(0, 3), 2), "dtype": dtype}
    if kind == "ortho":
        rows, width = _log(rng, 2, 4000), _log(rng, 2, 4000)
        batch = _log(rng, 1, max(1, min(64, 2_000_000_000 // (min(rows, width) * rows * width))))
        return {"kind": kind, "batch": batch, "rows": rows, "width": width, "dtype": dtype}
    low = _log(rng, 8, 300)
    high = _log(rng, low, 1500)
    return {"kind": kind, "tensors": _log(rng, 1, 60), "low": low, "high": high,
            "batch": rng.choice([1, 1, 1, 2]), "dtype": dtype}


def _shapes(case):
    """The matrices of a model: widths that repeat, as layers do, some tall and some wide."""
    rng = random.Random("%(tensors)d of %(low)d to %(high)d" % case)
    widths = [case["low"], case["high"]] + [_log(rng, case["low"], case["high"]) for _ in range(2)]
    shapes = [(rng.choice(widths), rng.choice(widths)) for _ in range(case["tensors"])]
    shapes[0] = (case["low"], case["high"])  # both ends of the range, in both orders
    shapes[-1] = (case["high"], case["low"] if len(shapes) > 1 else case["high"])
    return [(case["batch"], *s) for s in shapes]


def work(case):
    s = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "indexed":
        R, K, N = case["rows"], case["width"], case["out"]
        weights = min(case["classes"], R) * K * N
        if case["direction"] == "forward":
            return {"bytes": s * (R * (K + N) + weights), "flops": 2 * R * K * N}
        # x, the gradient and the weights read; y and both gradients written
        return {"bytes": s * (2 * R * (K + N) + weights + case["classes"] * K * N), "flops": 6 * R * K * N}
    shapes = [(case["batch"], case["rows"], case["width"])] if case["kind"] == "ortho" else _shapes(case)
    n = sum(b * r * c for b, r, c in shapes)
    # of the symmetric products, half
    flops = sum(STEPS * b * min(r, c) ** 2 * (3 * max(r, c) + min(r, c)) for b, r, c in shapes)
    # parameters and momenta in and out, gradients in
    return {"bytes": n * (2 * s if case["kind"] == "ortho" else 3 * s + 8), "flops": flops}


def _gradients(normal, shape):
    """A few directions that carry most of it over noise, rows of different scale."""
    b, r, c = shape
    k = max(1, min(r, c) // 16)
    return (normal(b, r, k) @ normal(b, k, c) / math.sqrt(k) + 0.5 * normal(*shape)) * torch.exp(0.5 * normal(b, r, 1))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["kind"] == "indexed":
        R, S, K, N = (case[k] for k in ("rows", "classes", "width", "out"))
        # classes as elements are: some common, others rare or absent; a few padding rows behind the last atom
        u = torch.rand(R, generator=gen, device=DEV, dtype=torch.float64)
        z = (S * u ** (1 + case["skew"])).long().clamp(max=S - 1)
        z = z[torch.randperm(R, generator=gen, device=DEV)]
        if R > 50:
            z[R - R // 50:] = -1
        st = {"case": case, "z": z, "x": (normal(R, K) * torch.exp(0.5 * normal(R, 1))).to(dt),
              "w": (normal(S, K, N) / math.sqrt(K)).to(dt)}
        # rows by class, classes out of range last: what a program keeps while its atoms are the same
        key = torch.where((z >= 0) & (z < S), z, S)
        st["order"] = torch.argsort(key, stable=True).int()
        counts = torch.bincount(key, minlength=S + 1)
        st["starts"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
        st["counts"] = counts.tolist()
        if case["direction"] == "backward":
            st["g"] = (normal(R, N) * torch.exp(0.5 * normal(R, 1))).to(dt)
            st["x"].requires_grad_(True)
            st["w"].requires_grad_(True)
        return st
    if case["kind"] == "ortho":
        return {"case": case, "x": (1e-3 * _gradients(normal, (case["batch"], case["rows"], case["width"]))).to(dt)}
    # parameters, gradients and momenta lie in one buffer each, so that what a pass returns is whole and few
    shapes = _shapes(case)
    sizes = [b * r * c for b, r, c in shapes]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + -(-n // 64) * 64)
    flat = {"p": torch.zeros(starts[-1], dtype=dt, device=DEV), "g": torch.zeros(starts[-1], dtype=dt, device=DEV),
            "m": torch.zeros(starts[-1], device=DEV)}
    st = {"case": case, "shapes": shapes, "flat": flat}
    for key, t in flat.items():
        st[key] = [t[a:a + n].view(s if s[0] > 1 else s[1:]) for a, n, s in zip(starts, sizes, shapes)]
    for k, s in enumerate(shapes):
        view = s if s[0] > 1 else s[1:]
        scale = math.exp(random.Random(k).gauss(-5, 1.5))  # tensors' gradients differ by orders of magnitude
        st["p"][k].copy_((normal(*s) / math.sqrt(s[2])).view(view))
        st["g"][k].copy_((scale * _gradients(normal, s)).view(view))
        st["m"][k].copy_((0.3 * scale * _gradients(normal, s)).view(view))
    return st


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _classes(st):
    """(class, its rows) of the classes present."""
    parts = st["order"].long().split(st["counts"])[:-1]
    return [(e, rows) for e, rows in enumerate(parts) if len(rows)]


def _plain_indexed(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    if case["plan"]:
        classes = _classes(st)
    else:  # grouped on the spot
        key = torch.where((st["z"] >= 0) & (st["z"] < case["classes"]), st["z"], case["classes"])
        counts = torch.bincount(key, minlength=case["classes"] + 1).tolist()
        classes = _classes({"order": torch.argsort(key), "counts": counts})
    x, w = st["x"].detach().float(), st["w"].detach().float()
    y = x.new_zeros(case["rows"], case["out"])
    for e, rows in classes:
        y[rows] = x[rows] @ w[e]
    if case["direction"] == "forward":
        return {"y": y.to(dt)}
    g = st["g"].float()
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    for e, rows in classes:
        part = g[rows]
        gx[rows] = part @ w[e].t()
        gw[e] = x[rows].t() @ part
    return {"y": y.to(dt), "gx": gx.to(dt), "gw": gw.to(dt)}


def _plain_ortho(x):
    """Of a (batch, rows, width) float32 stack."""
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / x.double().square().sum((1, 2), keepdim=True).sqrt().clamp(min=EPS).float()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = torch.bmm(x, x.transpose(1, 2))
        x = a * x + torch.bmm(b * A + c * torch.bmm(A, A), x)
    return x.transpose(1, 2) if tall else x


def _plain_muon(st):
    dt = DTYPES[st["case"]["dtype"]]
    alike = {}  # matrices of one shape are multiplied together
    for k, s in enumerate(st["shapes"]):
        alike.setdefault(s[1:], []).append(k)
    for (r, c), ks in alike.items():
        stack = lambda ts: torch.cat([ts[k].view(-1, r, c) for k in ks]).float()  # noqa: E731, B023
        g, m = stack(st["g"]), stack(st["m"])
        m = MU * m + (1 - MU) * g
        o = _plain_ortho((1 - MU) * g + MU * m)
        p = (1 - LR * DECAY) * stack(st["p"]) - LR * math.sqrt(max(1.0, r / c)) * o
        parts = [st["shapes"][k][0] for k in ks]
        torch._foreach_copy_([st["m"][k].view(-1, r, c) for k in ks], list(m.split(parts)))
        torch._foreach_copy_([st["p"][k].view(-1, r, c) for k in ks], list(p.to(dt).split(parts)))
    return {"p": st["flat"]["p"], "m": st["flat"]["m"]}


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------


def _own_indexed(st):
    from molnex_amd.molix import F

    x, w, z = st["x"], st["w"], st["z"]
    y = F.indexed_linear(x, w, z, groups=(st["order"], st["starts"]) if st["case"]["plan"] else None)
    if st["case"]["direction"] == "forward":
        return {"y": y}
    gx, gw = torch.autograd.grad(y, (x, w), st["g"])
    return {"y": y.detach(), "gx": gx, "gw": gw}


def _own_ortho(st):
    from molnex_amd.molix import F

    return {"o": F.orthogonalize(st["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}


def _own_muon(st):
    from molnex_amd.molix import F

    F.muon_step(st["p"], st["g"], st["m"], lr=LR, momentum=MU, nesterov=True, weight_decay=DECAY, steps=STEPS,
                coefficients=COEFFICIENTS, eps=EPS, adjust="original")
    return {"p": st["flat"]["p"], "m": st["flat"]["m"]}


def run(state):
    kind = state["case"]["kind"]
    if kind == "indexed":
        return (_own_indexed if own else _plain_indexed)(state)
    if kind == "ortho":
        if own:
            return _own_ortho(state)
        return {"o": _plain_ortho(state["x"].float()).to(state["x"].dtype).contiguous()}
    return (_own_muon if own else _plain_muon)(state)


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------


def _exact_indexed(st):
    """Class by class with every row and a mask, differentiated by autograd."""
    case = st["case"]
    x, w = (st[k].detach().double().requires_grad_(True) for k in ("x", "w"))
    back = case["direction"] == "backward"
    y = torch.zeros(case["rows"], case["out"], dtype=torch.float64, device=DEV)
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    for e in range(case["classes"]):
        rows = (st["z"] == e).nonzero().flatten()
        part = torch.mm(x[rows], w[e])
        y[rows] = part.detach()
        if back:
            dx, dw = torch.autograd.grad(part, (x, w), st["g"].double()[rows])
            gx += dx
            gw += dw
    return {"y": y, "gx": gx, "gw": gw} if back else {"y": y}


def _exact_ortho(g):
    """Of one matrix, by the polynomial of each step as the definition has it."""
    x = g.double()
    x = x / max(float(torch.linalg.matrix_norm(x)), EPS)
    x = x.t().contiguous() if x.shape[0] > x.shape[1] else x
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = torch.mm(x, x.t().contiguous())
        x = a * x + b * torch.mm(s, x) + c * torch.mm(s, torch.mm(s, x))
    return x.t() if g.shape[0] > g.shape[1] else x


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "indexed":
        if case["direction"] == "backward" and case["classes"] * case["rows"] * case["width"] > 2_000_000_000:
            return _exact_large(st)
        return _exact_indexed(st)
    if case["kind"] == "ortho":
        return {"o": torch.stack([_exact_ortho(x) for x in st["x"]])}
    p, m = st["flat"]["p"].double(), st["flat"]["m"].double()
    for k, (b, r, c) in enumerate(st["shapes"]):
        at = st["p"][k].storage_offset()
        put = lambda flat, t: flat[at:at + b * r * c].copy_(t.reshape(-1))  # noqa: E731, B023
        g, old, par = (st[key][k].double().view(b, r, c) for key in ("g", "m", "p"))
        new = old + (1 - MU) * (g - old)
        o = torch.stack([_exact_ortho(u) for u in g + MU * (new - g)])
        put(m, new)
        put(p, par - LR * DECAY * par - LR * math.sqrt(max(1.0, r / c)) * o)
    return {"p": p, "m": m}


def _exact_large(st):
    """The same with the gradients' formulas, for cases whose dense gradients per class would take too long."""
    case = st["case"]
    x, w, g = (st[k].detach().double() for k in ("x", "w", "g"))
    y, gx, gw = x.new_zeros(case["rows"], case["out"]), torch.zeros_like(x), torch.zeros_like(w)
    for e in range(case["classes"]):
        rows = (st["z"] == e).nonzero().flatten()
        xs, gs = x[rows], g[rows]
        y[rows] = torch.mm(xs, w[e])
        gx[rows] = torch.mm(gs, w[e].t().contiguous())
        gw[e] = torch.mm(xs.t().contiguous(), gs)
    return {"y": y, "gx": gx, "gw": gw}
