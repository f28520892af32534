"""The matrix products next to the exact-GP engine's own: products grouped by expert with ragged sizes (forward and
gradients) and products in 8-bit integers with one scale per row of either operand.

``listed`` names the cases, ``draw`` draws more of the same ranges, ``prepare`` makes what a program has in hand before
the call, ``run`` is one pass - elementary torch operations where ``own`` is false, the calls of ``battgp_amd.products``
where it is true - and ``exact`` gives the result in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # a battery system: the pack's and the 8 cells' query rows (300 points of a time grid each) against each one's
        # own inverse factor of 1000 training points, the reference's default size
        dict(name="grouped f64 system of 9 cells", op="grouped", dtype="f64", groups=9, rows=2700, n=1000, k=1000, split="even", tail=0, wt=False),
        # serving: a handful of rows routed over many experts, where reading the weights is all there is
        dict(name="grouped bf16 single rows", op="grouped", dtype="bf16", groups=64, rows=8, n=2048, k=1024, split="routed", tail=0, wt=False),
        # an ordinary batch of odd length, weights stored with the output axis contiguous, padding rows at the end
        dict(name="grouped bf16 odd batch", op="grouped", dtype="bf16", groups=8, rows=4099, n=2816, k=1000, split="routed", tail=37, wt=True),
        # the largest: a long prompt or a large training batch over 16 experts
        dict(name="grouped bf16 large", op="grouped", dtype="bf16", groups=16, rows=16384, n=4096, k=4096, split="routed", tail=0, wt=False),
        # gradients of the system's products at the default training size of 2000 rows a cell
        dict(name="grad f64 system of 9 cells", op="grad", dtype="f64", groups=9, rows=18000, n=500, k=512, split="even", tail=0, wt=False),
        # a small odd layer in single precision: nothing is a multiple of a tile or of 16 bytes
        dict(name="grad f32 odd", op="grad", dtype="f32", groups=5, rows=1237, n=333, k=513, split="routed", tail=11, wt=False),
        # a training step of an expert layer
        dict(name="grad bf16 training", op="grad", dtype="bf16", groups=16, rows=8192, n=2048, k=2048, split="routed", tail=0, wt=False),
        # serving in 8 bits: one row against a quantised layer
        dict(name="int8 bf16 one row", op="int8", dtype="bf16", m=1, n=4096, k=4096, add=False),
        # the grid of 300 query points, odd sizes, half precision
        dict(name="int8 f16 query grid", op="int8", dtype="f16", m=300, n=1001, k=2000, add=False),
        # one 8-bit slice of the operands of a 64-bit panel update (panel width 1024), added to what is there; the rest
        # of the rows is kept for the next slice
        dict(name="int8 f64 slice of a panel update", op="int8", dtype="f64", m=8192, n=1024, k=1024, add=True),
        # a large batch through a quantised layer
        dict(name="int8 bf16 large", op="int8", dtype="bf16", m=8192, n=8192, k=8192, add=False),
    ]


# floating point operations of the largest drawn case, by type: below the largest listed one's time in either form
MOST_FLOPS = {"f64": 4.0e10, "f32": 6.0e10, "bf16": 4.0e11, "f16": 4.0e11}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range: any integer in one case of two, else a multiple of 8."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.5 else max(lo, n // 8 * 8)


def draw(rng):
    op = rng.choice(["grouped", "grad", "int8"])
    while True:
        if op == "int8":
            dtype = rng.choice(["bf16", "f16", "f32", "f64"])
            case = dict(op=op, dtype=dtype, m=_log(rng, 1, 8192), n=_size(rng, 64, 8192), k=_size(rng, 64, 8192),
                        add=dtype in ("f64", "f32") and rng.random() < 0.5)
            if work(case)["flops"] <= MOST_FLOPS["bf16"]:
                return case
        else:
            dtype = rng.choice(["bf16", "bf16", "f16", "f32", "f64"])
            case = dict(op=op, dtype=dtype, groups=_log(rng, 1, 64), rows=_log(rng, 1, 16384), n=_size(rng, 64, 4096), k=_size(rng, 64, 4096),
                        split=rng.choice(["even", "routed"]), tail=rng.choice([0, 0, rng.randint(1, 100)]), wt=rng.random() < 0.3)
            w = work(case)
            if w["flops"] <= MOST_FLOPS[dtype] and w["bytes"] <= 3.0e9:
                return case


def _counts(case, seed):
    """Rows of each group: equal ones, or as a router deals them - uneven, some groups without any."""
    g, t = case["groups"], case["rows"]
    if case["split"] == "even":
        return np.array([t // g + (i < t % g) for i in range(g)], dtype=np.int64)
    rng = np.random.default_rng(seed)
    weight = rng.gamma(1.0, 1.0, g) + 0.02
    return rng.multinomial(t, weight / weight.sum()).astype(np.int64)


def prepare(case, seed):
    dtype, dev = DTYPES[case["dtype"]], torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dtype)

    st = dict(case)
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        # rows of different size, as activations are; the weights come quantised, one scale a channel
        st["x"] = normal(m, k) * torch.exp(normal(m, 1, dtype=torch.float32)).to(dtype)
        st["wq"] = torch.randint(-127, 128, (n, k), generator=gen, device=dev, dtype=torch.int8)
        st["wscale"] = (torch.rand(n, generator=gen, device=dev, dtype=torch.float32) + 0.5) / (127.0 * math.sqrt(k))
        st["wscale"] = st["wscale"].to(torch.float64 if dtype == torch.float64 else torch.float32)
        st["c"] = normal(m, n) if case["add"] else None
        return st
    g, n, k = case["groups"], case["n"], case["k"]
    bounds = np.concatenate(([0], np.cumsum(_counts(case, seed))))
    t = int(bounds[-1]) + case["tail"]
    st["bounds"] = [int(b) for b in bounds]  # the plain form's loop; the kernels read the device's copy
    st["offsets"] = torch.tensor(st["bounds"], dtype=torch.int64, device=dev)
    st["x"] = normal(t, k)
    st["w"] = normal(g, k, n, scale=1.0 / math.sqrt(k)).transpose(1, 2) if case["wt"] else normal(g, n, k, scale=1.0 / math.sqrt(k))
    if case["op"] == "grad":
        st["dy"] = normal(t, n, scale=1.0 / math.sqrt(n))
    return st


def _wide(t):
    """32 bits for the sums, 64 where the type has them."""
    return t if t.dtype == torch.float64 else t.float()


def _plain_quantize(x, slices):
    """Whole numbers within +-127 and a scale for each row; ``slices``: scales that are powers of two, and the rest."""
    stype = torch.float64 if x.dtype == torch.float64 else torch.float32
    tiny = torch.finfo(stype).tiny
    top = x.to(torch.float64).abs().amax(1, keepdim=True)
    scale = (top / 127.0).to(stype).clamp_min(tiny).to(torch.float64)
    if slices:
        mant, expo = torch.frexp(top)
        expo = expo - 7 + (mant > 127.0 / 128.0).to(expo.dtype)
        scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), expo), top).clamp_min(tiny)
    q = torch.round(x.to(torch.float64) / scale).clamp(-127, 127)  # in 64 bits: the border between two numbers
    rest = (x.to(torch.float64) - q * scale).to(x.dtype) if slices else None
    return q, scale.to(stype), rest


def run(state):
    op = state["op"]
    if own:
        from battgp_amd import products

        if op == "grouped":
            return products.grouped_matmul(state["x"], state["w"], state["offsets"])
        if op == "grad":
            return products.grouped_matmul_grad(state["dy"], state["x"], state["w"], state["offsets"])
        if state["add"]:
            q, scale, rest = products.quantize_rows(state["x"], pow2=True, residual=True)
            return products.int8_matmul(q, state["wq"], scale, state["wscale"], c=state["c"], dtype=state["x"].dtype), scale, rest
        q, scale = products.quantize_rows(state["x"])
        return products.int8_matmul(q, state["wq"], scale, state["wscale"], dtype=state["x"].dtype)

    x = state["x"]
    if op == "int8":
        q, scale, rest = _plain_quantize(x, state["add"])
        # sums of products of whole numbers: 32-bit floats hold them to 2^24 only
        y = (q @ state["wq"].to(torch.float64).T) * (scale.to(torch.float64) * state["wscale"].to(torch.float64))
        if state["add"]:
            return (y + state["c"]).to(x.dtype), scale[:, 0], rest
        return y.to(x.dtype)
    w, bounds = state["w"], state["bounds"]
    xw = _wide(x)
    if op == "grouped":
        y = torch.zeros(x.shape[0], w.shape[1], dtype=x.dtype, device=x.device)
        for g in range(w.shape[0]):
            a, b = bounds[g], bounds[g + 1]
            if b > a:
                y[a:b] = (xw[a:b] @ _wide(w[g]).T).to(x.dtype)
        return y
    dyw = _wide(state["dy"])
    dx = torch.zeros_like(x)
    dw = torch.zeros(w.shape, dtype=w.dtype, device=w.device)
    for g in range(w.shape[0]):
        a, b = bounds[g], bounds[g + 1]
        if b > a:
            dx[a:b] = (dyw[a:b] @ _wide(w[g])).to(x.dtype)
            dw[g] = (dyw[a:b].T @ xw[a:b]).to(w.dtype)
    return dx, dw


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        ssize = 8 if case["dtype"] == "f64" else 4
        more = (m * n + m * k) * size + m * ssize if case["add"] else 0  # what is added to, the rest, the scales
        return {"bytes": (m * k + m * n) * size + n * k + n * ssize + more, "flops": 2 * m * n * k}
    t, n, k, g = case["rows"], case["n"], case["k"], case["groups"]
    used = g if case["split"] == "even" else sum(1 for c in _counts(case, 0) if c)
    used = min(used, t)
    if case["op"] == "grouped":
        return {"bytes": (t * k + (t + case["tail"]) * n + used * n * k) * size + 8 * (g + 1), "flops": 2 * t * n * k}
    return {"bytes": (t * k + t * n + (t + case["tail"]) * k + used * n * k + g * n * k) * size + 8 * (g + 1), "flops": 4 * t * n * k}


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].double()
    if case["op"] == "int8":
        wide = case["dtype"] == "f64"
        top, _ = torch.max(torch.abs(x), dim=1)
        if case["add"]:
            # the smallest power of two p with max |x| <= 127 p
            p = torch.ldexp(torch.ones_like(top), torch.ceil(torch.log2(top / 127.0)).to(torch.int32))
            p = torch.where(top <= 127.0 * p / 2, p / 2, p)
            scale = torch.where(top > 127.0 * p, p * 2, p)
        else:
            scale = top / 127.0
            scale = scale if wide else scale.float().double()
        scale = torch.clamp(scale, min=2.0 ** -1022 if wide else 2.0 ** -126)
        ratio = x / scale[:, None]
        low = torch.floor(ratio)
        up = ratio - low
        q = torch.where((up > 0.5) | ((up == 0.5) & (torch.remainder(low, 2.0) == 1.0)), low + 1, low)
        q = torch.minimum(torch.maximum(q, torch.full_like(q, -127.0)), torch.full_like(q, 127.0))
        y = torch.matmul(q, st["wq"].double().t()) * scale[:, None] * st["wscale"].double()[None, :]
        if not case["add"]:
            return y
        return y + st["c"].double(), scale, x - scale[:, None] * q
    w = st["w"].double()
    group = torch.full((x.shape[0],), -1, dtype=torch.int64)
    for g, (a, b) in enumerate(zip(st["bounds"], st["bounds"][1:])):
        group[a:b] = g
    group = group.to(x.device)
    if case["op"] == "grouped":
        y = x.new_zeros(x.shape[0], case["n"])
        for g in range(case["groups"]):
            rows = torch.nonzero(group == g)[:, 0]
            y[rows] = torch.matmul(x[rows], w[g].t())
        return y
    dy = st["dy"].double()
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for g in range(case["groups"]):
        rows = torch.nonzero(group == g)[:, 0]
        dx[rows] = torch.matmul(dy[rows], w[g])
        dw[g] = torch.matmul(dy[rows].t(), x[rows])
    return dx, dw
