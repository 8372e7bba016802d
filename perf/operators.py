"""Workloads of the microscaled 4-bit operators and of the grouped product's gradients.

Three operators, each on the shapes of this framework's MoE layers:

* ``quantise``  rows -> 4-bit floating point (E2M1) with one scale per block of 32 (``mxfp4``,
  power-of-two scales) or 16 (``nvfp4``, E4M3 scales under a tensor scale) values, and the
  values these stand for;
* ``product``   the experts' product of two 4-bit operands over ragged row segments, plain or
  with the SwiGLU of a gate and an up projection;
* ``gradient``  the gradients of the experts' dense product: input gradient and weight gradient
  over ragged row segments.

``run`` computes them in elementary torch operations, or with ``own`` by the framework.
"""
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = {"mxfp4": 32, "nvfp4": 16}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_FLOPS, MOST_BYTES = 4.0e12, 3.0e9


# ------------------------------------------------------------------------------------ cases
def listed():
    q, p, g = "quantise", "product", "gradient"
    return [
        # one generated token's hidden state: latency
        {"name": "quantise mx token", "op": q, "format": "mxfp4", "type": "bf16", "rows": 1, "cols": 4096},
        # a prompt batch's hidden states, before the gate / up product
        {"name": "quantise mx prompt", "op": q, "format": "mxfp4", "type": "bf16", "rows": 8192, "cols": 4096},
        # the experts' hidden rows of a small batch, half precision, before the down product
        {"name": "quantise nv rows", "op": q, "format": "nvfp4", "type": "fp16", "rows": 1021, "cols": 2816},
        # one projection of 64 fine-grained experts, from fp32 weights, when a checkpoint is loaded
        {"name": "quantise nv weights", "op": q, "format": "nvfp4", "type": "fp32", "rows": 64 * 1408, "cols": 2048},
        # one token with two of eight experts: gate / up, the weights' bytes count
        {"name": "product mx token", "op": p, "format": "mxfp4", "rows": 2, "experts": 8, "n": 14336, "k": 4096,
         "swiglu": True, "skew": 0.0},
        # 64 decoded tokens' two experts each: down projection
        {"name": "product nv decode", "op": p, "format": "nvfp4", "rows": 128, "experts": 8, "n": 4096, "k": 14336,
         "swiglu": False, "skew": 0.3},
        # a prompt batch of 8192 tokens: gate / up with SwiGLU
        {"name": "product mx prompt", "op": p, "format": "mxfp4", "rows": 16384, "experts": 8, "n": 14336, "k": 4096,
         "swiglu": True, "skew": 0.3},
        # 16384 tokens' six of 64 fine-grained experts: down projection, uneven load
        {"name": "product nv fine", "op": p, "format": "nvfp4", "rows": 98304, "experts": 64, "n": 2048, "k": 1408,
         "swiglu": False, "skew": 0.5},
        # the small layer (512 tokens, two of eight experts): one training step's two gradients
        {"name": "gradient bf16 small", "op": g, "type": "bf16", "rows": 1024, "experts": 8, "n": 2816, "k": 1024,
         "skew": 0.3},
        # 4096 tokens' two experts each, the large layer's projection
        {"name": "gradient bf16 large", "op": g, "type": "bf16", "rows": 8192, "experts": 8, "n": 14336, "k": 4096,
         "skew": 0.3},
        # 2048 tokens' six of 64 fine-grained experts, uneven load, some experts without a row
        {"name": "gradient fp16 fine", "op": g, "type": "fp16", "rows": 12288, "experts": 64, "n": 1408, "k": 2048,
         "skew": 1.0},
        # full-precision training of the small layer, odd row count
        {"name": "gradient fp32 small", "op": g, "type": "fp32", "rows": 1021, "experts": 8, "n": 1024, "k": 2816,
         "skew": 0.3},
    ]


def draw(rng):
    def size(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(step, int(v / step + 0.5) * step)

    while True:
        op = rng.choice(("quantise", "product", "gradient"))
        if op == "quantise":
            c = {"op": op, "format": rng.choice(("mxfp4", "nvfp4")), "type": rng.choice(("bf16", "fp16", "fp32")),
                 "rows": size(1, 100000), "cols": size(64, 16384, 32)}
        elif op == "product":
            c = {"op": op, "format": rng.choice(("mxfp4", "nvfp4")), "rows": size(1, 50000),
                 "experts": size(1, 64), "n": size(64, 16384, rng.choice((1, 8, 64))), "k": size(64, 16384, 32),
                 "swiglu": rng.random() < 0.5, "skew": rng.choice((0.0, 0.3, 0.5, 1.0))}
        else:
            kind = rng.choice(("bf16", "bf16", "fp16", "fp32"))
            step = rng.choice((1, 8, 64))
            c = {"op": op, "type": kind, "rows": size(1, 20000), "experts": size(1, 64),
                 "n": size(64, 8192, step), "k": size(64, 8192, step), "skew": rng.choice((0.0, 0.3, 0.5, 1.0))}
            if kind == "fp32" and 4.0 * c["rows"] * c["n"] * c["k"] > 4.0e10:
                continue
        w = work(c)
        held = c.get("experts", 1) * c.get("n", 1) * c.get("k", 1)   # weight values, widened by the plain form
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and held <= 1.0e9:
            return c


def work(case):
    if case["op"] == "quantise":
        n = case["rows"] * case["cols"]
        elem = 4 if case["type"] == "fp32" else 2
        # read the rows; write the values (bf16) and one scale byte a block
        return {"bytes": n * (elem + 2) + n // BLOCK[case["format"]], "flops": 0}
    R, E, n, k = case["rows"], case["experts"], case["n"], case["k"]
    used = min(E, R)   # experts with rows
    if case["op"] == "product":
        bits = 0.5 + 1.0 / BLOCK[case["format"]]
        mats = 2 if case["swiglu"] else 1
        return {"bytes": R * k * bits + used * mats * n * k * bits + R * n * 2, "flops": 2.0 * mats * R * n * k}
    elem = 4 if case["type"] == "fp32" else 2
    # dY, X and the used weights in; dX and every expert's dW out
    return {"bytes": elem * (R * n + 2 * R * k + used * n * k + E * n * k), "flops": 4.0 * R * n * k}


# ------------------------------------------------------------------------------------ inputs
def _segments(case, gen, device):
    """Row counts of the experts (a multinomial over uneven loads), their offsets, and the most."""
    E, R = case["experts"], case["rows"]
    cpu = torch.Generator().manual_seed(gen.initial_seed())
    load = torch.exp(case["skew"] * torch.randn(E, generator=cpu))
    if case["skew"] >= 1.0 and E > 1:
        load[torch.rand(E, generator=cpu) < 0.15] = 0.0   # experts that get nothing
        load[0] += 1e-3
    if R <= E:   # a few rows: an expert each
        counts = torch.zeros(E, dtype=torch.int64)
        counts[torch.randperm(E, generator=cpu)[:R]] = 1
    else:
        counts = torch.bincount(torch.multinomial(load, R, replacement=True, generator=cpu), minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = torch.cumsum(counts, 0)
    return offsets.to(device), int(counts.max())


def _padded_rows(rows, n, device):
    """Scale rows as the quantiser lays them out: each padded to a multiple of 32 bytes."""
    return torch.zeros(*rows, (n + 31) // 32 * 32, dtype=torch.uint8, device=device)[..., :n]


def _operand(shape, fmt, std, gen, device):
    """4-bit codes, scale bytes and tensor scales of normal values, one leading index at a time."""
    rows, k = shape[:-1], shape[-1]
    q = torch.empty(*rows, k // 2, dtype=torch.uint8, device=device)
    s = _padded_rows(rows, k // BLOCK[fmt], device)
    lead = rows[0] if len(rows) == 2 else 1
    g = torch.ones(lead, dtype=torch.float32, device=device)
    for i in range(lead):
        x = torch.randn(rows[-1], k, generator=gen, device=device) * std
        if fmt == "nvfp4":
            g[i] = x.abs().amax() / 2688.0
        code, scale = _encode(x, fmt, g[i])
        (q[i] if len(rows) == 2 else q).copy_(code[:, 0::2] | (code[:, 1::2] << 4))
        (s[i] if len(rows) == 2 else s).copy_(scale)
    return q, s, g


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    if case["op"] == "quantise":
        t = TYPES[case["type"]]
        std = 0.02 if case["type"] == "fp32" else 1.0
        x = (torch.randn(case["rows"], case["cols"], generator=gen, device=device) * std).to(t)
        x[:, ::97] *= 8   # a few channels of a hidden state are much larger than the others
        # the tensor scale of nvfp4, as a calibration keeps it
        g = (x.float().abs().amax() / 2688.0).reshape(1) if case["format"] == "nvfp4" else None
        return {"case": case, "x": x, "global_scale": g}
    offsets, most = _segments(case, gen, device)
    R, E, n, k = case["rows"], case["experts"], case["n"], case["k"]
    st = {"case": case, "offsets": offsets, "most": most}
    if case["op"] == "product":
        fmt = case["format"]
        st["xq"], st["xs"], gx = _operand((R, k), fmt, 1.0, gen, device)
        st["wq"], st["ws"], gw = _operand((E, n, k), fmt, 0.02, gen, device)
        st["alpha"] = gx * gw
        if case["swiglu"]:
            st["uq"], st["us"], gu = _operand((E, n, k), fmt, 0.02, gen, device)
            st["alpha_up"] = gx * gu
        return st
    t = TYPES[case["type"]]
    st["x"] = torch.randn(R, k, generator=gen, device=device).to(t)
    st["dy"] = (torch.randn(R, n, generator=gen, device=device) * 0.1).to(t)
    st["w"] = torch.empty(E, n, k, dtype=t, device=device)
    for e in range(E):
        st["w"][e] = torch.randn(n, k, generator=gen, device=device) * 0.02
    return st


# ------------------------------------------------------------------------------------ plain forms
def _steps(t):
    """|t| to the nearest E2M1 code 0..7, ties to the even code."""
    c = (t > 0.25).to(torch.uint8)
    c += t >= 0.75
    c += t > 1.25
    c += t >= 1.75
    c += t > 2.5
    c += t >= 3.5
    c += t > 5.0
    return c


def _encode(x, fmt, g):
    """E2M1 codes (sign in bit 3) [rows, k] and scale bytes [rows, k / block] of x."""
    rows, k = x.shape
    b = BLOCK[fmt]
    xb = x.float().reshape(rows, k // b, b)
    amax = xb.abs().amax(-1)
    if fmt == "mxfp4":
        e = torch.frexp(amax)[1] - 3             # floor(log2(amax)) - 2
        e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
        scale = (e + 127).to(torch.uint8)
        c = _steps(torch.ldexp(xb.abs(), -e[..., None]))      # exact: a power of two
    else:
        # values next to a border: 64 bits
        t = amax.double() / (6.0 * g.double())
        step = torch.ldexp(torch.ones_like(t), torch.frexp(t)[1].clamp(min=-5) - 4)
        s = (torch.round(t / step) * step).clamp(max=448.0)
        scale = s.float().to(torch.float8_e4m3fn).view(torch.uint8)
        d = (s * g.double())[..., None]
        c = _steps(torch.where(d > 0, xb.abs().double() / d, torch.zeros_like(d)))
    c |= (xb < 0).to(torch.uint8) << 3
    return c.reshape(rows, k), scale.reshape(rows, k // b)


def _table(device):
    return torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=device)


def _scale_values(s, fmt):
    if fmt == "mxfp4":
        return torch.ldexp(torch.ones(1, dtype=torch.float32, device=s.device), s.int() - 127)
    return s.contiguous().view(torch.float8_e4m3fn).float()


def _decode(q, s, fmt):
    """The values [..., k] in fp32 (the tensor scale left out)."""
    v = _table(q.device)[torch.stack((q & 15, q >> 4), -1).int()].flatten(-2)
    b = BLOCK[fmt]
    return (v.unflatten(-1, (-1, b)) * _scale_values(s, fmt)[..., None]).flatten(-2)


def _places(offsets, R, most):
    """Expert and place within its segment of each row."""
    r = torch.arange(R, device=offsets.device, dtype=torch.int32)
    e = torch.searchsorted(offsets[1:].contiguous(), r, right=True)
    return e, (r - offsets[e]).long()


def _spread(rows, e, p, E, most):
    """Rows as [E, most, ...], zero behind each expert's last row."""
    out = torch.zeros(E, most, rows.shape[-1], dtype=torch.float32, device=rows.device)
    out[e, p] = rows
    return out


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "quantise":
        x, fmt, g = state["x"], case["format"], state["global_scale"]
        code, scale = _encode(x, fmt, g)
        v = _table(x.device)[code.int()].unflatten(-1, (-1, BLOCK[fmt])) * _scale_values(scale, fmt)[..., None]
        v = v.flatten(-2)
        return {"values": (v if g is None else v * g).to(torch.bfloat16), "scales": scale}
    R, E, most = case["rows"], case["experts"], state["most"]
    e, p = _places(state["offsets"], R, most)
    if case["op"] == "product":
        fmt = case["format"]
        x = _spread(_decode(state["xq"], state["xs"], fmt), e, p, E, most)
        y = torch.bmm(x, _decode(state["wq"], state["ws"], fmt).transpose(1, 2))[e, p] * state["alpha"][e][:, None]
        if case["swiglu"]:
            u = torch.bmm(x, _decode(state["uq"], state["us"], fmt).transpose(1, 2))[e, p]
            y = y / (1.0 + torch.exp(-y)) * (u * state["alpha_up"][e][:, None])
        return y.to(torch.bfloat16)
    t = state["x"].dtype
    x = _spread(state["x"].float(), e, p, E, most)
    dy = _spread(state["dy"].float(), e, p, E, most)
    dx = torch.bmm(dy, state["w"].float())[e, p]
    dw = torch.bmm(dy.transpose(1, 2), x)
    return {"dx": dx.to(t), "dw": dw.to(t)}


def _run_own(state, case):
    from light_moe_b200 import ops

    if case["op"] == "quantise":
        q, s = ops.quantize_fp4(state["x"], case["format"], global_scale=state["global_scale"])
        return {"values": ops.dequantize_fp4(q, s, case["format"], global_scale=state["global_scale"]), "scales": s}
    if case["op"] == "product":
        up = {}
        if case["swiglu"]:
            up = {"weights_up": state["uq"], "weight_scales_up": state["us"], "alpha_up": state["alpha_up"]}
        return ops.fp4_grouped_gemm(state["xq"], state["xs"], state["wq"], state["ws"], state["offsets"],
                                    case["experts"], case["format"], alpha=state["alpha"], **up)
    dx = ops.grouped_gemm_dgrad(state["dy"], state["w"], state["offsets"], case["experts"])
    dw = ops.grouped_gemm_wgrad(state["dy"], state["x"], state["offsets"], case["experts"])
    return {"dx": dx, "dw": dw}


# ------------------------------------------------------------------------------------ 64 bits
def _nearest(t):
    """The E2M1 value nearest to t >= 0, by distance; of two as near the one of the even code."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=t.device)
    best = torch.zeros_like(t)
    dist = t.clone()
    for i in range(1, 8):
        d = (t - grid[i]).abs()
        near = (d < dist) | ((d == dist) & (i % 2 == 0))
        best = torch.where(near, grid[i], best)
        dist = torch.where(near, d, dist)
    return best


def _exact_values(x, fmt, g):
    """What a block-scaled row stands for, and the scale bytes, from the definition in 64 bits."""
    b = BLOCK[fmt]
    xb = x.double().reshape(x.shape[0], -1, b)
    top = xb.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)))
        e = torch.where(2.0 ** (e + 1) <= top, e + 1, torch.where(2.0 ** e > top, e - 1, e))
        e = (e - 2).clamp(-127, 127)
        unit, byte = 2.0 ** e, e + 127
    else:
        grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
        want = (top / (6.0 * g)).clamp(max=448.0)
        hi = torch.searchsorted(grid, want.flatten().contiguous()).clamp(max=126).view_as(want)
        lo = (hi - 1).clamp(min=0)
        dl, dh = want - grid[lo], grid[hi] - want
        byte = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
        unit = grid[byte] * g
    v = torch.where(unit > 0, _nearest(xb.abs() / unit) * unit, torch.zeros_like(xb)) * torch.sign(xb)
    return v.reshape(x.shape), byte.reshape(x.shape[0], -1).to(torch.uint8)


def _read(q, s, fmt):
    """Values of codes and scale bytes in 64 bits."""
    sign = torch.tensor((1.0, -1.0), dtype=torch.float64, device=q.device)
    grid = torch.tensor(E2M1, dtype=torch.float64, device=q.device)
    v = torch.empty(*q.shape[:-1], q.shape[-1] * 2, dtype=torch.float64, device=q.device)
    for half, c in ((0, q & 15), (1, q >> 4)):
        v[..., half::2] = grid[(c & 7).long()] * sign[(c >> 3).long()]
    unit = 2.0 ** (s.double() - 127) if fmt == "mxfp4" else s.contiguous().view(torch.float8_e4m3fn).double()
    return v * torch.repeat_interleave(unit, BLOCK[fmt], dim=-1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantise":
        g = 1.0 if st["global_scale"] is None else st["global_scale"].double()
        got = [_exact_values(part, case["format"], g) for part in st["x"].split(8192)]
        return {"values": torch.cat([v for v, _ in got]), "scales": torch.cat([b for _, b in got])}
    R, n, k = case["rows"], case["n"], case["k"]
    bounds = st["offsets"].tolist()
    device = st["offsets"].device
    if case["op"] == "product":
        fmt = case["format"]
        y = torch.zeros(R, n, dtype=torch.float64, device=device)
        for e in range(case["experts"]):
            a, b = bounds[e], bounds[e + 1]
            if a == b:
                continue
            x = _read(st["xq"][a:b], st["xs"][a:b], fmt)
            v = x @ _read(st["wq"][e], st["ws"][e], fmt).T * st["alpha"][e].double()
            if case["swiglu"]:
                u = x @ _read(st["uq"][e], st["us"][e], fmt).T * st["alpha_up"][e].double()
                v = v * torch.sigmoid(v) * u
            y[a:b] = v
        return y
    dx = torch.zeros(R, k, dtype=torch.float64, device=device)
    dw = torch.zeros(case["experts"], n, k, dtype=torch.float64, device=device)
    for e in range(case["experts"]):
        a, b = bounds[e], bounds[e + 1]
        dy = st["dy"][a:b].double()
        dx[a:b] = dy @ st["w"][e].double()
        dw[e] = dy.T @ st["x"][a:b].double()
    return {"dx": dx, "dw": dw}
