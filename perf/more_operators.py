"""Workloads of the 8-bit floating-point operators and of the MoE layer for a few tokens.

Three operators, each on the shapes of this framework's MoE layers:

* ``quantise``  values -> 8-bit floating point (E4M3) with one fp32 scale per 128 columns of a row
  (activations) or per block of 128 x 128 (weights), and the values these stand for;
* ``product``   the experts' product of two such operands over ragged row segments, plain or with
  the SwiGLU of a gate and an up projection;
* ``layer``     a whole MoE layer (router, experts, weighted sum) for up to 16 tokens, with dense
  16-bit or block-scaled 8-bit experts.

``run`` computes them in elementary torch operations, or with ``own`` by the framework.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -126
MOST_FLOPS, MOST_BYTES = 4.0e12, 3.0e9


# ------------------------------------------------------------------------------------ cases
def listed():
    q, p, m = "quantise", "product", "layer"
    return [
        # one generated token's hidden state: latency
        {"name": "quantise token", "op": q, "type": "bf16", "count": 1, "rows": 1, "cols": 4096, "block_rows": 1,
         "power": False},
        # a prompt batch's hidden states, before the gate / up product
        {"name": "quantise prompt", "op": q, "type": "bf16", "count": 1, "rows": 8192, "cols": 4096, "block_rows": 1,
         "power": False},
        # the experts' hidden rows of a small batch, half precision, scales that are powers of two
        {"name": "quantise rows", "op": q, "type": "fp16", "count": 1, "rows": 1021, "cols": 2816, "block_rows": 1,
         "power": True},
        # one projection of 64 fine-grained experts, from fp32 weights, when a checkpoint is converted
        {"name": "quantise weights", "op": q, "type": "fp32", "count": 64, "rows": 1408, "cols": 2048,
         "block_rows": 128, "power": False},
        # nine tokens' two of eight experts: gate / up, the weights' bytes count
        {"name": "product few", "op": p, "rows": 18, "experts": 8, "n": 14336, "k": 4096, "swiglu": True, "skew": 0.0},
        # 64 decoded tokens' two experts each: down projection
        {"name": "product decode", "op": p, "rows": 128, "experts": 8, "n": 4096, "k": 14336, "swiglu": False,
         "skew": 0.3},
        # a prompt batch of 8192 tokens: gate / up with SwiGLU
        {"name": "product prompt", "op": p, "rows": 16384, "experts": 8, "n": 14336, "k": 4096, "swiglu": True,
         "skew": 0.3},
        # 16384 tokens' six of 64 fine-grained experts: down projection, uneven load
        {"name": "product fine", "op": p, "rows": 98304, "experts": 64, "n": 2048, "k": 1408, "swiglu": False,
         "skew": 0.5},
        # one generated token through the large layer
        {"name": "layer fp8 token", "op": m, "weights": "fp8", "type": "bf16", "tokens": 1, "experts": 8, "top_k": 2,
         "shared": 0, "d": 4096, "ffn": 14336, "bias": False},
        # seven tokens (a small batch of streams) through the fine-grained layer with its shared experts
        {"name": "layer fp8 fine", "op": m, "weights": "fp8", "type": "bf16", "tokens": 7, "experts": 64, "top_k": 6,
         "shared": 2, "d": 2048, "ffn": 1408, "bias": False},
        # four tokens through the large layer with dense experts
        {"name": "layer bf16 four", "op": m, "weights": "dense", "type": "bf16", "tokens": 4, "experts": 8,
         "top_k": 2, "shared": 0, "d": 4096, "ffn": 14336, "bias": False},
        # one token through the small layer in half precision, a router with a bias: latency
        {"name": "layer fp16 small", "op": m, "weights": "dense", "type": "fp16", "tokens": 1, "experts": 8,
         "top_k": 2, "shared": 0, "d": 1024, "ffn": 2816, "bias": True},
    ]


def draw(rng):
    def size(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(step, int(v / step + 0.5) * step)

    while True:
        op = rng.choice(("quantise", "product", "layer"))
        if op == "quantise":
            block = rng.choice((1, 1, 128))
            c = {"op": op, "type": rng.choice(("bf16", "fp16", "fp32")), "count": size(1, 64) if block > 1 else 1,
                 "rows": size(1, 100000 if block == 1 else 16384), "cols": size(64, 16384, rng.choice((16, 128))),
                 "block_rows": block, "power": rng.random() < 0.3}
            held = c["count"] * c["rows"] * c["cols"]
            if held > 2.0e8:
                continue
        elif op == "product":
            c = {"op": op, "rows": size(1, 50000), "experts": size(1, 64), "n": size(64, 16384, rng.choice((1, 8, 64))),
                 "k": size(64, 16384, rng.choice((16, 128))), "swiglu": rng.random() < 0.5,
                 "skew": rng.choice((0.0, 0.3, 0.5, 1.0))}
            held = c["experts"] * c["n"] * c["k"]
        else:
            E = size(1, 128)
            c = {"op": op, "weights": rng.choice(("fp8", "fp8", "dense")), "type": rng.choice(("bf16", "bf16", "fp16")),
                 "tokens": size(1, 16), "experts": E, "top_k": min(E, size(1, 8)), "shared": rng.choice((0, 0, 1, 2)),
                 "d": size(128, 8192, 64), "ffn": size(64, 16384, 32), "bias": rng.random() < 0.3}
            held = (E + c["shared"]) * c["d"] * c["ffn"]
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and held <= 5.0e8:
            return c


def work(case):
    if case["op"] == "quantise":
        rows, cols = case["count"] * case["rows"], case["cols"]
        elem = 4 if case["type"] == "fp32" else 2
        blocks = case["count"] * -(-case["rows"] // case["block_rows"]) * -(-cols // BLOCK)
        # read the values; write what they stand for (in their type) and the scales
        return {"bytes": rows * cols * 2 * elem + 4 * blocks, "flops": 0}
    if case["op"] == "product":
        R, E, n, k = case["rows"], case["experts"], case["n"], case["k"]
        mats, kb = (2 if case["swiglu"] else 1), -(-k // BLOCK)
        used = min(E, R)   # experts with rows
        return {"bytes": R * (k + 4 * kb) + used * mats * (n * k + 4 * kb * -(-n // BLOCK)) + R * n * 2,
                "flops": 2.0 * mats * R * n * k}
    T, E, k, S, d, f = (case[i] for i in ("tokens", "experts", "top_k", "shared", "d", "ffn"))
    used = E * (1.0 - (1.0 - k / E) ** T) + S   # experts that T tokens reach, on average
    per = 3 * d * f * (1 + 4 / BLOCK ** 2 if case["weights"] == "fp8" else 2)
    return {"bytes": int(used * per + E * d * 2 + T * d * 4 + T * k * 8),
            "flops": 2.0 * T * (3 * d * f * (k + S) + E * d)}


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


def _rows_operand(rows, k, gen, device):
    """Codes of normal rows and their scales, which the quantiser lays out block by block."""
    kb = -(-k // BLOCK)
    q = torch.empty(rows, k, dtype=torch.float8_e4m3fn, device=device)
    s = torch.ones(kb, (rows + 3) // 4 * 4, dtype=torch.float32, device=device).t()[:rows]
    for a in range(0, rows, 8192):
        x = torch.randn(min(8192, rows - a), k, generator=gen, device=device)
        code, scale = _encode(x, 1, False, torch.float32)
        q[a:a + 8192] = code.to(torch.float8_e4m3fn)
        s[a:a + 8192] = scale
    return q, s


def _weights(shape, std, gen, device):
    """Codes [count, n, k] and scales of normal weights, a matrix at a time."""
    q = torch.empty(shape, dtype=torch.float8_e4m3fn, device=device)
    s = torch.empty(shape[0], -(-shape[1] // BLOCK), -(-shape[2] // BLOCK), dtype=torch.float32, device=device)
    for i in range(shape[0]):
        x = torch.randn(shape[1:], generator=gen, device=device) * std
        code, s[i] = _encode(x, BLOCK, False, torch.float32)
        q[i] = code.to(torch.float8_e4m3fn)
    return q, s


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    if case["op"] == "quantise":
        t = TYPES[case["type"]]
        std = 0.02 if case["block_rows"] > 1 else 1.0
        x = torch.empty(case["count"], case["rows"], case["cols"], dtype=t, device=device)
        for part in x:
            part.copy_(torch.randn(part.shape, generator=gen, device=device) * std)
        if case["block_rows"] == 1:
            x[..., ::97] *= 8   # a few channels of a hidden state are much larger than the others
        return {"case": case, "x": x if case["block_rows"] > 1 else x[0]}
    if case["op"] == "product":
        offsets, most = _segments(case, gen, device)
        R, E, n, k = case["rows"], case["experts"], case["n"], case["k"]
        st = {"case": case, "offsets": offsets, "most": most}
        st["xq"], st["xs"] = _rows_operand(R, k, gen, device)
        st["wq"], st["ws"] = _weights((E, n, k), 0.02, gen, device)
        if case["swiglu"]:
            st["uq"], st["us"] = _weights((E, n, k), 0.02, gen, device)
        return st
    t = TYPES[case["type"]]
    T, E, S, d, f = (case[i] for i in ("tokens", "experts", "shared", "d", "ffn"))
    x = torch.randn(T, d, generator=gen, device=device)
    x[:, ::97] *= 8
    st = {"case": case, "x": x.to(t), "gate": (torch.randn(E, d, generator=gen, device=device) * 0.02).to(t)}
    st["bias"] = torch.randn(E, generator=gen, device=device) * 0.1 if case["bias"] else None
    for name, shape in (("w1", (E + S, f, d)), ("w3", (E + S, f, d)), ("w2", (E + S, d, f))):
        if case["weights"] == "fp8":
            st[name], st[name + "_scales"] = _weights(shape, 0.02, gen, device)
        else:
            st[name] = torch.empty(shape, dtype=t, device=device)
            for part in st[name]:
                part.copy_(torch.randn(part.shape, generator=gen, device=device) * 0.02)
    return st


# ------------------------------------------------------------------------------------ plain forms
def _blocks(x, block_rows):
    """[rows, cols] -> [row blocks, block_rows, column blocks, 128], zero behind the ends."""
    rows, cols = x.shape
    pad = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    return pad.reshape(-1, block_rows, pad.shape[1] // BLOCK, BLOCK)


def _encode(x, block_rows, power, dtype=torch.float64):
    """The E4M3 values of the codes of x [rows, cols] and the scales [row blocks, column blocks]."""
    rows, cols = x.shape
    xb = _blocks(x.float(), block_rows)
    top = xb.abs().amax((1, 3))
    scale = (top / torch.full_like(top, TOP)).clamp(min=LEAST)   # by a number it would be times its reciprocal
    if power:
        m, e = torch.frexp(scale)                    # scale = m * 2^e, m in [0.5, 1)
        scale = torch.ldexp(torch.ones_like(scale), torch.where(m > 0.5, e, e - 1))
    t = xb.to(dtype) / scale.to(dtype)[:, None, :, None]   # values next to a border: 64 bits
    step = torch.ldexp(torch.ones_like(t), torch.frexp(t)[1].clamp(min=-5) - 4)
    code = (torch.round(t / step) * step).clamp(-TOP, TOP).float()
    return code.reshape(xb.shape[0] * block_rows, -1)[:rows, :cols], scale


def _decode(q, s, block_rows):
    """Values [rows, cols] in fp32 of codes and their block scales."""
    rows, cols = q.shape
    each = s.repeat_interleave(BLOCK, 1)[:, :cols]
    if block_rows > 1:
        each = each.repeat_interleave(block_rows, 0)[:rows]
    return q.float() * each


def _silu(g):
    return g / (1.0 + torch.exp(-g))


def _route(x, gate, bias, top_k):
    """Experts [T, k] (most probable first, ties to the lower id) and their weights in fp32."""
    # which experts are chosen: 64 bits; their weights: 32
    logits = x.double() @ gate.double().T
    if bias is not None:
        logits = logits + bias.double()
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top_k]
    l32 = x.float() @ gate.float().T
    if bias is not None:
        l32 = l32 + bias
    p = torch.exp(l32 - l32.amax(1, keepdim=True)).gather(1, ids)
    return ids.int(), p / p.sum(1, keepdim=True)


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "quantise":
        x, b = state["x"], case["block_rows"]
        values = torch.empty_like(x)
        parts, scales = (x, []) if x.dim() == 3 else (x[None], [])
        for i, part in enumerate(parts):
            code, scale = _encode(part, b, case["power"])
            (values[i] if x.dim() == 3 else values).copy_(_decode(code, scale, b))
            scales.append(scale)
        return {"values": values, "scales": torch.stack(scales) if x.dim() == 3 else scales[0]}
    if case["op"] == "product":
        R, E, most, off = case["rows"], case["experts"], state["most"], state["offsets"]
        y = torch.empty(R, case["n"], dtype=torch.bfloat16, device=off.device)
        x = _decode(state["xq"], state["xs"], 1)
        r = torch.arange(R, device=off.device)
        place = torch.arange(most, device=off.device)
        for e in range(E):
            # this expert's rows, padded to the largest segment: the counts stay on the device
            rows = off[e] + place
            mine = x[rows.clamp(max=R - 1)]
            v = mine @ _decode(state["wq"][e], state["ws"][e], BLOCK).T
            if case["swiglu"]:
                v = _silu(v) * (mine @ _decode(state["uq"][e], state["us"][e], BLOCK).T)
            inside = ((r >= off[e]) & (r < off[e + 1]))[:, None]
            v = v.to(torch.bfloat16)[(r - off[e]).clamp(0, most - 1)]
            y = torch.where(inside, v, y)
        return y
    x = state["x"].float()
    ids, weights = _route(state["x"], state["gate"], state["bias"], case["top_k"])
    E, S = case["experts"], case["shared"]
    share = torch.zeros(case["tokens"], E + S, dtype=torch.float32, device=x.device)
    share.scatter_(1, ids.long(), weights)
    share[:, E:] = 1.0
    y = torch.zeros_like(x)
    for e in range(E + S):
        if case["weights"] == "fp8":
            w1, w3, w2 = (_decode(state[i][e], state[i + "_scales"][e], BLOCK) for i in ("w1", "w3", "w2"))
        else:
            w1, w3, w2 = (state[i][e].float() for i in ("w1", "w3", "w2"))
        part = (_silu(x @ w1.T) * (x @ w3.T)) @ w2.T
        y += torch.where(share[:, e:e + 1] != 0, part * share[:, e:e + 1], torch.zeros_like(part))
    return {"y": y.to(state["x"].dtype), "ids": ids, "weights": weights}


def _run_own(state, case):
    from light_moe_b200 import ops

    if case["op"] == "quantise":
        q, s = ops.quantize_fp8(state["x"], block_rows=case["block_rows"], power_of_two=case["power"])
        return {"values": ops.dequantize_fp8(q, s, block_rows=case["block_rows"], out_dtype=state["x"].dtype),
                "scales": s}
    if case["op"] == "product":
        up = {"weights_up": state["uq"], "weight_scales_up": state["us"]} if case["swiglu"] else {}
        return ops.fp8_grouped_gemm(state["xq"], state["xs"], state["wq"], state["ws"], state["offsets"],
                                    case["experts"], **up)
    scales = {i + "_scales": state[i + "_scales"] for i in ("w1", "w3", "w2")} if case["weights"] == "fp8" else {}
    y, ids, weights = ops.moe_layer_few_tokens(state["x"], state["gate"], state["w1"], state["w3"], state["w2"],
                                               case["top_k"], num_shared=case["shared"], gate_bias=state["bias"],
                                               **scales)
    return {"y": y, "ids": ids, "weights": weights}


# ------------------------------------------------------------------------------------ 64 bits
def _read(q, s, block_rows):
    """Values of codes [rows, cols] and scales in 64 bits."""
    out = q.double()
    for j in range(s.shape[1]):
        cols = slice(j * BLOCK, (j + 1) * BLOCK)
        if block_rows == 1:
            out[:, cols] *= s[:, j:j + 1].double()
        else:
            for i in range(s.shape[0]):
                out[i * block_rows:(i + 1) * block_rows, cols] *= s[i, j].double()
    return out


def _nearest(t):
    """The E4M3 value nearest to t >= 0, of two as near the one of the even code; at most 448."""
    grid = torch.arange(127, dtype=torch.uint8, device=t.device).view(torch.float8_e4m3fn).double()
    hi = torch.searchsorted(grid, t.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = (t - grid[lo]).abs(), (grid[hi] - t).abs()
    return grid[torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)]


def _exact_quantise(x, block_rows, power):
    rows, cols = x.shape
    values = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    scales = torch.empty(-(-rows // block_rows), -(-cols // BLOCK), dtype=torch.float64, device=x.device)
    for j in range(scales.shape[1]):
        v = x[:, j * BLOCK:(j + 1) * BLOCK].double()
        top = v.abs().amax(1)
        if block_rows > 1:
            top = torch.nn.functional.pad(top, (0, -rows % block_rows)).reshape(-1, block_rows).amax(1)
        # the scale is an fp32 number: the nearest one
        s = (top.double() / TOP).float().double().clamp(min=LEAST)
        if power:
            def two_to(e):   # (a power function may be a step off)
                return torch.ldexp(torch.ones_like(s), e.int())

            e = torch.floor(torch.log2(s))
            e = torch.where(two_to(e) < s, e + 1, e)
            s = two_to(torch.where(two_to(e - 1) >= s, e - 1, e))
        scales[:, j] = s
        each = s.repeat_interleave(block_rows)[:rows, None]
        values[:, j * BLOCK:(j + 1) * BLOCK] = _nearest(v.abs() / each) * torch.sign(v) * each
    return values, scales


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantise":
        x, b = st["x"], case["block_rows"]
        if x.dim() == 2:
            values, scales = _exact_quantise(x, b, case["power"])
            return {"values": values, "scales": scales}
        got = [_exact_quantise(part, b, case["power"]) for part in x]
        return {"values": torch.stack([v for v, _ in got]), "scales": torch.stack([s for _, s in got])}
    if case["op"] == "product":
        bounds = st["offsets"].tolist()
        y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=st["offsets"].device)
        for e in range(case["experts"]):
            a, b = bounds[e], bounds[e + 1]
            if a == b:
                continue
            x = _read(st["xq"][a:b], st["xs"][a:b], 1)
            v = x @ _read(st["wq"][e], st["ws"][e], BLOCK).T
            if case["swiglu"]:
                v = v * torch.sigmoid(v) * (x @ _read(st["uq"][e], st["us"][e], BLOCK).T)
            y[a:b] = v
        return y
    x, k, E, S = st["x"].double(), case["top_k"], case["experts"], case["shared"]
    logits = x @ st["gate"].double().T
    if st["bias"] is not None:
        logits = logits + st["bias"].double()
    p = torch.softmax(logits, 1)
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]
    weights = p.gather(1, ids)
    weights = weights / weights.sum(1, keepdim=True)
    y = torch.zeros_like(x)

    def matrix(name, e):
        return _read(st[name][e], st[name + "_scales"][e], BLOCK) if case["weights"] == "fp8" else st[name][e].double()

    for e in range(E + S):
        hit = (ids == e).nonzero() if e < E else None
        if hit is not None and hit.shape[0] == 0:
            continue
        t = hit[:, 0] if hit is not None else torch.arange(x.shape[0], device=x.device)
        w = weights[hit[:, 0], hit[:, 1]][:, None] if hit is not None else 1.0
        g = x[t] @ matrix("w1", e).T
        h = g * torch.sigmoid(g) * (x[t] @ matrix("w3", e).T)
        y[t] += w * (h @ matrix("w2", e).T)
    return {"y": y, "ids": ids.int(), "weights": weights}
