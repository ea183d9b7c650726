"""Performance cases of microscaled 4-bit floating point (MXFP4).

A block of 32 consecutive values along K shares a power of two 2^e, e the
exponent of the block's largest magnitude less 2, and each value is one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^e with a sign: the nearest one, ties to the
even code, what lies beyond 6 to 6.  Codes are packed two a byte (the lower k in
the low bits), the exponent is a byte e + 127.

Three kinds of work, each called as a serving program calls it:

  quantize  activations or a weight to blocks and back to values
  linear    decoder projections (fused qkv, o, gated gate/up, down) with MXFP4
            weights: x is quantised on the way, y = Q(x) W^T (+ bias), for the
            gate/up projection followed by silu(gate) * up
  experts   the two products of a block of MXFP4 experts: gate/up with
            silu(gate) * up over the tokens' routed rows, and down times the
            routed weight; the rows are quantised on the way

Up to GRAPH_MAX rows a step is captured in one graph, as a serving program
captures its decode step, over a stack of layers whose weights are larger than
the Infinity Cache where they can be; longer inputs run eagerly, and so do the
smallest calls.

Inputs: activations N(0, 1) with channels of different spread (a log-normal of
0.5, as behind a norm's weights), weights N(0, 1 / K) quantised; expert choices
the top of N(0, 1) logits, where a case says so shifted by a preference for some
experts.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 32

# Largest batch that a serving program captures; longer inputs run eagerly.
GRAPH_MAX = 160


def _quantize(name, rows, cols, dtype="bf16"):
    return {"name": name, "kind": "quantize", "M": rows, "K": cols, "dtype": dtype}


def _linear(name, dims, M, layers, dtype="fp16", bias=False, proj="layer"):
    hidden, q, kv, attn, inter = dims
    return {"name": name, "kind": "linear", "proj": proj, "hidden": hidden, "q": q, "kv": kv, "attn": attn,
            "inter": inter, "M": M, "layers": layers, "dtype": dtype, "bias": bias}


def _experts(name, E, top_k, hidden, inter, T, layers, dtype="fp16", skew=0.0):
    return {"name": name, "kind": "experts", "E": E, "top_k": top_k, "hidden": hidden, "inter": inter, "M": T,
            "layers": layers, "dtype": dtype, "skew": skew}


# (hidden, q columns, k and v columns each, attention width, intermediate):
# Qwen3-4B, Llama-3-8B and one GPU's share of tensor-parallel Llama-3.1-70B (TP8)
# and Llama-3-8B (TP4).
QWEN3_4B = (2560, 4096, 1024, 4096, 9728)
LLAMA3_8B = (4096, 4096, 1024, 4096, 14336)
LLAMA3_70B_TP8 = (8192, 1024, 128, 1024, 3584)
LLAMA3_8B_TP4 = (4096, 1024, 256, 1024, 3584)
DIMS = (QWEN3_4B, LLAMA3_8B, LLAMA3_70B_TP8, LLAMA3_8B_TP4)


def listed():
    return [
        # A few tokens' activations, called eagerly.
        _quantize("quantize_x_m7", 7, 2560),
        # A 16-bit checkpoint's gate/up weight as it is loaded.
        _quantize("quantize_w_8b", 28672, 4096),
        # One o projection for one token, called eagerly.
        _linear("linear_o_m1", QWEN3_4B, 1, 1, proj="o"),
        # Decode of a single sequence.
        _linear("linear_4b_m1", QWEN3_4B, 1, 12),
        # A decode batch.
        _linear("linear_4b_m24_bf16", QWEN3_4B, 24, 12, dtype="bf16"),
        # A large captured decode batch.
        _linear("linear_8b_m128", LLAMA3_8B, 128, 4, bias=True),
        # The ragged last chunk of a few prompts.
        _linear("linear_4b_m333", QWEN3_4B, 333, 1, dtype="bf16"),
        # The largest prefill chunk the scheduler forms.
        _linear("linear_8b_m8192_bf16", LLAMA3_8B, 8192, 1, dtype="bf16"),
        # Qwen3-30B-A3B-shaped experts: one token, a decode batch and a long chunk.
        _experts("experts_t1", 128, 8, 2048, 768, 1, 4),
        _experts("experts_t24_bf16", 128, 8, 2048, 768, 24, 2, dtype="bf16"),
        _experts("experts_t4096_bf16", 128, 8, 2048, 768, 4096, 1, dtype="bf16"),
        # Few wide experts, an uneven load, an odd chunk.
        _experts("experts_wide_t777", 16, 2, 4096, 1408, 777, 1, skew=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    dtype = rng.choice(("fp16", "bf16"))
    kind = rng.random()
    if kind < 0.2:
        M = _log_int(rng, 1, 28672)
        c = _quantize("", M, BLOCK * _log_int(rng, 8, 448 if M <= 8192 else 128),
                      rng.choice(("fp16", "bf16", "fp32")))
    elif kind < 0.6:
        dims = rng.choice(DIMS)
        M = _log_int(rng, 1, 8192)
        proj = "o" if rng.random() < 0.15 else "layer"
        layers = rng.choice((3, 4, 6)) if M <= GRAPH_MAX and proj == "layer" else 1
        c = _linear("", dims, M, layers, dtype, rng.random() < 0.4, proj)
    else:
        E = rng.choice((16, 32, 64, 128))
        top_k = rng.choice((2, 4, 6, 8))
        hidden = rng.choice((1024, 2048, 4096))
        inter = rng.choice((384, 512, 768, 1024, 1408))
        while E * hidden * inter > 128 * 2048 * 768:
            E //= 2
        T = _log_int(rng, 1, 4096)
        while T * top_k * hidden * inter > 4096 * 8 * 2048 * 768:
            T = T * 3 // 4
        layers = rng.choice((1, 2, 3)) if T <= GRAPH_MAX else 1
        c = _experts("", E, top_k, hidden, inter, T, layers, dtype, rng.choice((0.0, 0.5, 1.0)))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# Inputs, from the seed alone.
# ---------------------------------------------------------------------------

def _parts(case):
    """(K, columns, activation, bias) of a layer's projections."""
    qkv = case["q"] + 2 * case["kv"]
    o = (case["attn"], case["hidden"], None, False)
    if case["proj"] == "o":
        return [o]
    return [(case["hidden"], qkv, None, case["bias"]), o, (case["hidden"], 2 * case["inter"], "silu", False),
            (case["inter"], case["hidden"], None, False)]


def _activations(gen, rows, K, dtype):
    spread = torch.exp(0.5 * torch.randn(K, generator=gen, device=DEVICE))
    return (torch.randn((rows, K), generator=gen, device=DEVICE) * spread).to(dtype)


def _pow2(e):
    """2^e in 32 bits for whole e in [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x):
    """Codes' magnitudes (0 .. 7), signs and exponents of x's blocks, in 32 bits."""
    b = x.float().reshape(x.shape[:-1] + (x.shape[-1] // BLOCK, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent.to(torch.int32) - 3).clamp(-126, 127)
    q = b * _pow2(-e)
    a = q.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8)
            + (a >= 1.75).to(torch.uint8) + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8)
            + (a > 5.0).to(torch.uint8))
    return code, q < 0, e


def _values(code):
    """0, 0.5, 1, 1.5, 2, 3, 4, 6 of a magnitude's code."""
    c = code.float()
    return torch.where(c < 4, 0.5 * c, torch.where(c < 6, c - 2.0, 2.0 * c - 8.0))


def _weight(gen, shape):
    """(codes [.., K / 2], exponent bytes [.., K / 32]) of a weight [.., K], made in runs of rows."""
    K, rows = shape[-1], math.prod(shape[:-1])
    codes = torch.empty((rows, K // 2), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((rows, K // BLOCK), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 26) // K)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        code, neg, e = _blocks(torch.randn((n, K), generator=gen, device=DEVICE) / math.sqrt(K))
        code = (code | (neg.to(torch.uint8) << 3)).reshape(n, K // 2, 2)
        codes[r:r + n] = code[..., 0] | (code[..., 1] << 4)
        scales[r:r + n] = (e[..., 0] + 127).to(torch.uint8)
    return codes.reshape(shape[:-1] + (K // 2,)), scales.reshape(shape[:-1] + (K // BLOCK,))


def _held(codes, scales):
    """The weight as a program keeps it: laid out once for the framework's products, or as a checkpoint holds it."""
    if not own:
        return codes, scales
    from sglite_amd import ops

    return ops.mx4_repack(ops.Mx4(codes, scales))


def _inputs(case, seed, held):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, M, layers = DTYPES[case["dtype"]], case["M"], []
    if case["kind"] == "quantize":
        return [{"x": _activations(gen, M, case["K"], dt)}]
    if case["kind"] == "linear":
        for _ in range(case["layers"]):
            for K, N, act, biased in _parts(case):
                bias = torch.randn(N, generator=gen, device=DEVICE).to(dt) if biased else None
                layers.append({"x": _activations(gen, M, K, dt), "w": held(*_weight(gen, (N, K))), "act": act,
                               "bias": bias})
        return layers
    E, k, H, I = case["E"], case["top_k"], case["hidden"], case["inter"]
    prefer = case["skew"] * torch.randn(E, generator=gen, device=DEVICE)
    for _ in range(case["layers"]):
        logits = torch.randn((M, E), generator=gen, device=DEVICE) + prefer
        top = torch.topk(torch.softmax(logits, -1), k, -1)
        layers.append({"x": _activations(gen, M, H, dt), "h": _activations(gen, M * k, I, dt),
                       "w1": held(*_weight(gen, (E, 2 * I, H))), "w2": held(*_weight(gen, (E, H, I))),
                       "ids": top.indices.to(torch.int32), "weights": top.values / top.values.sum(-1, keepdim=True)})
    return layers


def prepare(case, seed):
    state = {"kind": case["kind"], "top_k": case.get("top_k"), "graph": None, "layers": _inputs(case, seed, _held)}
    if case["kind"] != "quantize" and case["M"] <= GRAPH_MAX and case.get("proj") != "o":
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _step(state)
        torch.cuda.current_stream().wait_stream(stream)
        state["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(state["graph"]):
            state["out"] = _step(state)
    return state


# ---------------------------------------------------------------------------
# The program.
# ---------------------------------------------------------------------------

def _silu_and_mul(v):
    g, u = v.chunk(2, -1)
    return g / (1.0 + torch.exp(-g)) * u


def _plain_quantized(x):
    """The values that x's blocks hold, in 32 bits."""
    code, neg, e = _blocks(x)
    v = _values(code) * _pow2(e)
    return torch.where(neg, -v, v).reshape(x.shape)


def _plain_weight(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(scales.shape + (BLOCK,))
    v = _values(c & 7) * _pow2(scales.to(torch.int32)[..., None] - 127)
    return torch.where(c >= 8, -v, v).reshape(scales.shape[:-1] + (-1,))


def _plain_linear(p):
    y = _plain_quantized(p["x"]) @ _plain_weight(*p["w"]).t()
    if p["bias"] is not None:
        y = y + p["bias"].float()
    return (y if p["act"] is None else _silu_and_mul(y)).to(p["x"].dtype)


def _plain_product(a, w, ids, top_k, weights, act):
    """Routed row r (token r // top_k of `a`) by its expert's weight, the rows sorted and cut into blocks of one
    expert's rows, in 32 bits."""
    w = _plain_weight(*w)
    E, N, K = w.shape
    dev, n, dt = a.device, ids.numel(), a.dtype
    step = 64
    a = _plain_quantized(a)
    ids = ids.reshape(-1).long()
    order = torch.argsort(ids, stable=True)
    experts = torch.arange(E, device=dev)
    start = torch.searchsorted(ids[order], experts)
    count = torch.searchsorted(ids[order], experts, right=True) - start
    last = torch.cumsum((count + step - 1) // step, 0)
    block = torch.arange(min(n, n // step + E), device=dev)
    e = torch.searchsorted(last, block, right=True).clamp(max=E - 1)
    nth = block - (last[e] - (count[e] + step - 1) // step)
    row = nth[:, None] * step + torch.arange(step, device=dev)
    here = (row < count[e][:, None]) & (block < last[-1])[:, None]
    row = order[torch.where(here, start[e][:, None] + row, torch.zeros_like(row))]
    y = torch.bmm(a[row // top_k], w[e].transpose(1, 2).contiguous())
    y = y * weights.reshape(-1)[row][:, :, None] if weights is not None else y
    y = y if act is None else _silu_and_mul(y)
    # Rows of no block land in the row behind the last one.
    out = torch.empty((n + 1, y.shape[-1]), dtype=dt, device=dev)
    out[torch.where(here, row, torch.full_like(row, n))] = y.to(dt)
    return out[:n]


def _own_step(state):
    from sglite_amd import ops

    if state["kind"] == "quantize":
        return [ops.mx4_dequantize(ops.mx4_quantize(p["x"]), p["x"].dtype) for p in state["layers"]]
    if state["kind"] == "linear":
        return [ops.mx4_gemm(p["x"], p["w"], bias=p["bias"], activation=p["act"]) for p in state["layers"]]
    out, k = [], state["top_k"]
    for p in state["layers"]:
        rows = p["ids"].numel()
        align = ops.moe_align_block_size(p["ids"], 16, p["w1"].num_experts)
        out.append([ops.mx4_moe_gemm(p["x"], p["w1"], align, None, rows, k, activation="silu"),
                    ops.mx4_moe_gemm(p["h"], p["w2"], align, p["weights"], rows, 1, mul_routed_weight=True)])
    return out


def _step(state):
    if own:
        return _own_step(state)
    if state["kind"] == "quantize":
        return [_plain_quantized(p["x"]).to(p["x"].dtype) for p in state["layers"]]
    if state["kind"] == "linear":
        return [_plain_linear(p) for p in state["layers"]]
    k = state["top_k"]
    return [[_plain_product(p["x"], p["w1"], p["ids"], k, None, "silu"),
             _plain_product(p["h"], p["w2"], p["ids"], 1, p["weights"], None)] for p in state["layers"]]


def run(state):
    if state["graph"] is None:
        return _step(state)
    state["graph"].replay()
    return state["out"]


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what its results are.
# ---------------------------------------------------------------------------

# Bytes of a quantised value: half a byte and its share of the block's exponent.
HELD = 0.5 + 1.0 / BLOCK


def work(case):
    M = case["M"]
    if case["kind"] == "quantize":
        # x in, what it is quantised to, and that read back as values.
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": M * case["K"] * (2.0 * size + HELD), "flops": 2.0 * M * case["K"]}
    if case["kind"] == "linear":
        b = f = 0.0
        for K, N, act, biased in _parts(case):
            b += HELD * K * N + 2.0 * M * (K + (N // 2 if act else N)) + (2.0 * N if biased else 0.0)
            f += 2.0 * M * K * N
    else:
        E, k, H, I = case["E"], case["top_k"], case["hidden"], case["inter"]
        # Expected number of experts that M tokens of k distinct, equally
        # likely experts reach.
        touched = E * (1.0 - (1.0 - k / E) ** M)
        b = touched * 3.0 * H * I * HELD + 2.0 * M * (H + k * (I + I + H)) + 8.0 * M * k
        f = 2.0 * M * k * 3 * H * I
    return {"bytes": b * case["layers"], "flops": f * case["layers"]}


def _quantized64(x):
    """Q(x) in 64 bits: the step between neighbours is 1/2 below 2, 1 below 4, then 2, times the block's 2^e."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for r in range(0, x.shape[0], 2048):
        b = x[r:r + 2048].double().unflatten(-1, (-1, BLOCK))
        top = b.abs().max(dim=-1, keepdim=True).values
        # floor(log2): the exponent bits of the largest magnitude.
        e = ((top.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127)
        unit = ((e + 1023) << 52).view(torch.float64)
        a = b / unit
        step = 0.5 + 0.5 * (a.abs() >= 2).double() + (a.abs() >= 4).double()
        out[r:r + 2048] = (torch.round(a / step) * step).clamp(-6, 6).mul_(unit).flatten(-2)
    return out


def _weight64(codes, scales):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
    table = torch.cat((table, -table))
    v = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device=codes.device)
    v[..., 0::2] = table[(codes % 16).long()]
    v[..., 1::2] = table[(codes // 16).long()]
    unit = ((scales.long() - 127 + 1023) << 52).view(torch.float64)
    return v * unit.repeat_interleave(BLOCK, -1)


def _gated64(y):
    half = y.shape[-1] // 2
    return y[..., :half] * torch.sigmoid(y[..., :half]) * y[..., half:]


def _experts64(p, k):
    flat = p["ids"].reshape(-1).long()
    x, h = _quantized64(p["x"]), _quantized64(p["h"])
    up = torch.empty((flat.numel(), h.shape[1]), dtype=torch.float64, device=DEVICE)
    down = torch.empty((flat.numel(), x.shape[1]), dtype=torch.float64, device=DEVICE)
    for e in range(p["w1"][0].shape[0]):
        rows = torch.nonzero(flat == e).reshape(-1)
        if rows.numel():
            up[rows] = _gated64(x[rows // k] @ _weight64(p["w1"][0][e], p["w1"][1][e]).t())
            down[rows] = (h[rows] @ _weight64(p["w2"][0][e], p["w2"][1][e]).t()) * p["weights"].reshape(-1)[rows, None]
    return [up, down]


def exact(case, seed):
    layers = _inputs(case, seed, lambda codes, scales: (codes, scales))
    if case["kind"] == "quantize":
        return [_quantized64(p["x"]) for p in layers]
    if case["kind"] == "experts":
        return [_experts64(p, case["top_k"]) for p in layers]
    out = []
    for p in layers:
        y = _quantized64(p["x"]) @ _weight64(*p["w"]).t()
        if p["bias"] is not None:
            y = y + p["bias"].double()
        out.append(y if p["act"] is None else _gated64(y))
    return out
