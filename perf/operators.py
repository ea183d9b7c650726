"""Performance cases of the products whose weight is chosen row by row.

Two kinds of work, each called as a serving program calls it:

  adapters  low-rank adapters of many requests beside the shared projections of
            decoder layers (fused qkv, o, gated gate/up, down): every row names
            its adapter or none, and its projection's output y becomes
            y + scaling * B (A x), for the gate/up projection followed by
            silu(gate) * up
  experts   the two products of a block of dense (fp16 or bf16) experts: gate/up
            with silu(gate) * up over the tokens' routed rows, and down times
            the routed weight

Up to GRAPH_MAX rows a step is captured in one graph, as a serving program
captures its decode step, over a stack of layers whose weights are larger than
the Infinity Cache; longer inputs run eagerly, and so does the smallest call.

Inputs: activations and projection outputs N(0, 1); A's rows of unit length in
the mean and B's such that an adapter adds about a third of the output's
spread; expert weights N(0, 1 / K); expert choices the top of N(0, 1) logits,
where a case says so shifted by a preference for some experts.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# Largest batch that a serving program captures; longer inputs run eagerly.
GRAPH_MAX = 160


def _adapters(name, dims, M, layers, slots, rank, dtype="fp16", mixed=False, idle=0.0, proj="layer"):
    hidden, q, kv, attn, inter = dims
    return {"name": name, "kind": "adapters", "proj": proj, "hidden": hidden, "q": q, "kv": kv, "attn": attn,
            "inter": inter, "M": M, "layers": layers, "slots": slots, "rank": rank, "dtype": dtype, "mixed": mixed,
            "idle": idle}


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
        # One adapter on one o projection for one token, called eagerly.
        _adapters("adapter_o_m1", QWEN3_4B, 1, 1, 4, 16, proj="o"),
        # Decode of a single sequence with its adapter.
        _adapters("adapters_4b_m1", QWEN3_4B, 1, 8, 8, 16),
        # A decode batch, many adapters of different ranks, some rows with none.
        _adapters("adapters_4b_m32_bf16", QWEN3_4B, 32, 8, 16, 32, dtype="bf16", mixed=True, idle=0.25),
        # A large captured decode batch over adapters of a high rank.
        _adapters("adapters_8b_m128", LLAMA3_8B, 128, 4, 32, 64),
        # The ragged last chunk of a few prompts.
        _adapters("adapters_4b_m333", QWEN3_4B, 333, 1, 8, 8, mixed=True),
        # The largest prefill chunk the scheduler forms: several prompts.
        _adapters("adapters_8b_m8192_bf16", LLAMA3_8B, 8192, 1, 8, 64, dtype="bf16", idle=0.1),
        # Qwen3-30B-A3B-shaped experts: one token, a decode batch, a short
        # chunk and a long one.
        _experts("experts_t1", 128, 8, 2048, 768, 1, 4),
        _experts("experts_t24_bf16", 128, 8, 2048, 768, 24, 2, dtype="bf16"),
        _experts("experts_t512", 128, 8, 2048, 768, 512, 1),
        _experts("experts_t4096_bf16", 128, 8, 2048, 768, 4096, 1, dtype="bf16"),
        # Few wide experts of an odd width and an uneven load, an odd chunk.
        _experts("experts_wide_t777", 16, 2, 4096, 1408, 777, 1, skew=1.0),
        # Long chunk over few experts: the products are large.
        _experts("experts_wide_t4001_bf16", 16, 4, 4096, 1408, 4001, 1, dtype="bf16", skew=0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    dtype = rng.choice(("fp16", "bf16"))
    if rng.random() < 0.5:
        dims = rng.choice(DIMS)
        rank = rng.choice((8, 16, 24, 32, 64))
        M = _log_int(rng, 1, 8192)
        slots = _log_int(rng, 1, 32 if M <= 1024 else 8)
        proj = "o" if rng.random() < 0.15 else "layer"
        layers = rng.choice((2, 3, 4)) if M <= GRAPH_MAX and proj == "layer" else 1
        c = _adapters("", dims, M, layers, slots, rank, dtype, rng.random() < 0.5, rng.choice((0.0, 0.1, 0.25)), proj)
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
    """(rows of x, columns of each part, activation) of a layer's projections."""
    o = (case["attn"], (case["hidden"],), None)
    if case["proj"] == "o":
        return [o]
    return [(case["hidden"], (case["q"], case["kv"], case["kv"]), None), o,
            (case["hidden"], (case["inter"], case["inter"]), "silu"), (case["inter"], (case["hidden"],), None)]


def _ranks(case):
    """Every second adapter of a mixed stack has about half the rank."""
    r = case["rank"]
    return [r // 2 + 1 if case["mixed"] and s % 2 else r for s in range(case["slots"])]


def _normal(gen, shape, dtype, scale=1.0):
    t = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32 if scale != 1.0 else dtype)
    return t if scale == 1.0 else (t * scale).to(dtype)


def _adapter_ids(case, gen):
    """Row's adapter, -1 for none: a decode batch's rows each their own, a prefill's sequence by sequence."""
    M, slots = case["M"], case["slots"]
    rows = M if M <= GRAPH_MAX else max(2, M // 700)
    ids = torch.randint(0, slots, (rows,), generator=gen, device=DEVICE, dtype=torch.int32)
    ids[torch.rand(rows, generator=gen, device=DEVICE) < case["idle"]] = -1
    if rows != M:
        ends = torch.sort(torch.randint(1, M, (rows - 1,), generator=gen, device=DEVICE)).values
        ids = ids[torch.searchsorted(ends, torch.arange(M, device=DEVICE), right=True)]
    return ids


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, M = DTYPES[case["dtype"]], case["M"]
    state = {"kind": case["kind"], "graph": None, "layers": []}
    if case["kind"] == "adapters":
        S, R = case["slots"], case["rank"]
        state["ids"] = _adapter_ids(case, gen)
        state["slots"], state["rank"] = S, R
        state["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32, device=DEVICE)
        for _ in range(case["layers"]):
            for K, cols, act in _parts(case):
                N = sum(cols)
                below = torch.arange(R, device=DEVICE) < state["ranks"][:, None]
                a = _normal(gen, (S, len(cols), R, K), dt, 1.0 / math.sqrt(K)) * below[:, None, :, None]
                b = _normal(gen, (S, N, R), dt, 0.3 / math.sqrt(R)) * below[:, None, :]
                # alpha / rank of common adapters
                scaling = torch.tensor([0.5, 1.0, 2.0], device=DEVICE)[
                    torch.randint(0, 3, (S,), generator=gen, device=DEVICE)]
                state["layers"].append({"x": _normal(gen, (M, K), dt), "y": _normal(gen, (M, N), dt),
                                        "a": a.reshape(S, len(cols) * R, K), "b": b, "scaling": scaling, "cols": cols,
                                        "act": act})
    else:
        E, k, H, I = case["E"], case["top_k"], case["hidden"], case["inter"]
        state["top_k"] = k
        bias = case["skew"] * torch.randn(E, generator=gen, device=DEVICE)
        for _ in range(case["layers"]):
            logits = torch.randn((M, E), generator=gen, device=DEVICE) + bias
            top = torch.topk(torch.softmax(logits, -1), k, -1)
            state["layers"].append({"x": _normal(gen, (M, H), dt), "h": _normal(gen, (M * k, I), dt),
                                    "w1": _normal(gen, (E, 2 * I, H), dt, 1.0 / math.sqrt(H)),
                                    "w2": _normal(gen, (E, H, I), dt, 1.0 / math.sqrt(I)),
                                    "ids": top.indices.to(torch.int32),
                                    "weights": top.values / top.values.sum(-1, keepdim=True)})
    if M <= GRAPH_MAX and case.get("proj") != "o":
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


def _plain_adapters(state, p):
    """Every row by every adapter of the stack, the others' products zeroed, in 32 bits."""
    S, R, P = state["slots"], state["rank"], len(p["cols"])
    M, K = p["x"].shape
    N = p["y"].shape[1]
    dev = p["x"].device
    mine = state["ids"][:, None] == torch.arange(S, device=dev)
    v = (p["x"].float() @ p["a"].float().reshape(S * P * R, K).t()).view(M, S, P, R)
    live = mine[:, :, None, None] & (torch.arange(R, device=dev) < state["ranks"][:, None])[None, :, None, :]
    v = torch.where(live, v * p["scaling"][:, None, None], torch.zeros_like(v))
    part = torch.cat([torch.full((n,), i, device=dev) for i, n in enumerate(p["cols"])])
    b = p["b"].float().permute(0, 2, 1)[:, None] * (part == torch.arange(P, device=dev)[:, None])[None, :, None, :]
    out = p["y"].float() + v.reshape(M, S * P * R) @ b.reshape(S * P * R, N)
    return (out if p["act"] is None else _silu_and_mul(out)).to(p["y"].dtype)


def _plain_product(a, w, ids, top_k, weights, act):
    """Routed row r (token r // top_k of `a`) by its expert's weight, the rows sorted and cut into blocks of one
    expert's rows, in 32 bits."""
    E, N, K = w.shape
    dev, n = a.device, ids.numel()
    step = 64
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
    y = torch.bmm(a.float()[row // top_k], w.float()[e].transpose(1, 2).contiguous())
    y = y * weights.reshape(-1)[row][:, :, None] if weights is not None else y
    y = y if act is None else _silu_and_mul(y)
    # Rows of no block land in the row behind the last one.
    out = torch.empty((n + 1, y.shape[-1]), dtype=a.dtype, device=dev)
    out[torch.where(here, row, torch.full_like(row, n))] = y.to(a.dtype)
    return out[:n]


def _own_adapters(state):
    from sglite_amd import ops

    batch = ops.lora_route(state["ids"], state["slots"])
    return [ops.lora_add(p["y"], p["x"], ops.LoraStack(p["a"], p["b"], p["scaling"], state["ranks"], p["cols"]), batch,
                         activation=p["act"]) for p in state["layers"]]


def _own_experts(p, k):
    from sglite_amd import ops

    rows, E = p["ids"].numel(), p["w1"].shape[0]
    align = ops.moe_align_block_size(p["ids"], 16, E)
    return [ops.moe_dense_gemm(p["x"], p["w1"], align, None, rows, k, activation="silu"),
            ops.moe_dense_gemm(p["h"], p["w2"], align, p["weights"], rows, 1, mul_routed_weight=True)]


def _step(state):
    if state["kind"] == "adapters":
        return _own_adapters(state) if own else [_plain_adapters(state, p) for p in state["layers"]]
    k = state["top_k"]
    if own:
        return [_own_experts(p, k) for p in state["layers"]]
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

def work(case):
    M = case["M"]
    if case["kind"] == "adapters":
        S = case["slots"]
        rows = M * (1.0 - case["idle"])
        seqs = rows if M <= GRAPH_MAX else max(2, M // 700) * (1.0 - case["idle"])
        # Adapters that the batch's sequences reach, each named equally often.
        touched = S * (1.0 - (1.0 - 1.0 / S) ** seqs)
        rank = sum(_ranks(case)) / S
        b = f = 0.0
        for K, cols, act in _parts(case):
            N = sum(cols)
            b += 2.0 * touched * rank * (len(cols) * K + N)
            b += 2.0 * (rows * K + M * N + M * (N // 2 if act else N)) + 4.0 * M
            f += 2.0 * rows * rank * (len(cols) * K + N)
    else:
        E, k, H, I = case["E"], case["top_k"], case["hidden"], case["inter"]
        # Expected number of experts that M tokens of k distinct, equally
        # likely experts reach.
        touched = E * (1.0 - (1.0 - k / E) ** M)
        b = touched * 3.0 * H * I * 2 + 2.0 * M * (H + k * (I + I + H)) + 8.0 * M * k
        f = 2.0 * M * k * 3 * H * I
    return {"bytes": b * case["layers"], "flops": f * case["layers"]}


def _adapters64(state, p):
    """y + scaling * B A x of each row's adapter, adapter by adapter and part by part."""
    y = p["y"].double()
    P, R = len(p["cols"]), state["rank"]
    for s, r in enumerate(state["ranks"].tolist()):
        rows = torch.nonzero(state["ids"] == s).reshape(-1)
        if not rows.numel():
            continue
        x, c0 = p["x"][rows].double(), 0
        for i in range(P):
            A = p["a"][s, i * R:i * R + r].double()
            B = p["b"][s, c0:c0 + p["cols"][i], :r].double()
            y[rows, c0:c0 + p["cols"][i]] += (x @ A.t()) @ B.t() * p["scaling"][s].double()
            c0 += p["cols"][i]
    if p["act"] is None:
        return y
    half = y.shape[1] // 2
    return y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]


def _experts64(p, k):
    flat = p["ids"].reshape(-1).long()
    I, H = p["h"].shape[1], p["x"].shape[1]
    up = torch.empty((flat.numel(), I), dtype=torch.float64, device=DEVICE)
    down = torch.empty((flat.numel(), H), dtype=torch.float64, device=DEVICE)
    for e in range(p["w1"].shape[0]):
        rows = torch.nonzero(flat == e).reshape(-1)
        if rows.numel():
            gu = p["x"][rows // k].double() @ p["w1"][e].double().t()
            up[rows] = gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:]
            down[rows] = (p["h"][rows].double() @ p["w2"][e].double().t()) * p["weights"].reshape(-1)[rows, None].double()
    return [up, down]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "adapters":
        return [_adapters64(state, p) for p in state["layers"]]
    return [_experts64(p, state["top_k"]) for p in state["layers"]]
