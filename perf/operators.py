"""What the speed of the projections in 8 bits and of the adapters beside them is measured on: single operators, at the layer sizes of
``bench.py`` (hidden 4,096 and 5,120, intermediate 12,288, one product for queries, keys and values of 6,144 outputs).

``kind`` names the operator:

``norm``      the residual's addition, the root-mean-square norm and its rows in 8 bits (e4m3) with a scale a row;
``silu_mul``  silu(gate) * up, its rows in 8 bits;
``quantise``  rows in 8 bits as they are (what an attention hands to its output projection);
``product``   the product of rows in 8 bits with a weight in 8 bits, a scale a row on either side;
``adapters``  the low-rank adapters of many requests, added to what the shared projection made of the same rows.

A row in 8 bits stands for its numbers times the row's scale, the largest magnitude of the row over 448 (the largest number of e4m3).
"""
import math

import torch

own = False

EPS = 1e-6
TOP = 448.0                # the largest number of e4m3
LEAST = 2.0 ** -126        # a scale is at least this, so that a row of zeros has one
F32, F64, BF16, E4M3 = torch.float32, torch.float64, torch.bfloat16, torch.float8_e4m3fn


def listed():
    return [
        # a server's decode step of eight requests in front of every projection: latency is the time
        {"name": "norm decode 8", "kind": "norm", "tokens": 8, "hidden": 4096, "stream": "bfloat16", "keep": False},
        # the prompts of a long step: the memory's rate is the time
        {"name": "norm prompt 8192", "kind": "norm", "tokens": 8192, "hidden": 4096, "stream": "bfloat16", "keep": False},
        # the feed-forward's middle in a decode step, and in a prompt with gate and up interleaved as the fused products want them
        {"name": "silu_mul decode 16", "kind": "silu_mul", "tokens": 16, "inner": 12288, "block": 0},
        {"name": "silu_mul prompt 4096", "kind": "silu_mul", "tokens": 4096, "inner": 12288, "block": 128},
        # an attention's output ahead of its projection: a large decode batch, and a ragged prompt held in 32 bits
        {"name": "quantise decode 64", "kind": "quantise", "tokens": 64, "width": 4096, "dtype": "bfloat16"},
        {"name": "quantise prompt 3001 float32", "kind": "quantise", "tokens": 3001, "width": 5120, "dtype": "float32"},
        # a decode step's gate and up projection (the weight's bytes are the time), a portion of a prompt beside decoding requests, a
        # long prompt's down projection
        {"name": "product decode 8", "kind": "product", "rows": 8, "outputs": 24576, "inputs": 4096, "out": "bfloat16"},
        {"name": "product portion 333", "kind": "product", "rows": 333, "outputs": 6144, "inputs": 4096, "out": "bfloat16"},
        {"name": "product prompt 4096", "kind": "product", "rows": 4096, "outputs": 4096, "inputs": 12288, "out": "bfloat16"},
        # one user with an adapter; 64 decoding requests over 32 adapters of different ranks beside the queries', keys' and values'
        # product; a step of five prompts beside the gate and up product
        {"name": "adapter decode 1", "kind": "adapters", "requests": 1, "tokens": 1, "slots": 4, "rank": 16, "inputs": 4096,
         "widths": "4096", "ragged": False, "bare": 0, "out": "bfloat16"},
        {"name": "adapters decode 64", "kind": "adapters", "requests": 64, "tokens": 64, "slots": 32, "rank": 64, "inputs": 4096,
         "widths": "4096,1024,1024", "ragged": True, "bare": 9, "out": "bfloat16"},
        {"name": "adapters prompts 4001", "kind": "adapters", "requests": 5, "tokens": 4001, "slots": 8, "rank": 32, "inputs": 4096,
         "widths": "12288,12288", "ragged": False, "bare": 0, "out": "bfloat16"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("norm", "silu_mul", "quantise", "product", "product", "adapters", "adapters"))
    if kind == "norm":
        hidden = _spread(rng, 64, 8192)
        hidden = hidden if rng.random() < 0.2 else -(-hidden // 16) * 16          # odd sizes among the aligned ones
        return {"kind": kind, "tokens": _spread(rng, 1, min(8192, 33554432 // hidden)), "hidden": hidden,
                "stream": rng.choice(("bfloat16", "bfloat16", "float32")), "keep": rng.random() < 0.3}
    if kind == "silu_mul":
        inner = -(-_spread(rng, 128, 25600) // 16) * 16
        block = rng.choice((0, 128))
        inner = -(-inner // 128) * 128 if block else inner
        return {"kind": kind, "tokens": _spread(rng, 1, min(8192, 50331648 // inner)), "inner": inner, "block": block}
    if kind == "quantise":
        width = _spread(rng, 64, 12288)
        width = width if rng.random() < 0.2 else -(-width // 16) * 16
        dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
        return {"kind": kind, "tokens": _spread(rng, 1, min(8192, (30720000 if dtype == "bfloat16" else 15360000) // width)), "width": width, "dtype": dtype}
    if kind == "product":
        inputs = -(-_spread(rng, 128, 16384) // 16) * 16
        outputs = min(_spread(rng, 100, 32768), 201326592 // inputs)
        rows = _spread(rng, 1, min(4096, 206158430208 // (inputs * outputs)))
        return {"kind": kind, "rows": max(1, rows), "outputs": outputs, "inputs": inputs, "out": rng.choice(("bfloat16", "bfloat16", "float32"))}
    requests = _spread(rng, 1, 64)
    inputs = -(-_spread(rng, 256, 8192) // 8) * 8
    widths = [-(-_spread(rng, 64, 8192) // 8) * 8 for _ in range(rng.choice((1, 1, 2, 3)))]
    tokens = requests if rng.random() < 0.5 else max(requests, _spread(rng, requests, max(requests, min(4096, 65000000 // (sum(widths) + inputs)))))
    return {"kind": kind, "requests": requests, "tokens": tokens, "slots": _spread(rng, 1, 32), "rank": 8 * _spread(rng, 1, 8), "inputs": inputs,
            "widths": ",".join(map(str, widths)), "ragged": rng.random() < 0.5, "bare": rng.choice((0, 0, 3, 9)),
            "out": rng.choice(("bfloat16", "bfloat16", "float32"))}


# ---------------------------------------------------------------------------------------------------- what a case's requests are
def _requests(case):
    """(tokens of each request, its adapter or -1, the adapters' ranks): a request in ``bare`` has none, ranks differ where ``ragged``."""
    n, tokens, slots, rank = case["requests"], case["tokens"], case["slots"], case["rank"]
    shares = [i * 3 % 7 + 1 for i in range(n)]
    counts = [1 + (tokens - n) * s // sum(shares) for s in shares]
    counts[-1] += tokens - sum(counts)
    of = [-1 if case["bare"] and i % case["bare"] == case["bare"] - 1 else i * 5 % slots for i in range(n)]
    ranks = [rank if not case["ragged"] or s % 3 == 0 else max(1, rank // (s % 3 + 1)) for s in range(slots)]
    return counts, of, ranks


def _widths(case):
    return tuple(int(w) for w in case["widths"].split(","))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def randn(*shape, dtype=F32):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)

    def weight(n):
        return (1.0 + 0.1 * randn(n)).to(BF16)

    def loud(n):    # a few channels of a hidden state are many times as large as the others
        return 1.0 + 20.0 * (torch.rand(n, device="cuda", generator=g) < 0.005).float()

    def codes(rows, cols, by):
        v = randn(rows, cols) * by
        scale = (v.abs().amax(1) / TOP).clamp_min(LEAST)
        return (v / scale[:, None]).clamp(-TOP, TOP).to(E4M3), scale

    state = {"kind": kind, "case": case}
    if kind == "norm":
        T, H = case["tokens"], case["hidden"]
        stream = getattr(torch, case["stream"])
        state |= {"x": randn(T, H).to(BF16), "residual": (2.0 * randn(T, H) * loud(H)).to(stream), "w": weight(H)}
    elif kind == "silu_mul":
        state["x"] = (1.5 * randn(case["tokens"], 2 * case["inner"])).to(BF16)
    elif kind == "quantise":
        state["x"] = (randn(case["tokens"], case["width"]) * loud(case["width"])).to(getattr(torch, case["dtype"]))
    elif kind == "product":
        state["q"], state["q_scale"] = codes(case["rows"], case["inputs"], loud(case["inputs"]))
        state["w"], state["w_scale"] = codes(case["outputs"], case["inputs"], 0.02)
    else:
        counts, of, ranks = _requests(case)
        widths, S, R, K, T = _widths(case), case["slots"], case["rank"], case["inputs"], case["tokens"]
        live = torch.arange(R, device="cuda") < torch.tensor(ranks, device="cuda")[:, None]        # [S, R]
        state |= {"y": randn(T, sum(widths)).to(getattr(torch, case["out"])), "x": randn(T, K).to(BF16),
                  "a": (randn(S, len(widths), R, K) / math.sqrt(K) * live[:, None, :, None]).to(BF16),
                  "b": (0.3 * randn(S, sum(widths), R) * live[:, None, :]).to(BF16),
                  "scale": torch.tensor([2.0 - 0.5 * (s % 2) for s in range(S)], device="cuda"), "widths": widths,
                  "ranks": torch.tensor(ranks, dtype=torch.int32, device="cuda"),
                  "of": torch.repeat_interleave(torch.tensor(of, device="cuda"), torch.tensor(counts, device="cuda"))}
        if own:    # the lists that a server makes once a step, for the adapters of all its layers
            from roost_b200.kernels import library
            state["plan"] = library.load().adapter_plan(counts, of, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------- the plain forms
def _rows_e4m3(v):
    scale = (v.abs().amax(1) / TOP).clamp_min(LEAST)
    return (v / scale[:, None]).clamp(-TOP, TOP).to(E4M3), scale


def run(state):
    kind = state["kind"]
    if own:
        from roost_b200.kernels import library
        lib = library.load()
        if kind == "norm":
            out = lib.add_rms_norm_e4m3(state["x"], state["residual"], state["w"], EPS, keep=state["case"]["keep"])
            return (*out, state["residual"])
        if kind == "silu_mul":
            return lib.silu_mul_e4m3(state["x"], state["case"]["block"])
        if kind == "quantise":
            return lib.quantise_e4m3(state["x"])
        if kind == "product":
            return lib.gemm_e4m3(state["q"], state["q_scale"], state["w"], state["w_scale"], getattr(torch, state["case"]["out"]))
        return lib.adapters_add_(state["y"], state["x"], state["a"], state["b"], state["scale"], state["plan"], widths=state["widths"], ranks=state["ranks"])
    if kind == "norm":
        state["residual"].copy_(state["x"].float() + state["residual"].float())
        r = state["residual"].float()
        v = r / torch.sqrt((r * r).mean(1, keepdim=True) + EPS) * state["w"].float()
        kept = (v.to(BF16),) if state["case"]["keep"] else ()
        return (*_rows_e4m3(v), *kept, state["residual"])
    if kind == "silu_mul":
        inner, block = state["case"]["inner"], state["case"]["block"] or state["case"]["inner"]
        x = state["x"].float().reshape(-1, inner // block, 2, block)
        gate, up = x[:, :, 0].reshape(-1, inner), x[:, :, 1].reshape(-1, inner)
        return _rows_e4m3(gate / (1.0 + torch.exp(-gate)) * up)
    if kind == "quantise":
        return _rows_e4m3(state["x"].float())
    if kind == "product":
        y = state["q"].float() @ state["w"].float().t() * state["q_scale"][:, None] * state["w_scale"]
        return y.to(getattr(torch, state["case"]["out"]))
    # every row against every adapter, and only its own kept: [T, S] of ones and zeros
    a, b, y, widths = state["a"].float(), state["b"].float(), state["y"], state["widths"]
    S, P, R, K = a.shape
    mine = (state["of"][:, None] == torch.arange(S, device=y.device)).float()
    live = (torch.arange(R, device=y.device) < state["ranks"][:, None]).float()
    h = (state["x"].float() @ a.reshape(S * P * R, K).t()).reshape(-1, S, P, R) * (mine * state["scale"])[:, :, None, None] * live[:, None]
    parts = torch.split(b, widths, dim=1)
    delta = torch.cat([h[:, :, p].reshape(-1, S * R) @ w.transpose(1, 2).reshape(S * R, -1) for p, w in enumerate(parts)], 1)
    return y.copy_(y.float() + delta)


# ---------------------------------------------------------------------------------------------------- the floor
def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, size = case["tokens"] * case["hidden"], 4 if case["stream"] == "float32" else 2
        return {"bytes": n * (2 + 2 * size + 1 + (2 if case["keep"] else 0)) + 2 * case["hidden"] + 4 * case["tokens"], "flops": 7 * n}
    if kind == "silu_mul":
        n = case["tokens"] * case["inner"]
        return {"bytes": n * 5 + 4 * case["tokens"], "flops": 7 * n}
    if kind == "quantise":
        n = case["tokens"] * case["width"]
        return {"bytes": n * (5 if case["dtype"] == "float32" else 3) + 4 * case["tokens"], "flops": 3 * n}
    if kind == "product":
        m, n, k = case["rows"], case["outputs"], case["inputs"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * (4 if case["out"] == "float32" else 2), "flops": 2 * m * n * k}
    counts, of, ranks = _requests(case)
    widths, K = _widths(case), case["inputs"]
    P, N, size = len(widths), sum(widths), 4 if case["out"] == "float32" else 2
    rows = sum(c for c, s in zip(counts, of) if s >= 0)
    numbers = sum(ranks[s] * (P * K + N) for s in set(of) if s >= 0)
    flops = sum(2 * c * ranks[s] * (P * K + N) for c, s in zip(counts, of) if s >= 0)
    return {"bytes": rows * (2 * K + 2 * size * N) + 2 * numbers, "flops": flops}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _nearest_e4m3(v):
    """The nearest numbers of e4m3, ties to the even one: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_rows(v):
    scale = torch.maximum(v.abs().amax(1) / TOP, torch.tensor(LEAST, dtype=F64, device=v.device))
    return _nearest_e4m3(v / scale[:, None]), scale


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        total = s["x"].to(F64) + s["residual"].to(F64)
        r = total.to(F32).to(s["residual"].dtype).to(F64)        # what is normed is the stream as it is stored
        v = r * torch.rsqrt(r.square().sum(1, keepdim=True) / case["hidden"] + EPS) * s["w"].to(F64)
        q, scale = _exact_rows(v)
        return [q, scale, v, total] if case["keep"] else [q, scale, total]
    if kind == "silu_mul":
        x, block = s["x"].to(F64), case["block"]
        at = torch.arange(case["inner"], device="cuda")
        gate_at = at // block * 2 * block + at % block if block else at
        gate, up = x[:, gate_at], x[:, gate_at + (block or case["inner"])]
        return list(_exact_rows(gate * torch.sigmoid(gate) * up))
    if kind == "quantise":
        return list(_exact_rows(s["x"].to(F64)))
    if kind == "product":
        rows = s["q"].to(F64) * s["q_scale"].to(F64)[:, None]
        return torch.matmul(rows, (s["w"].to(F64) * s["w_scale"].to(F64)[:, None]).t())
    counts, of, ranks = _requests(case)
    y, start = s["y"].to(F64), 0
    for count, slot in zip(counts, of):
        if slot >= 0:
            x, rank, column = s["x"][start:start + count].to(F64), ranks[slot], 0
            for p, width in enumerate(s["widths"]):
                down = torch.einsum("tk,rk->tr", x, s["a"][slot, p, :rank].to(F64))
                up = torch.einsum("tr,nr->tn", down, s["b"][slot, column:column + width, :rank].to(F64))
                y[start:start + count, column:column + width] += s["scale"][slot].to(F64) * up
                column += width
        start += count
    return y
