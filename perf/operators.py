"""The operators of quantised linear layers by which their speed is judged: a residual sum and RMS norm whose result leaves in
8 bits, rows to 8 bits, the product of 8-bit rows with 8-bit weights, and the product with weights of 4 bits in groups.

8 bits are e4m3 (``torch.float8_e4m3fn``) with one float32 scale a row (a token's, or an output channel's); 4 bits are whole
numbers 0 to 15 with one bfloat16 scale and one whole zero point a group of consecutive input channels.  Sizes are those of the
Llama-3-8B layer (width 4,096, joint gate and up matrix of 28,672 rows, hidden size 14,336, joint projection of 6,144 rows)
and of this repository's kernel tests.  ``own`` false: elementary torch operations in 32 bits; true: this library's kernels.
"""
import math

import torch

own = False
EPS = 1e-5
LARGEST = 448.0  # of e4m3


# ---- cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm in front of a layer's 8-bit product in a decode step of eight requests: the smallest call, all latency
        {"name": "norm_decode_8", "op": "norm", "rows": 8, "dim": 4096, "dtype": "bf16", "gain": "bf16"},
        # the same for one prompt of the benchmark's length
        {"name": "norm_prompt_2048", "op": "norm", "rows": 2048, "dim": 4096, "dtype": "bf16", "gain": "bf16"},
        # float32 rows and gains of a width that no vector divides, as a float32-stored norm has them
        {"name": "norm_f32_odd", "op": "norm", "rows": 1100, "dim": 5001, "dtype": "f32", "gain": "f32"},
        # a feed-forward's hidden values before its second product, in a decode step of eight
        {"name": "rows_decode_8", "op": "rows", "rows": 8, "dim": 14336, "dtype": "bf16"},
        # the same for a prompt
        {"name": "rows_prompt_2048", "op": "rows", "rows": 2048, "dim": 14336, "dtype": "bf16"},
        # the joint gate and up product of a decode step of eight: every weight is read once for eight rows
        {"name": "e4m3_decode_8", "op": "e4m3", "rows": 8, "out": 28672, "dim": 4096, "bias": False},
        # the feed-forward's second product in a decode step of 64: few output rows, a long sum
        {"name": "e4m3_decode_64", "op": "e4m3", "rows": 64, "out": 4096, "dim": 14336, "bias": False},
        # the same for a prompt of 8,192 tokens: the largest call
        {"name": "e4m3_prompt_8192", "op": "e4m3", "rows": 8192, "out": 4096, "dim": 14336, "bias": False},
        # the joint gate and up product of one request's decode step: a matrix-vector product
        {"name": "int4_decode_1", "op": "int4", "rows": 1, "out": 28672, "dim": 4096, "group": 128, "zeros": True, "bias": False},
        # the feed-forward's second product in a decode step of 64, weights around a fixed zero point
        {"name": "int4_decode_64", "op": "int4", "rows": 64, "out": 4096, "dim": 14336, "group": 128, "zeros": False, "bias": False},
        # the joint projection of queries, keys and values over a prompt that no tile divides, with a bias
        {"name": "int4_prompt_1100", "op": "int4", "rows": 1100, "out": 6144, "dim": 4096, "group": 64, "zeros": True, "bias": True},
        # the joint gate and up product of a prompt of the benchmark's length
        {"name": "int4_prompt_2048", "op": "int4", "rows": 2048, "out": 28672, "dim": 4096, "group": 128, "zeros": True, "bias": False},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rows", "e4m3", "e4m3", "int4", "int4"])
    rows = _spread(rng, 1, 8192)
    if op == "norm":
        return {"op": op, "rows": rows, "dim": _spread(rng, 16, 16384), "dtype": rng.choice(["bf16", "f32"]), "gain": rng.choice(["bf16", "f32"])}
    if op == "rows":
        return {"op": op, "rows": rows, "dim": _spread(rng, 16, 28672), "dtype": rng.choice(["bf16", "f32"])}
    out, dim = _spread(rng, 16, 28672), _spread(rng, 16, 14336)
    dim = dim if op == "e4m3" and rng.random() < 0.25 else max(1, dim // 16) * 16 if op == "e4m3" else max(4, dim // 8) * 8
    rows = max(1, min(rows, (8192 * 4096 * 14336) // (out * dim)))
    case = {"op": op, "rows": rows, "out": out, "dim": dim}
    if op == "int4":
        case.update(group=rng.choice([32, 64, 128, 128, 256, 0]), zeros=rng.random() < 0.5)
    case["bias"] = rng.random() < 0.3
    return case


def work(case):
    m, k = case["rows"], case["dim"]
    size = {"bf16": 2, "f32": 4}
    if case["op"] == "norm":
        return {"bytes": m * (k * (4 + size[case["dtype"]] + 4 + 1) + 4) + k * size[case["gain"]], "flops": 6 * m * k}
    if case["op"] == "rows":
        return {"bytes": m * (k * (size[case["dtype"]] + 1) + 4), "flops": 3 * m * k}
    n = case["out"]
    if case["op"] == "e4m3":
        read = m * k + n * k + 4 * (m + n)
    else:
        groups = -(-k // (case["group"] or k))
        read = 2 * m * k + n * k // 2 + n * groups * (2 + (0.5 if case["zeros"] else 0))
    return {"bytes": read + (2 * n if case["bias"] else 0) + 2 * m * n, "flops": 2 * m * n * k}


# ---- inputs ------------------------------------------------------------------------------------------------------------
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g)


def _activations(g, rows, dim):
    """Rows as a trained network's: one channel in 64 is some eight times as large as the others."""
    x = _normal(g, rows, dim)
    x[:, ::64] *= 8.0
    return x


def _to_e4m3(x):
    most = x.abs().amax(1)
    q = (x * LARGEST / most[:, None]).clamp_(-LARGEST, LARGEST)
    return torch.where(most[:, None] > 0, q, 0.0 * x).to(torch.float8_e4m3fn), most / LARGEST


def prepare(case, seed):
    g, rows, dim = _generator(seed), case["rows"], case["dim"]
    state = {"case": case}
    if case["op"] == "norm":
        state["residual"] = 3.0 * _activations(g, rows, dim)
        state["delta"] = _normal(g, rows, dim).to(DTYPES[case["dtype"]])
        state["gain"] = (1.0 + _normal(g, dim, std=0.1)).to(DTYPES[case["gain"]])
        return state
    if case["op"] == "rows":
        state["x"] = _activations(g, rows, dim).to(DTYPES[case["dtype"]])
        return state
    out = case["out"]
    state["bias"] = _normal(g, out, std=0.1).to(torch.bfloat16) if case["bias"] else None
    if case["op"] == "e4m3":
        state["x"], state["x_scale"] = _to_e4m3(_activations(g, rows, dim))
        state["w"], state["w_scale"] = _to_e4m3(_normal(g, out, dim, std=0.02))
        if own:  # rows and weights as this library's operators hand them on
            from fms_b200.kernels import ops

            state["own_x"] = ops.QuantizedRows.of(state["x"], state["x_scale"])
            state["own_w"] = ops.e4m3_weight(state["w"], state["w_scale"])
        return state
    groups = -(-dim // (case["group"] or dim))
    state["x"] = _activations(g, rows, dim).to(torch.bfloat16)
    state["q"] = (2.7 * _normal(g, out, dim) + 8.0).round_().clamp_(0, 15).to(torch.uint8)
    state["scale"] = (0.0074 * (1.0 + 0.3 * _normal(g, out, groups)).abs() + 1e-4).to(torch.bfloat16)
    state["zero"] = (1.2 * _normal(g, out, groups) + 8.0).round_().clamp_(0, 15).to(torch.uint8) if case["zeros"] else None
    if own:  # laid out once, as a model keeps its weights
        from fms_b200.kernels import ops

        state["own_w"] = ops.pack_int4(state["q"], state["scale"], state["zero"], case["group"] or dim)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        from fms_b200.kernels import ops

        if op == "norm":
            y = ops.add_rmsnorm_quantized(state["residual"], state["delta"], state["gain"], EPS)
            return {"values": y.values[:, : y.dim], "scales": y.scales, "residual": state["residual"]}
        if op == "rows":
            y = ops.quantize_rows(state["x"])
            return {"values": y.values[:, : y.dim], "scales": y.scales}
        if op == "e4m3":
            return {"y": ops.linear_e4m3(state["own_x"], state["own_w"], state["bias"])}
        return {"y": ops.linear_int4(state["x"], state["own_w"], state["bias"])}
    if op == "norm":
        x = state["residual"]
        x += state["delta"].float()
        y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * state["gain"].float()
        values, scales = _to_e4m3(y)
        return {"values": values, "scales": scales, "residual": x}
    if op == "rows":
        values, scales = _to_e4m3(state["x"].float())
        return {"values": values, "scales": scales}
    if op == "e4m3":
        y = (state["x"].float() @ state["w"].float().t()) * state["x_scale"][:, None] * state["w_scale"][None, :]
    else:
        y = state["x"].float() @ _weights(state).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return {"y": y.to(torch.bfloat16)}


def _weights(state):
    dim, group = state["case"]["dim"], state["case"]["group"] or state["case"]["dim"]
    at = torch.arange(dim, device="cuda") // group
    zero = state["zero"].float()[:, at] if state["zero"] is not None else 8.0
    return (state["q"].float() - zero) * state["scale"].float()[:, at]


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------
def _e4m3_exactly(y):
    """Scales and the nearest e4m3 values of rows in 64 bits; ties go to the value whose last bit is 0, as ``round`` does."""
    largest = y.abs().max(dim=1).values
    v = 448 * y / largest.unsqueeze(1)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)  # 8 values from a power of two to the next
    return (torch.round(v / step) * step).clamp(-448, 448), largest / 448


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        r = state["residual"].double() + state["delta"].double()
        y = r / torch.sqrt(r.square().sum(1, keepdim=True) / case["dim"] + EPS) * state["gain"].double()
        values, scales = _e4m3_exactly(y)
        return {"values": values, "scales": scales, "residual": r}
    if case["op"] == "rows":
        values, scales = _e4m3_exactly(state["x"].double())
        return {"values": values, "scales": scales}
    if case["op"] == "e4m3":
        x = state["x"].double() * state["x_scale"].double().unsqueeze(1)
        w = state["w"].double() * state["w_scale"].double().unsqueeze(1)
    else:
        x, w, group = state["x"].double(), state["q"].double(), case["group"] or case["dim"]
        for i in range(state["scale"].shape[1]):
            columns = w[:, i * group : (i + 1) * group]
            columns -= state["zero"][:, i : i + 1].double() if case["zeros"] else 8.0
            columns *= state["scale"][:, i : i + 1].double()
    y = torch.mm(x, w.t())
    return {"y": y if state["bias"] is None else y + state["bias"].double()}
