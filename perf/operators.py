"""Cases of the 8-bit operators (e4m3 values with one power-of-two scale per block of 128): storing rows in 8 bits and
restoring them, the linear map and the expert-grouped linear map on 8-bit operands, and SwiGLU that keeps its inputs
in 8 bits for the backward pass.

`run` computes a case with elementary torch operations, or, where `own` is set, through the package's operators.

The format: a block is 128 consecutive columns of one row (activations, gradients), or 128 x 128 (weights; blocks at
the edges are smaller).  Its exponent e is the smallest whole number with amax <= 448 * 2^e over the finite elements
(0 for a block of zeros, kept in [-127, 127]); an element x is held as e4m3(x * 2^-e), rounded to nearest even."""

import math
import sys

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the hidden states of 16384 tokens kept for the backward pass and read back
        {"name": "store bf16 16384x4096", "op": "store", "dtype": "bf16", "rows": 16384, "cols": 4096},
        # a ragged fp32 tensor: the last block of a row is short
        {"name": "store fp32 333x1000", "op": "store", "dtype": "fp32", "rows": 333, "cols": 1000},
        # serving one token: the weights are read once
        {"name": "linear 1 token", "op": "linear", "train": False, "dtype": "bf16", "rows": 1, "cols": 4096, "out": 14336},
        # a handful of tokens, widths that fill no block
        {"name": "linear 5 tokens odd", "op": "linear", "train": False, "dtype": "fp16", "rows": 5, "cols": 1000, "out": 1544},
        # a prompt
        {"name": "linear 2048 tokens", "op": "linear", "train": False, "dtype": "fp16", "rows": 2048, "cols": 4096, "out": 4096},
        # a training step: forward, input gradient, weight gradient
        {"name": "linear train 8192", "op": "linear", "train": True, "dtype": "bf16", "rows": 8192, "cols": 4096, "out": 14336},
        # one token through its 8 of 128 experts
        {"name": "experts 1 token", "op": "experts", "train": False, "dtype": "bf16", "rows": 8, "experts": 128, "cols": 2048, "out": 1536},
        # 64 tokens in flight, a few rows per expert, some experts without any
        {"name": "experts 64 tokens", "op": "experts", "train": False, "dtype": "bf16", "rows": 512, "experts": 128, "cols": 2048, "out": 1536},
        # a training step of 8192 tokens with 8 experts each
        {"name": "experts train 65536", "op": "experts", "train": True, "dtype": "bf16", "rows": 65536, "experts": 128, "cols": 2048, "out": 1536},
        # the same on a small ragged problem in half precision
        {"name": "experts train 777 odd", "op": "experts", "train": True, "dtype": "fp16", "rows": 777, "experts": 9, "cols": 264, "out": 520},
        # SwiGLU of the fine-grained layer's rows, forward and backward, inputs kept in 8 bits
        {"name": "swiglu 32781x1536", "op": "swiglu", "dtype": "bf16", "rows": 32781, "cols": 1536},
        # a small fp32 one
        {"name": "swiglu fp32 257x264", "op": "swiglu", "dtype": "fp32", "rows": 257, "cols": 264},
    ]


def _between(rng, low, high, step=1):
    """A multiple of `step` from [low, high], its logarithm uniform."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return int(min(high, max(low, round(v / step) * step)))


def draw(rng):
    op = rng.choice(["store", "linear", "linear", "experts", "experts", "swiglu"])
    if op in ("store", "swiglu"):
        cols = _between(rng, 64, 8192, 8)
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": _between(rng, 16, min(32768, (1 << 25) // cols)), "cols": cols}
    case = {"op": op, "train": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16"])}
    cols, out = _between(rng, 128, 4096, 8), _between(rng, 128, 4096, 8)
    if op == "linear":
        return {**case, "rows": _between(rng, 1, 8192), "cols": cols, "out": out}
    cols, out = _between(rng, 128, 2048, 8), _between(rng, 128, 1536, 8)
    experts = _between(rng, 2, 64)
    return {**case, "rows": _between(rng, 8, 16384), "experts": experts, "cols": cols, "out": out}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    rows, cols = case["rows"], case["cols"]
    state = {"case": dict(case)}
    if case["op"] == "swiglu":
        # up and gate are the two halves of one projection's output, as the layer has them
        state["up"], state["gate"] = normal(rows, 2 * cols, scale=1.5).chunk(2, dim=-1)
        state["d_out"] = normal(rows, cols)
        return state
    # activations: unit variance, a few channels that are eight times larger
    loud = 1.0 + 7.0 * (torch.rand(cols, generator=g, device="cuda") > 0.995)
    state["x"] = (torch.randn(rows, cols, generator=g, device="cuda") * loud).to(dtype)
    if case["op"] == "store":
        return state
    if case["op"] == "experts":
        experts = case["experts"]
        share = 1.0 + 2.0 * torch.rand(experts, generator=g, device="cuda")
        if experts >= 8:
            share[3::5] = 0.0  # experts that no token chose
        edge = torch.cumsum(share / share.sum(), 0)
        ids = torch.searchsorted(edge, torch.rand(rows, generator=g, device="cuda") * edge[-1], right=True).clamp_(max=experts - 1)
        state["expert_frequency"] = torch.bincount(ids, minlength=experts).to(torch.int32)
        state["longest"] = int(state["expert_frequency"].max())
        state["weight"] = normal(experts, case["out"], cols, scale=0.02)
    else:
        state["weight"] = normal(case["out"], cols, scale=0.02)
    if case["train"]:
        state["d_out"] = normal(rows, case["out"], scale=0.01)
    elif own:
        state["quantized"] = _package().quantize_fp8_weight(state.pop("weight"))  # a server keeps its weights in 8 bits
    else:
        state["quantized"] = _held(state.pop("weight"), True)
    return state


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "store":
        return _held(state["x"], False).to(state["x"].dtype)
    if op == "swiglu":
        return _plain_swiglu(state["gate"], state["up"], state["d_out"])
    if op == "linear":
        return _plain_linear(state)
    return _plain_experts(state)


# ---- the package's operators -----------------------------------------------------------------------
def _package():
    if "cute-kernels_b200" not in sys.path:
        sys.path.insert(0, "cute-kernels_b200")
    import fma_b200

    return fma_b200


def _run_own(state):
    fma = _package()
    case = state["case"]
    if case["op"] == "store":
        return fma.quantize_fp8(state["x"]).dequantize()
    if case["op"] == "swiglu":
        gate, up = state["gate"].detach().requires_grad_(), state["up"].detach().requires_grad_()
        out = fma.swiglu_fp8_checkpoint(gate, up)
        return (out.detach(), *torch.autograd.grad(out, (gate, up), state["d_out"]))
    grouped = case["op"] == "experts"
    if not case["train"]:
        with torch.no_grad():
            if grouped:
                return fma.grouped_linear_fp8(state["x"], state["quantized"], state["expert_frequency"])
            return fma.linear_fp8(state["x"], state["quantized"])
    x, weight = state["x"].detach().requires_grad_(), state["weight"].detach().requires_grad_()
    out = fma.grouped_linear_fp8(x, weight, state["expert_frequency"]) if grouped else fma.linear_fp8(x, weight)
    return (out.detach(), *torch.autograd.grad(out, (x, weight), state["d_out"]))


# ---- the plain form --------------------------------------------------------------------------------
def _held(x, square):
    """The values, in 32 bits, that the 8-bit form of x stands for: blocks of 1 x 128, or of 128 x 128 if `square`."""
    x = x.float()
    r, c = x.shape[-2:]
    tall = BLOCK if square else 1
    padded = torch.nn.functional.pad(x, (0, -c % BLOCK, 0, -r % tall))
    blocks = padded.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, tall))  # [..., block row, row, block column, column]
    size = blocks.abs()
    amax = torch.where(torch.isfinite(size), size, 0.0).amax(dim=(-3, -1), keepdim=True)
    mantissa, exponent = torch.frexp(amax)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(-127, 127)
    e = torch.where(amax > 0, e, 0)
    held = torch.ldexp(torch.ldexp(blocks, -e).to(torch.float8_e4m3fn).float(), e)
    return held.flatten(-2, -1).flatten(-3, -2)[..., :r, :c]


def _plain_linear(state):
    x, dtype = state["x"], state["x"].dtype
    held_x = _held(x, False)
    if not state["case"]["train"]:
        return (held_x @ state["quantized"].T).to(dtype)
    held_w = _held(state["weight"], True)
    d_out = state["d_out"]
    return (held_x @ held_w.T).to(dtype), (_held(d_out, False) @ held_w).to(dtype), (d_out.float().T @ held_x).to(dtype)


def _plain_experts(state):
    case, x = state["case"], state["x"]
    dtype, count, longest = x.dtype, state["expert_frequency"].long(), state["longest"]
    ends = torch.cumsum(count, 0)
    held_x = _held(x, False)
    held_w = _held(state["weight"], True) if case["train"] else state["quantized"]
    if not case["train"] and x.size(0) <= case["experts"]:  # fewer rows than experts: each row with its expert's weight
        expert = torch.searchsorted(ends, torch.arange(x.size(0), device=x.device), right=True)
        return torch.einsum("rk,rnk->rn", held_x, held_w[expert]).to(dtype)
    # each expert's rows, padded with zeros to the longest
    place = torch.arange(longest, device=x.device)
    filled = place < count[:, None]
    row = torch.where(filled, (ends - count)[:, None] + place, 0)
    back = torch.nonzero(filled.flatten()).squeeze(1)
    spread = lambda t: torch.where(filled[..., None], t[row], 0.0)  # noqa: E731
    out = (spread(held_x) @ held_w.transpose(1, 2)).flatten(0, 1)[back].to(dtype)
    if not case["train"]:
        return out
    d_out = state["d_out"]
    d_x = (spread(_held(d_out, False)) @ held_w).flatten(0, 1)[back].to(dtype)
    return out, d_x, (spread(d_out.float()).transpose(1, 2) @ spread(held_x)).to(dtype)


def _plain_swiglu(gate, up, d_out):
    dtype = gate.dtype
    g, u, d = gate.float(), up.float(), d_out.float()
    out = u * g * torch.sigmoid(g)
    g, u = _held(gate, False), _held(up, False)
    s = torch.sigmoid(g)
    return out.to(dtype), (d * u * (s + g * s * (1 - s))).to(dtype), (d * g * s).to(dtype)


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "store":
        # read, kept in 8 bits, read again, written
        return {"bytes": rows * cols * (2 * size + 2), "flops": 2 * rows * cols}
    if case["op"] == "swiglu":
        # gate, up in; out; both kept in 8 bits and read again; d_out in; two gradients
        return {"bytes": rows * cols * (6 * size + 4), "flops": 30 * rows * cols}
    out, experts = case["out"], case.get("experts", 1)
    used = min(experts, rows)
    if case["train"]:
        return {"bytes": size * (2 * rows * (cols + out) + 2 * experts * cols * out), "flops": 6 * rows * cols * out}
    return {"bytes": size * rows * (cols + out) + used * cols * out, "flops": 2 * rows * cols * out}


# ---- the definition in 64 bits ---------------------------------------------------------------------
def _exact_held(x, tall):
    """As the module's text defines the format, block row by block row."""
    x = x.double()
    out = torch.empty_like(x)
    for r in range(0, x.size(0), tall) if tall > 1 else [0]:
        for c in range(0, x.size(1), BLOCK):
            part = x[r : r + tall, c : c + BLOCK] if tall > 1 else x[:, c : c + BLOCK]
            amax = part.abs().max() if tall > 1 else part.abs().max(1, keepdim=True).values
            e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448.0))
            e = e + (amax > 448.0 * torch.exp2(e)).double() - (amax <= 448.0 * torch.exp2(e - 1)).double()
            unit = torch.exp2(torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e)))
            scaled = part / unit
            # e4m3 by its definition: 3 fraction bits, smallest normal 2^-6, subnormals in steps of 2^-9
            place = torch.floor(torch.log2(scaled.abs().clamp(min=2.0**-6)))
            place = place - (torch.exp2(place) > scaled.abs().clamp(min=2.0**-6)).double()
            step = torch.exp2(place - 3)
            held = torch.round(scaled / step) * step * unit
            if tall > 1:
                out[r : r + tall, c : c + BLOCK] = held
            else:
                out[:, c : c + BLOCK] = held
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    weight = None
    try:
        if case["op"] in ("linear", "experts") and not case["train"]:
            state = prepare({**case, "train": True}, seed)  # the same draws up to the weight
        else:
            state = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "store":
        return _exact_held(state["x"], 1)
    if case["op"] == "swiglu":
        g, u, d = state["gate"].double(), state["up"].double(), state["d_out"].double()
        out = u * g / (1 + torch.exp(-g))
        g, u = _exact_held(state["gate"], 1), _exact_held(state["up"], 1)
        s = 1 / (1 + torch.exp(-g))
        return out, d * u * s * (1 + g * (1 - s)), d * g * s
    x, weight = _exact_held(state["x"], 1), state["weight"]
    counts = state["expert_frequency"].tolist() if case["op"] == "experts" else [case["rows"]]
    weights = weight if case["op"] == "experts" else weight[None]
    outs, d_xs, d_ws = [], [], []
    at = 0
    if case["train"]:
        d_out = state["d_out"].double()
        held_d = _exact_held(state["d_out"], 1)
    for n, w in zip(counts, weights):
        if not n and not case["train"]:
            continue
        rows = slice(at, at + n)
        at += n
        w = _exact_held(w, BLOCK) if n else w.double()
        outs.append(x[rows] @ w.T)
        if case["train"]:
            d_xs.append(held_d[rows] @ w)
            d_ws.append(d_out[rows].T @ x[rows])
    if not case["train"]:
        return torch.cat(outs)
    d_w = torch.stack(d_ws)
    return torch.cat(outs), torch.cat(d_xs), d_w if case["op"] == "experts" else d_w[0]
