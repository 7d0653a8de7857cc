"""The 8-bit integer linears of a decoder layer, and the operators that make their inputs, as cases for timing.

``op`` of a case is one public entry point, or the chain of them that an MLP runs:

* ``norm``: RMSNorm (after the residual's addition, or without one) to 8-bit codes with a scale per token;
* ``quantize``: a row's codes and scale (an attention output on its way to the O projection);
* ``swiglu``: the codes and scales of silu(gate) * up, both views of one fused projection's output;
* ``linear``: codes times codes with a scale per token and one per output channel;
* ``mlp``: add + norm, gate/up linear, SwiGLU, down linear.

Widths are those of the Qwen2-0.5B shape that the model builders, the tests and the benchmark use (hidden 896,
projections 1152 = 896 + 2 * 128, intermediate 4864, vocabulary 151936), and odd ones, over 1 to 32768 tokens.
Codes are returned as the values they stand for, code * scale.

Plain forms decide a code in 64 bits, since a value next to a rounding border is lost in 32; their sums over K are exact
in 32 bits while they stay under 2^24, which those of these inputs do.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
HIDDEN, INTERMEDIATE, VOCAB, EPS = 896, 4864, 151936, 1e-6


def listed():
    return [
        # One token of one conversation: the norm in front of a projection.
        {"name": "norm, one token", "op": "norm", "rows": 1, "k": HIDDEN, "dtype": "bf16", "residual": True},
        # A prefill of eight prompts of 512 tokens.
        {"name": "norm, prefill", "op": "norm", "rows": 4096, "k": HIDDEN, "dtype": "bf16", "residual": True},
        # The first norm of a model in fp32, of a width that no vector divides.
        {"name": "norm, ragged fp32", "op": "norm", "rows": 9001, "k": 1001, "dtype": "fp32", "residual": False},
        # The attention output of a long prefill, in front of the O projection.
        {"name": "quantize, long prefill", "op": "quantize", "rows": 16384, "k": HIDDEN, "dtype": "fp16"},
        # A decode batch's MLP activation.
        {"name": "swiglu, decode", "op": "swiglu", "rows": 32, "k": INTERMEDIATE, "dtype": "bf16"},
        # The same of a prefill: the most bytes that an elementwise step of a layer moves.
        {"name": "swiglu, prefill", "op": "swiglu", "rows": 4096, "k": INTERMEDIATE, "dtype": "bf16"},
        # Q, K and V of a decode batch in one product, with their bias.
        {"name": "linear, decode QKV", "op": "linear", "rows": 8, "n": 1152, "k": HIDDEN, "bias": True, "dtype": "bf16"},
        # The vocabulary head of a decode step: bound by the weight's bytes.
        {"name": "linear, decode head", "op": "linear", "rows": 8, "n": VOCAB, "k": HIDDEN, "bias": False,
         "dtype": "bf16"},
        # Gate and up of a prefill in one product: bound by the matrix cores and the output's bytes.
        {"name": "linear, prefill gate/up", "op": "linear", "rows": 4096, "n": 2 * INTERMEDIATE, "k": HIDDEN,
         "bias": False, "dtype": "bf16"},
        # The down projection of the largest prefill.
        {"name": "linear, prefill down", "op": "linear", "rows": 32768, "n": HIDDEN, "k": INTERMEDIATE, "bias": False,
         "dtype": "bf16"},
        # Sizes that no tile and no vector divides.
        {"name": "linear, ragged", "op": "linear", "rows": 301, "n": 1003, "k": 1001, "bias": True, "dtype": "fp16"},
        # The MLP of a decode batch between the usual sizes.
        {"name": "mlp, 48 rows", "op": "mlp", "rows": 48, "k": HIDDEN, "n": INTERMEDIATE, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "swiglu", "linear", "linear", "linear", "mlp"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "mlp":
        return {"op": op, "rows": _spread(rng, 1, 4096), "k": HIDDEN, "n": rng.choice([INTERMEDIATE, 1216, 1187]),
                "dtype": rng.choice(["bf16", "fp16"])}
    if op == "linear":
        k = rng.choice([HIDDEN, HIDDEN, INTERMEDIATE, 16 * _spread(rng, 1, 300), _spread(rng, 1, 4000)])
        n = rng.choice([HIDDEN, 1152, 2 * INTERMEDIATE, VOCAB, _spread(rng, 1, 20000)])
        # At most the largest listed products and outputs.
        most = min(32768, 32768 * HIDDEN * INTERMEDIATE // (n * k), 4096 * 2 * INTERMEDIATE // n)
        return {"op": op, "rows": _spread(rng, 1, most), "n": n, "k": k, "bias": rng.random() < 0.5, "dtype": dtype}
    k = rng.choice([HIDDEN, INTERMEDIATE, 8 * _spread(rng, 1, 1024), _spread(rng, 1, 9000)])
    case = {"op": op, "rows": _spread(rng, 1, min(32768, 4096 * 4864 // k)), "k": k, "dtype": dtype}
    if op == "norm":
        case["residual"] = rng.random() < 0.6
    return case


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _codes(rows, k, g):
    """Codes spread as a weight's or an activation's are, and their scales."""

    codes = torch.randn(rows, k, device=DEVICE, generator=g).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.rand(rows, device=DEVICE, generator=g).mul_(0.002).add_(0.001)
    return codes, scales


def _activations(rows, k, dtype, g, scale=1.0):
    """Tokens of unlike sizes with a few strong channels; one token in 64 is padding, all zero."""

    x = torch.randn(rows, k, device=DEVICE, generator=g)
    x *= torch.rand(rows, 1, device=DEVICE, generator=g).mul_(2).add_(0.25) * scale
    x[:, :: max(1, k // 5)] *= 8.0
    if rows >= 64:
        x[63::64] = 0.0
    return x.to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    dtype, op, rows, k = DTYPES[case["dtype"]], case["op"], case["rows"], case["k"]
    state = {"op": op, "dtype": dtype}
    if op in ("norm", "mlp"):
        state["x"] = _activations(rows, k, dtype, g)
        state["residual"] = _activations(rows, k, dtype, g, 4.0) if op == "mlp" or case["residual"] else None
        state["weight"] = torch.randn(k, device=DEVICE, generator=g).mul_(0.2).add_(1.0).to(dtype)
    if op == "quantize":
        state["x"] = _activations(rows, k, dtype, g)
    if op == "swiglu":
        both = _activations(rows, 2 * k, dtype, g, 1.5)
        state["gate"], state["up"] = both[:, :k], both[:, k:]
    if op == "linear":
        state["codes"], state["scales"] = _codes(rows, k, g)
        state["w"], state["ws"] = _codes(case["n"], k, g)
        state["bias"] = torch.randn(case["n"], device=DEVICE, generator=g).to(dtype) if case["bias"] else None
    if op == "mlp":
        state["w"], state["ws"] = _codes(2 * case["n"], k, g)
        state["w_down"], state["ws_down"] = _codes(k, case["n"], g)
    return state


def _q8(y):
    """Codes (as 64-bit values) and scales of the rows of a 64-bit y."""

    amax = y.abs().amax(-1, keepdim=True)
    codes = torch.where(amax > 0, torch.round(y * 127 / amax), 0.0)
    return codes, amax.squeeze(-1) / 127


def _values(codes, scales):
    return codes.float() * scales.float().unsqueeze(-1)


def _norm(x, residual, weight):
    summed = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    h = summed.double()
    # The statistic divides every value of a row alike, so it scales the row and leaves its codes.
    codes, scales = _q8(h * weight.double())
    return summed, codes, scales * torch.rsqrt(h.square().mean(-1) + EPS)


def _swiglu(gate, up):
    g = gate.double()
    return _q8(g / (1 + torch.exp(-g)) * up.double())


def _linear(codes, scales, w, ws, bias, dtype):
    y = codes.float() @ w.float().t() * scales.float().unsqueeze(-1) * ws
    return (y if bias is None else y + bias.float()).to(dtype)


def _import_backends():
    """The framework's kernels, imported once as a program does, not in every pass."""

    package = str(Path("llm-compiler_amd").resolve())
    if package not in sys.path:
        sys.path.insert(0, package)
    from stateful_llm_compiler_hip import backends

    _run_own.backends = backends
    return backends


def _run_own(state):
    backends = getattr(_run_own, "backends", None) or _import_backends()
    op = state["op"]
    if op == "linear":
        return backends.hip_linear_q8(state["codes"], state["scales"], state["w"], state["ws"], state["bias"],
                                      output_dtype=state["dtype"])
    if op == "mlp":
        summed, codes, scales = backends.hip_add_rms_norm_q8(state["x"], state["residual"], state["weight"],
                                                             epsilon=EPS)
        both = backends.hip_linear_q8(codes, scales, state["w"], state["ws"], output_dtype=state["dtype"])
        gate, up = both.chunk(2, dim=-1)
        codes, scales = backends.hip_swiglu_q8(gate, up)
        return summed, backends.hip_linear_q8(codes, scales, state["w_down"], state["ws_down"],
                                              output_dtype=state["dtype"])
    if op == "quantize":
        codes, scales = backends.hip_quantize_q8(state["x"])
    elif op == "swiglu":
        codes, scales = backends.hip_swiglu_q8(state["gate"], state["up"])
    elif state["residual"] is None:
        codes, scales = backends.hip_rms_norm_q8(state["x"], state["weight"], epsilon=EPS)
    else:
        summed, codes, scales = backends.hip_add_rms_norm_q8(state["x"], state["residual"], state["weight"],
                                                             epsilon=EPS)
        return summed, codes * scales.unsqueeze(-1)
    return codes * scales.unsqueeze(-1)


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "linear":
        return _linear(state["codes"], state["scales"], state["w"], state["ws"], state["bias"], state["dtype"])
    if op == "mlp":
        summed, codes, scales = _norm(state["x"], state["residual"], state["weight"])
        both = _linear(codes, scales, state["w"], state["ws"], None, state["dtype"])
        codes, scales = _swiglu(*both.chunk(2, dim=-1))
        return summed, _linear(codes, scales, state["w_down"], state["ws_down"], None, state["dtype"])
    if op == "quantize":
        return _values(*_q8(state["x"].double()))
    if op == "swiglu":
        return _values(*_swiglu(state["gate"], state["up"]))
    summed, codes, scales = _norm(state["x"], state["residual"], state["weight"])
    return _values(codes, scales) if state["residual"] is None else (summed, _values(codes, scales))


def work(case):
    op, rows, k, size = case["op"], case["rows"], case["k"], BYTES[case["dtype"]]
    if op == "linear":
        n = case["n"]
        read = (rows + n) * (k + 4) + (n * size if case["bias"] else 0)
        return {"bytes": read + rows * n * size, "flops": 2 * rows * n * k}
    if op == "mlp":
        n = case["n"]
        return {"bytes": 3 * n * k + 4 * (2 * n + k) + k * size + 4 * rows * k * size, "flops": 6 * rows * n * k}
    if op == "norm":
        return {"bytes": rows * k * size * (3 if case["residual"] else 1) + rows * (k + 4) + k * size,
                "flops": 6 * rows * k}
    reads = 2 if op == "swiglu" else 1
    return {"bytes": rows * k * size * reads + rows * (k + 4), "flops": (10 if op == "swiglu" else 4) * rows * k}


def exact(case, seed):
    state = prepare(case, seed)
    op, dtype = state["op"], state["dtype"]

    def coded(y):
        # The step of a row is its largest magnitude over 127; a code is the nearest whole number of steps.
        top = torch.maximum(y.amax(-1), -y.amin(-1))
        steps = (127 * y) / torch.clamp(top, min=torch.finfo(torch.float64).tiny)[:, None]
        return steps.round(), top / 127

    def normed():
        h = state["x"].double()
        if state["residual"] is not None:
            h = (h + state["residual"].double()).to(dtype).double()
        codes, step = coded(h * state["weight"].double())
        return h, codes, step / ((h * h).sum(-1) / h.shape[-1] + EPS).sqrt()

    def product(codes, step, w, ws):
        return (codes * step[:, None]) @ (w.double() * ws.double()[:, None]).t()

    if op == "linear":
        y = product(state["codes"].double(), state["scales"].double(), state["w"], state["ws"])
        return y if state["bias"] is None else y + state["bias"].double()
    if op in ("quantize", "swiglu"):
        y = state["x"].double() if op == "quantize" else (
            state["gate"].double() * torch.sigmoid(state["gate"].double()) * state["up"].double())
        codes, step = coded(y)
        return codes * step[:, None]
    h, codes, step = normed()
    if op == "norm":
        values = codes * step[:, None]
        return values if state["residual"] is None else (h, values)
    # Between its operators the MLP's tensors are stored in their type: those roundings are part of it.
    gate, up = product(codes, step, state["w"], state["ws"]).to(dtype).double().chunk(2, dim=-1)
    codes, step = coded(gate * torch.sigmoid(gate) * up)
    return h, product(codes, step, state["w_down"], state["ws_down"])
