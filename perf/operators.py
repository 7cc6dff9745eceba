"""The operators of a decoder layer whose matrix products take 8-bit operands (e4m3 with a 32-bit scale a row), one call at a time.

``norm``: residual add, RMS norm and its output in 8 bits. ``quantize``: rows (an attention's or a gated unit's output) to 8 bits.
``linear``: product with bias, activation and residual in its epilogue. ``gated``: gate and up projections, activation and product in one.

Sizes are those of the Qwen2.5 shapes (hidden 896 to 5,120, feed-forward 4,864 to 18,944) and of a squared-relu feed-forward of width
2,048; tokens go from one decoded token to prompt bursts of 8,192.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
LARGEST = 448.0  # of e4m3
SMALLEST_SCALE = 2.0**-126

TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed() -> list[dict]:
    return [
        # The norm in front of q/k/v for one decoded token of the 7B shape: nothing but latency.
        dict(name="norm_1", kind="norm", rows=1, columns=3584, delta="bfloat16"),
        # The same for a prompt portion of the 14B shape.
        dict(name="norm_2048", kind="norm", rows=2048, columns=5120, delta="bfloat16"),
        # A continuous-batching step of no round size whose rows are no whole 16-byte steps, branch output in 32 bits.
        dict(name="norm_ragged", kind="norm", rows=1777, columns=1001, delta="float32"),
        # The gated unit's output of a prompt portion, in front of the 7B down product.
        dict(name="quantize_2048", kind="quantize", rows=2048, columns=18944, dtype="bfloat16"),
        # The attention outputs of 24 decoded tokens of the 1.5B shape, in front of the output product.
        dict(name="quantize_24", kind="quantize", rows=24, columns=1536, dtype="bfloat16"),
        # q/k/v of one decoded token, 7B: 16 MB of weights, latency counts.
        dict(name="qkv_1", kind="linear", tokens=1, inner=3584, outer=4608, bias=True, activation="", residual=False, out="bfloat16"),
        # The attention's output product of 64 requests, added into the 32-bit residual stream, 14B.
        dict(name="output_64", kind="linear", tokens=64, inner=5120, outer=5120, bias=False, activation="", residual=True, out="float32"),
        # An up projection with a squared relu over a prompt whose length is a multiple of nothing.
        dict(name="squared_relu_777", kind="linear", tokens=777, inner=2048, outer=8192, bias=False, activation="squared_relu", residual=False, out="bfloat16"),
        # The down product of a prompt portion into the residual stream, 7B.
        dict(name="down_2048", kind="linear", tokens=2048, inner=18944, outer=3584, bias=False, activation="", residual=True, out="float32"),
        # Gate and up of one decoded token, 7B: 136 MB of weights.
        dict(name="gate_up_1", kind="gated", tokens=1, inner=3584, width=18944, activation="silu", out="bfloat16"),
        # Gate and up of 48 requests, 1.5B, the gelu unit.
        dict(name="gate_up_48", kind="gated", tokens=48, inner=1536, width=8960, activation="gelu", out="bfloat16"),
        # Gate and up of a prompt burst of 8,192 tokens, 7B: the largest product of a step.
        dict(name="gate_up_8192", kind="gated", tokens=8192, inner=3584, width=18944, activation="silu", out="bfloat16"),
    ]


def draw(rng) -> dict:
    """Another case of the same ranges: one token to 8,192, layers from 64 channels to the 7B feed-forward's, any alignment."""

    def spread(low: int, high: int) -> int:
        return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    def channels(low: int, high: int) -> int:
        n = spread(low, high)
        return n if rng.random() < 0.25 else max(low, (n + 32) // 64 * 64)

    kind = rng.choice(("norm", "quantize", "linear", "linear", "gated", "gated"))
    tokens = spread(1, 8192)
    if kind == "norm":
        return dict(kind=kind, rows=tokens, columns=channels(64, 8192), delta=rng.choice(("bfloat16", "float32", "")))
    if kind == "quantize":
        return dict(kind=kind, rows=min(tokens, 4096), columns=channels(64, 18944), dtype=rng.choice(("bfloat16", "float32")))
    inner = channels(64, 18944)
    most = 8192 * 3584 * 37888 // (tokens * inner)
    if kind == "gated":
        return dict(kind=kind, tokens=tokens, inner=inner, width=channels(64, min(18944, max(64, most // 2))), activation=rng.choice(("silu", "gelu")),
                    out=rng.choice(("bfloat16", "bfloat16", "float32")))
    return dict(kind=kind, tokens=tokens, inner=inner, outer=channels(64, min(37888, max(64, most))), bias=rng.random() < 0.5,
                activation=rng.choice(("", "", "silu", "gelu", "squared_relu")), residual=rng.random() < 0.5, out=rng.choice(("bfloat16", "float32")))


# --- inputs --------------------------------------------------------------------------------------


def rows8(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of numbers in e4m3 with a scale a row; a row's 8-bit numbers start on a 16-byte boundary, as a matrix product takes them."""
    rows, columns = v.shape
    scales = torch.clamp(v.abs().amax(1) / LARGEST, min=SMALLEST_SCALE)
    held = torch.zeros(rows, -(-columns // 16) * 16, dtype=torch.float8_e4m3fn, device=v.device)
    held[:, :columns] = (v / scales[:, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    return held[:, :columns], scales


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)

    def normal(*shape: int, std: float = 1.0, mean: float = 0.0) -> torch.Tensor:
        return torch.randn(*shape, generator=gen, device=DEVICE) * std + mean

    kind = case["kind"]
    state = dict(case=case)
    if kind == "norm":
        rows, columns = case["rows"], case["columns"]
        # A residual stream: a few channels are far larger than the rest.
        loud = 1.0 + 30.0 * (torch.rand(columns, generator=gen, device=DEVICE) < 0.004)
        state["x"] = normal(rows, columns) * loud
        state["delta"] = normal(rows, columns, std=0.3).to(TYPES[case["delta"]]) if case["delta"] else None
        state["weight"] = normal(columns, std=0.2, mean=1.0)
        state["stream"] = torch.empty_like(state["x"])
        state["out"] = rows8(torch.zeros_like(state["x"]))
    elif kind == "quantize":
        v = normal(case["rows"], case["columns"])
        state["x"] = (v * torch.sigmoid(v) * normal(case["rows"], case["columns"], std=0.5)).to(TYPES[case["dtype"]])  # what a gated unit leaves
        state["out"] = rows8(torch.zeros(case["rows"], case["columns"], device=DEVICE))
    else:
        tokens, inner = case["tokens"], case["inner"]
        outer = case["outer"] if kind == "linear" else 2 * case["width"]
        state["x"] = rows8(normal(tokens, inner))
        state["w"] = rows8(normal(outer, inner, std=0.02))
        state["bias"] = normal(outer) if case.get("bias") else None
        state["residual"] = normal(tokens, outer, std=2.0) if case.get("residual") else None
        state["out"] = torch.empty(tokens, outer if kind == "linear" else case["width"], dtype=TYPES[case["out"]], device=DEVICE)
    return state


# --- the calls that are measured -----------------------------------------------------------------

_CONTEXT = None


def context():
    """The step context that a program of this framework runs its operators in: library, error word and workspace."""
    global _CONTEXT
    if _CONTEXT is None:
        import numpy as np

        from llm_inference_b200.csrc.library import kernels
        from llm_inference_b200.parts.context import HostBatch, StepContext, Workspace

        names = ("token_ids", "positions", "token_seq", "seq_q_start", "seq_q_len", "seq_kv_len", "seq_slot", "logit_rows")
        device = torch.device(DEVICE)
        none = torch.zeros(0, dtype=torch.int32, device=device)
        _CONTEXT = StepContext(
            lib=kernels(), dtype=torch.bfloat16, device=device, num_tokens=0, num_seqs=0, host=HostBatch(**{n: np.zeros(0, np.int32) for n in names}),
            err=torch.zeros(1, dtype=torch.int32, device=device), workspace=Workspace(device), **{n: none for n in names})
    return _CONTEXT


def run(state: dict):
    return run_own(state) if own else run_plain(state)


def run_own(state: dict):
    from llm_inference_b200.parts import float8

    case, ctx = state["case"], context()
    if case["kind"] == "norm":
        out = float8.rmsnorm(ctx, state["x"], state["delta"], state["weight"], EPS, float8.Float8Rows(*state["out"]), stream=state["stream"])
        return (out.values, out.scales, state["stream"]) if state["delta"] is not None else (out.values, out.scales)
    if case["kind"] == "quantize":
        out = float8.quantize(ctx, state["x"], float8.Float8Rows(*state["out"]))
        return out.values, out.scales
    x, w = float8.Float8Rows(*state["x"]), float8.Float8Rows(*state["w"], constant=True)
    if case["kind"] == "gated":
        return float8.linear_gated(ctx, x, w, state["out"], activation=case["activation"])
    return float8.linear(ctx, x, w, state["out"], bias=state["bias"], activation=case["activation"] or None, residual=state["residual"])


def activated(v: torch.Tensor, name: str) -> torch.Tensor:
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "squared_relu":
        return torch.clamp(v, min=0.0) ** 2
    return v


def to_rows8(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    scales = torch.clamp(v.abs().amax(1) / LARGEST, min=SMALLEST_SCALE)
    return (v / scales[:, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn), scales


def run_plain(state: dict):
    case = state["case"]
    if case["kind"] == "norm":
        s = state["x"] if state["delta"] is None else state["x"] + state["delta"].float()
        values, scales = to_rows8(s * torch.rsqrt((s * s).mean(1, keepdim=True) + EPS) * state["weight"])
        return (values, scales, s) if state["delta"] is not None else (values, scales)
    if case["kind"] == "quantize":
        return to_rows8(state["x"].float())
    (x, xs), (w, ws) = state["x"], state["w"]
    y = (x.float() @ w.float().t()) * xs[:, None] * ws
    if case["kind"] == "gated":
        y = activated(y[:, 0::2], case["activation"]) * y[:, 1::2]
    else:
        if state["bias"] is not None:
            y = y + state["bias"]
        y = activated(y, case["activation"])
        if state["residual"] is not None:
            y = y + state["residual"]
    return y.to(TYPES[case["out"]])


# --- the definition in 64 bits, and what a pass cannot do without -----------------------------------


def exact_rows8(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Nearest e4m3 numbers (even on ties) of rows over their scales, found in 64 bits: steps of 2^-9 below 2^-6, else of 1/8 of the binade."""
    scales = torch.clamp(v.abs().amax(1) / LARGEST, min=SMALLEST_SCALE)
    u = v / scales[:, None]
    step = torch.exp2(torch.clamp(torch.frexp(u).exponent - 1, min=-6).double() - 3.0)
    return torch.clamp(torch.round(u / step) * step, -LARGEST, LARGEST), scales


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        s = state["x"].double()
        if state["delta"] is not None:
            s = s + state["delta"].double()
        norm = torch.sqrt(torch.sum(s**2, dim=1, keepdim=True) / case["columns"] + EPS)
        values, scales = exact_rows8(s / norm * state["weight"].double())
        return (values, scales, s) if state["delta"] is not None else (values, scales)
    if kind == "quantize":
        return exact_rows8(state["x"].double())
    (x, xs), (w, ws) = state["x"], state["w"]
    a, b = x.double() * xs.double()[:, None], w.double() * ws.double()[:, None]
    halves = []
    for part in a.split(1024):  # 64-bit products of a whole burst would not fit beside their operands
        z = torch.einsum("mk,nk->mn", part, b)
        if state["bias"] is not None:
            z = z + state["bias"].double()
        first = z[:, 0::2] if kind == "gated" else z
        name = case["activation"]
        if name == "silu":
            r = first * torch.sigmoid(first)
        elif name == "gelu":
            r = first * torch.sigmoid(math.sqrt(8.0 / math.pi) * (first + 0.044715 * first**3))
        elif name == "squared_relu":
            r = torch.where(first > 0, first * first, torch.zeros_like(first))
        else:
            r = first
        halves.append(r * z[:, 1::2] if kind == "gated" else r)
    y = torch.cat(halves)
    return y if state["residual"] is None else y + state["residual"].double()


def work(case: dict) -> dict:
    kind = case["kind"]
    size = {"bfloat16": 2, "float32": 4, "": 0}
    if kind == "norm":
        rows, columns = case["rows"], case["columns"]
        return dict(bytes=rows * columns * (4 + 1 + (4 + size[case["delta"]] if case["delta"] else 0)) + 4 * columns + 4 * rows, flops=8 * rows * columns)
    if kind == "quantize":
        rows, columns = case["rows"], case["columns"]
        return dict(bytes=rows * columns * (size[case["dtype"]] + 1) + 4 * rows, flops=3 * rows * columns)
    m, k = case["tokens"], case["inner"]
    n = case["outer"] if kind == "linear" else 2 * case["width"]
    outputs = m * (n if kind == "linear" else n // 2)
    moved = m * k + n * k + 4 * (m + n) + outputs * size[case["out"]]
    moved += (4 * n if case.get("bias") else 0) + (4 * m * n if case.get("residual") else 0)
    return dict(bytes=moved, flops=2 * m * n * k)
