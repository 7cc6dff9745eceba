"""Products whose terms are all of one sign: what adding toward zero takes from their sums.

An addition on the tensor core drops what lies below the last bit of the sum, of the sum and of the products that come to it, so sums of one sign come out too
small: by up to 1.6e-8 of themselves an addition of 32 products in chains of 320, 4e-8 in chains of up to 4,096 (measured, with a tenth to spare). Chains are cut after
320 additions into 32 bits and after 1,024 into bfloat16, and their sums are added with ordinary rounding (2^-24 each at most). The mean of the outputs'
relative errors shows the loss: roundings to bfloat16 fall to either side (standard deviation at most 2^-8 / sqrt 3 each) and leave five standard
deviations of their mean at most. No output is off by more than four times the loss beside its own roundings."""

from __future__ import annotations

import math

import pytest
import torch

from test_kernels import make_ctx
from llm_inference_b200.parts import float8

gpu = pytest.mark.gpu

CHAIN = {torch.float32: 320, torch.bfloat16: 1024}  # additions
LOSS = {torch.float32: 1.6e-8, torch.bfloat16: 4e-8}  # of a sum of one sign, an addition


def positive(rows: int, columns: int) -> float8.Float8Rows:
    """Magnitudes of normal numbers; scales from 1 to 2, so that outputs are spread over all mantissas."""
    held = torch.empty(rows, columns, dtype=torch.float8_e4m3fn, device="cuda")
    for at in range(0, columns, 1 << 18):
        part = held[:, at : at + (1 << 18)]
        part.copy_((torch.randn(part.shape, device="cuda").abs() * 100).clamp(max=448).to(torch.float8_e4m3fn))
    return float8.Float8Rows(held, 1 + torch.rand(rows, device="cuda"), constant=True)


# Up to 16 tokens, few tokens, tiles; a layer's inner size and a far longer one.
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(9, 4096, 18944), (128, 4096, 18944), (600, 4096, 18944), (4, 2048, 1 << 21), (300, 256, 1 << 21), (600, 256, 1 << 21), (600, 254, 40000)])
def test_sums_of_one_sign(m, n, k, dtype):
    from llm_inference_b200.csrc.library import kernels

    torch.manual_seed(50)
    x, w = positive(m, k), positive(n, k)
    ctx = make_ctx(kernels(), positions=[0])
    out = float8.linear(ctx, x, w, torch.empty(m, n, device="cuda", dtype=dtype))
    y = torch.zeros(m, n, device="cuda", dtype=torch.float64)
    for at in range(0, k, 1 << 16):
        y += x.values[:, at : at + (1 << 16)].double() @ w.values[:, at : at + (1 << 16)].double().t()
    y *= x.scales.double()[:, None] * w.scales.double()
    error = (out.double() - y) / y
    additions = math.ceil(k / 32)
    loss = LOSS[dtype] * min(additions, CHAIN[dtype])
    roundings = (math.ceil(additions / CHAIN[dtype]) + 16 + 4) * 2.0**-24  # chains, members of a cluster, scales
    half_step = torch.finfo(dtype).eps / 2
    assert float(error.abs().max()) <= 4 * loss + roundings + 1.01 * half_step
    assert abs(float(error.mean())) <= loss + roundings + (5 * half_step / math.sqrt(3 * m * n) if dtype == torch.bfloat16 else 0.0)
    assert int(ctx.err.item()) == 0


@gpu
@pytest.mark.parametrize("kind", ["squared_relu", "gated"])
@pytest.mark.parametrize("m", [40, 600])
def test_long_rows_under_an_activation(m, kind):
    """bfloat16 outputs of rows of several chains, numbers of both signs: a sum is off by 2^-23 of its magnitudes' sum an addition at most, 1,024 in a chain."""
    from llm_inference_b200.csrc.library import kernels
    from test_float8 import half_step, operand, slope, wide_activation, wide_product

    torch.manual_seed(51)
    n, k = 250, 70000
    x, w = operand(m, k), operand(n, k, 0.02)
    ctx = make_ctx(kernels(), positions=[0])
    y, magnitudes = wide_product(x, w)
    off = magnitudes * 2.0**-23 * (1024 + 3 + 16 + 16 + 4)
    if kind == "gated":
        out = float8.linear_gated(ctx, x, w, torch.empty(m, n // 2, device="cuda", dtype=torch.bfloat16))
        g, u, og, ou = y[:, 0::2], y[:, 1::2], off[:, 0::2], off[:, 1::2]
        a = wide_activation(g, "silu")
        want, limit = a * u, slope(g, og, "silu") * (u.abs() + ou) + a.abs() * ou
    else:
        out = float8.linear(ctx, x, w, torch.empty(m, n, device="cuda", dtype=torch.bfloat16), activation=kind)
        want, limit = wide_activation(y, kind), slope(y, off, kind)
    assert torch.all((out.double() - want).abs() <= limit + (half_step(torch.bfloat16) * 1.01 + 2.0**-22) * want.abs())
    assert int(ctx.err.item()) == 0
