"""The numbers of 8-bit rows: a quotient by the scale is rounded to 32 bits and then to the nearest e4m3 number, wherever it is computed."""

from __future__ import annotations

import math

import pytest
import torch

from test_kernels import make_ctx
from llm_inference_b200.parts import float8

gpu = pytest.mark.gpu


def elementary(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """8-bit rows by elementary 32-bit operations: NaN counts for nothing in a row's largest magnitude."""
    v = x.float()
    largest = torch.where(torch.isnan(v), torch.zeros_like(v), v.abs()).amax(1)
    scales = torch.clamp(largest * (1.0 / 448.0), min=2.0**-126)
    return (v / scales[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scales


def same_numbers(rows: float8.Float8Rows, values: torch.Tensor, scales: torch.Tensor) -> None:
    assert torch.equal(rows.scales.cpu(), scales.cpu())
    got, want = rows.values.float().cpu(), values.float().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_inputs_lie_on_middles():
    """Rows of bfloat16 numbers often have quotients that are exactly between two e4m3 numbers: the inputs below do test ties."""
    torch.manual_seed(40)
    x = torch.randn(64, 1536).bfloat16()
    u = (x.float() / (x.float().abs().amax(1) * (1.0 / 448.0))[:, None]).double()
    step = torch.exp2(torch.clamp(torch.frexp(u).exponent - 1, min=-6).double() - 3.0)
    assert int(((u / step).abs() % 1 == 0.5).sum()) > 50


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 3584), (24, 1536), (600, 96), (7, 1001), (3, 9001), (4, 40000), (320, 18944), (2, 1)])
def test_quantize_is_the_elementary_operations(dtype, shape):
    """Bit by bit (zeros of either sign are one number), as `from_tensor` on either device."""
    from llm_inference_b200.csrc.library import kernels

    torch.manual_seed(41)
    x = torch.randn(shape, device="cuda").to(dtype)
    if shape[0] > 2:
        x[1] *= 1e-38
        x[2] *= 1e36
    if shape[0] > 20:
        x[3] *= 1e-30
        x[4] = 0.0
        x[5, 7], x[6, 8], x[6, 9] = math.nan, math.inf, -math.inf
        x[7] = math.nan
        x[8] *= 1e30
        x[9] *= 2.0**-120
        x[10] = torch.arange(shape[1], device="cuda").to(dtype)  # whole numbers: exact quotients
        x[11] = 448.0
    out = float8.quantize(make_ctx(kernels(), positions=[0]), x, float8.empty_rows(*shape, "cuda:0"))
    same_numbers(out, *elementary(x))
    x = x[~torch.isnan(x).any(1)]
    same_numbers(float8.from_tensor(x), *elementary(x))
    same_numbers(float8.from_tensor(x.cpu()), *elementary(x))


@gpu
def test_quantize_beside_every_middle():
    """Rows whose largest number is any, and whose others are the products of its scale with the middles between e4m3 numbers, one or two steps to either side."""
    from llm_inference_b200.csrc.library import kernels

    torch.manual_seed(42)
    rows = 4096
    most = torch.rand(rows, 1, device="cuda") + 1.0
    most[:64] = torch.linspace(1.0, 2.0, 64, device="cuda")[:, None]
    most = most * torch.exp2(torch.randint(-90, 90, (rows, 1), device="cuda").float())
    scale = most * (1.0 / 448.0)
    numbers = torch.arange(0, 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).float()
    middles = (numbers[1:] + numbers[:-1]) / 2  # 5 bits: their products with a scale are rounded once
    near = (middles * scale).view(torch.int32)[:, :, None] + torch.arange(-2, 3, dtype=torch.int32, device="cuda")
    x = torch.cat([near.view(torch.float32).reshape(rows, -1), most], dim=1).contiguous()
    x = torch.where(x.abs() > most, most, x)
    out = float8.quantize(make_ctx(kernels(), positions=[0]), x, float8.empty_rows(*x.shape, "cuda:0"))
    same_numbers(out, *elementary(x))


def test_from_tensor_keeps_a_nan_in_its_place():
    """As `quantize` does: the row's other numbers and its scale are what they would be beside a zero."""
    torch.manual_seed(43)
    w = torch.randn(6, 80)
    clean = w.clone()
    clean[1, 5] = clean[2, 3] = clean[2, 70] = 0.0
    w[1, 5] = w[2, 3] = w[2, 70] = math.nan
    w[3] = math.nan
    w[4, 9], w[4, 10] = math.inf, math.nan
    rows, beside = float8.from_tensor(w), float8.from_tensor(clean)
    same_numbers(rows, *elementary(w))
    assert torch.equal(rows.scales[:3], beside.scales[:3]) and torch.equal(rows.scales[5:], beside.scales[5:])
    q = rows.values.float()
    assert torch.isnan(q).nonzero().tolist() == [[1, 5], [2, 3], [2, 70], *([3, i] for i in range(80)), [4, 9], [4, 10]]
    assert torch.equal(q[:3].nan_to_num(), beside.values.float()[:3]) and float(rows.scales[3]) == 2.0**-126 and math.isinf(float(rows.scales[4]))


def test_from_tensor_of_a_parameter_has_no_gradients():
    """Weights laid out are numbers only: no graph that holds their 32-bit copies."""
    torch.manual_seed(44)
    weight = torch.nn.Parameter(torch.randn(5, 40))
    rows = float8.from_tensor(weight)
    assert not rows.scales.requires_grad and rows.scales.grad_fn is None and not rows.values.requires_grad and rows.values.grad_fn is None
    same_numbers(rows, *elementary(weight.detach()))
