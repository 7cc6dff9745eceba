"""Products right behind the kernel that makes their operands, in each of the product's forms."""

from __future__ import annotations

import pytest
import torch

from test_kernels import make_ctx
from llm_inference_b200.parts import float8

gpu = pytest.mark.gpu

# `mma.sync`; weights streamed past few tokens, by single blocks and by clusters; tiles.
FORMS = [(4, 4096, 4096), (16, 37888, 3584), (64, 5120, 5120), (777, 4096, 4096)]


@gpu
@pytest.mark.parametrize("m,n,k", FORMS)
def test_weights_come_from_the_kernel_in_front(m, n, k):
    """Weights that nobody promised constant are waited for, whichever form takes the call."""
    from llm_inference_b200.csrc.library import kernels

    torch.manual_seed(60)
    ctx = make_ctx(kernels(), positions=[0])
    x = float8.from_tensor(torch.randn(m, k, device="cuda"))
    sources = [torch.randn(n, k, device="cuda") * 0.05 for _ in range(2)]
    want = []
    for source in sources:
        w = float8.quantize(ctx, source, float8.empty_rows(n, k, "cuda:0"))
        torch.cuda.synchronize()
        want.append(float8.linear(ctx, x, w, torch.empty(m, n, device="cuda", dtype=torch.bfloat16)))
        torch.cuda.synchronize()
    w = float8.empty_rows(n, k, "cuda:0")
    outs = [torch.empty(m, n, device="cuda", dtype=torch.bfloat16) for _ in range(12)]
    for turn, out in enumerate(outs):
        float8.quantize(ctx, sources[turn % 2], w)
        float8.linear(ctx, x, w, out)
    for turn, out in enumerate(outs):
        assert torch.equal(out, want[turn % 2])
    assert int(ctx.err.item()) == 0


@gpu
@pytest.mark.parametrize("m,n,k", FORMS)
def test_tokens_come_from_the_kernel_in_front(m, n, k):
    """Weights promised constant are fetched ahead; the tokens, their scales and the residual are not."""
    from llm_inference_b200.csrc.library import kernels

    torch.manual_seed(61)
    ctx = make_ctx(kernels(), positions=[0])
    w = float8.from_tensor(torch.randn(n, k, device="cuda") * 0.05)
    sources = [torch.randn(m, k, device="cuda") * s for s in (1.0, 3.0)]
    want = []
    for source in sources:
        rows = float8.quantize(ctx, source, float8.empty_rows(m, k, "cuda:0"))
        torch.cuda.synchronize()
        want.append(float8.linear(ctx, rows, w, torch.empty(m, n, device="cuda")))
        torch.cuda.synchronize()
    rows = float8.empty_rows(m, k, "cuda:0")
    outs = [torch.empty(m, n, device="cuda") for _ in range(12)]
    for turn, out in enumerate(outs):
        float8.quantize(ctx, sources[turn % 2], rows)
        float8.linear(ctx, rows, w, out)
    for turn, out in enumerate(outs):
        assert torch.equal(out, want[turn % 2])
    # Out of one product into the next one's residual.
    for turn in range(6):
        stream = float8.linear(ctx, rows, w, torch.empty(m, n, device="cuda"))
        float8.linear(ctx, rows, w, stream, residual=stream)
        assert torch.equal(stream, 2 * want[1])
    assert int(ctx.err.item()) == 0
