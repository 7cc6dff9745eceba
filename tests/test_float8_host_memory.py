"""Operands in host memory never reach a kernel."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from llm_inference_b200.csrc.library import KernelError
from llm_inference_b200.parts import float8


class Launches:
    """Stands in for the kernel library: remembers what would have been launched."""

    def __init__(self) -> None:
        self.names: list[str] = []

    def call(self, name: str, *args) -> None:
        self.names.append(name)


@pytest.mark.parametrize("rows", [0, 4])
def test_a_context_of_the_host_is_refused(rows):
    """Operands that fit each other and their context in every way, but lie where no kernel can read them."""
    lib = Launches()
    ctx = SimpleNamespace(device=torch.device("cpu"), lib=lib, stream=0, err=torch.zeros(1, dtype=torch.int32))
    x, weight = torch.zeros(rows, 48), torch.ones(48)
    rows8, w = float8.empty_rows(rows, 48, "cpu"), float8.from_tensor(torch.ones(6, 48))
    calls = [
        lambda: float8.quantize(ctx, x, rows8),
        lambda: float8.rmsnorm(ctx, x, None, weight, 1e-6, rows8),
        lambda: float8.rmsnorm(ctx, x, x.bfloat16(), weight, 1e-6, rows8, stream=torch.zeros(rows, 48)),
        lambda: float8.linear(ctx, rows8, w, torch.zeros(rows, 6), bias=torch.zeros(6), residual=torch.zeros(rows, 6)),
        lambda: float8.linear_gated(ctx, rows8, w, torch.zeros(rows, 3)),
    ]
    for call in calls:
        with pytest.raises(KernelError, match="host memory"):
            call()
    assert lib.names == []
