"""Matrices in 8 bits: rows of e4m3 numbers with a 32-bit scale each, and a decoder layer's operators over them.

``rmsnorm`` and ``quantize`` make rows in 8 bits, ``linear`` and ``linear_gated`` multiply them on the tensor cores at twice the rate and
half the bytes of bfloat16. Like the functions of :mod:`.ops` each checks its operands (:class:`KernelError`), launches on the current
stream of the step's device and writes into tensors that it is handed. The kernels are ``csrc/kernels/float8_rows.cu`` and
``gemm_float8*.cu``. There are no gradients: the engine does not train.
"""

from __future__ import annotations

from ctypes import c_float, c_int, c_int64
from dataclasses import dataclass

import torch

from ..csrc.library import DTYPE_CODES, KernelError, ptr
from .context import StepContext

LARGEST = 448.0  # of e4m3
SMALLEST_SCALE = 2.0**-126
ROW_BYTES = 16  # rows start on multiples of this

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "squared_relu": 3}  # gelu in its tanh form
GATED_ACTIVATIONS = ("silu", "gelu")


@dataclass
class Float8Rows:
    """The matrix ``values * scales[:, None]``: ``values`` is ``[rows, columns]`` e4m3 (``torch.float8_e4m3fn``) whose rows are contiguous and start
    on 16-byte boundaries, ``scales`` float32 ``[rows]``. ``constant`` promises that nothing still running on the stream writes it (weights laid out
    before the step): a product may then fetch it before the kernel in front has ended."""

    values: torch.Tensor
    scales: torch.Tensor
    constant: bool = False

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.values.shape)

    @property
    def row_stride(self) -> int:
        """Bytes from row to row (of a single row: what they would be)."""
        rows, columns = self.values.shape
        return self.values.stride(0) if rows > 1 else -(-columns // ROW_BYTES) * ROW_BYTES

    def bytes(self) -> int:
        return self.values.numel() + 4 * self.scales.numel()

    def dequantized(self) -> torch.Tensor:
        """The numbers themselves, in 32 bits."""
        return self.values.float() * self.scales[:, None]


def empty_rows(rows: int, columns: int, device: torch.device | str) -> Float8Rows:
    """Room for a matrix in 8 bits."""
    held = torch.empty(rows, -(-columns // ROW_BYTES) * ROW_BYTES, dtype=torch.float8_e4m3fn, device=device)
    return Float8Rows(held[:, :columns], torch.empty(rows, dtype=torch.float32, device=device))


def buffer_rows(ctx: StepContext, name: str, rows: int, columns: int) -> Float8Rows:
    """The same out of the step's workspace."""
    pitch = -(-columns // ROW_BYTES) * ROW_BYTES
    held = ctx.buffer(name, (rows, pitch), torch.float8_e4m3fn)
    return Float8Rows(held if pitch == columns else held[:, :columns], ctx.buffer(name + "_scales", (rows,), torch.float32))


def from_tensor(weight: torch.Tensor) -> Float8Rows:
    """A weight matrix in 8 bits, laid out once (torch operations on the weight's own device; nothing of a step)."""
    if weight.dim() != 2:
        raise KernelError(f"float8: a matrix has two dimensions, not {weight.dim()}")
    out = empty_rows(*weight.shape, weight.device)
    for at in range(0, weight.shape[0], 4096):  # bounds the 32-bit copies
        rows = weight[at : at + 4096].float()
        scales = torch.clamp(rows.abs().amax(1) / LARGEST, min=SMALLEST_SCALE) if rows.shape[1] else torch.full_like(out.scales[at : at + 4096], SMALLEST_SCALE)
        out.scales[at : at + 4096] = scales
        out.values[at : at + 4096] = (rows / scales[:, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    out.constant = True
    return out


def _need(cond: bool, message: str) -> None:
    if not cond:
        raise KernelError(message)


def _need_rows(name: str, m: Float8Rows, device: torch.device) -> None:
    v, s = m.values, m.scales
    if (v.dtype == torch.float8_e4m3fn and v.dim() == 2 and (v.stride(1) == 1 or v.shape[1] <= 1) and v.device == device and v.data_ptr() % ROW_BYTES == 0
            and (v.shape[0] <= 1 or (v.stride(0) % ROW_BYTES == 0 and v.stride(0) >= v.shape[1]))
            and s.dtype == torch.float32 and s.shape == v.shape[:1] and s.is_contiguous() and s.device == device):
        return
    _need(False, f"float8: {name} must be e4m3 [rows, columns] whose rows are contiguous on 16-byte boundaries, with float32 [rows] scales, on {device}; "
                 f"got {v.dtype} {list(v.shape)} (strides {list(v.stride())}, {v.device}) and {s.dtype} {list(s.shape)} ({s.device})")


def _need_matrix(name: str, t: torch.Tensor, shape: tuple[int, int], dtypes: tuple[torch.dtype, ...], device: torch.device) -> int:
    """Checks a matrix with contiguous rows, some distance apart; returns that distance."""
    if t.dtype not in dtypes or tuple(t.shape) != shape or t.device != device or (t.stride(1) != 1 and shape[1] > 1) or (shape[0] > 1 and t.stride(0) < shape[1]):
        _need(False, f"float8: {name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)} {list(shape)} with contiguous rows on {device}; "
                     f"got {t.dtype} {list(t.shape)} (strides {list(t.stride())}, {t.device})")
    return t.stride(0) if shape[0] > 1 else -(-shape[1] // 8) * 8


_BOTH = (torch.float32, torch.bfloat16)
_F32 = (torch.float32,)


def _call(ctx: StepContext, name: str, *args) -> None:
    """Launches on the step's device, whichever is current."""
    if torch.cuda.current_device() == ctx.device.index or ctx.device.index is None:
        ctx.lib.call(name, *args, ctx.stream)
    else:
        with torch.cuda.device(ctx.device):
            ctx.lib.call(name, *args, ctx.stream)


def _need_size(*sizes: int) -> None:
    _need(all(s < 2**31 for s in sizes), "float8: rows and columns are counted in 31 bits")


def quantize(ctx: StepContext, x: torch.Tensor, out: Float8Rows) -> Float8Rows:
    """``out`` = the rows of ``x`` (float32 or bfloat16, rows contiguous) in 8 bits: ``scale = max(max |row| / 448, 2**-126)``, numbers over it
    rounded to the nearest (ties to even). NaN stays in its place; a row with an infinity has scale infinity, zeros and NaN."""
    rows, columns = out.shape
    _need(columns > 0, "float8: rows without numbers have no scale")
    _need_rows("out", out, x.device)
    stride = _need_matrix("x", x, out.shape, _BOTH, ctx.device)
    _need_size(rows, columns)
    _call(ctx, "b200_float8_quantize", ptr(x), c_int(DTYPE_CODES[x.dtype]), c_int64(stride), ptr(out.values), c_int64(out.row_stride), ptr(out.scales),
          c_int(rows), c_int(columns))
    return out


def rmsnorm(ctx: StepContext, x: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float, out: Float8Rows,
            stream: torch.Tensor | None = None) -> Float8Rows:
    """``s = x + delta`` and ``out`` = the rows ``s * rsqrt(mean(s^2) + eps) * weight`` in 8 bits (:func:`quantize`). ``x`` is the 32-bit residual stream;
    the sum goes to ``stream``, by default back into ``x`` (with no ``delta`` nothing is written unless ``stream`` is given)."""
    rows, columns = out.shape
    _need(columns > 0, "float8: rows without numbers have no scale")
    _need_rows("out", out, x.device)
    x_stride = _need_matrix("x", x, out.shape, _F32, ctx.device)
    delta_stride = _need_matrix("delta", delta, out.shape, _BOTH, ctx.device) if delta is not None else 0
    if stream is None and delta is not None:
        stream = x
    stream_stride = _need_matrix("stream", stream, out.shape, _F32, ctx.device) if stream is not None else 0
    _need(weight.dtype == torch.float32 and weight.shape == (columns,) and weight.is_contiguous() and weight.device == ctx.device,
          "float8: the norm's weight must be float32 [columns]")
    _need_size(rows, columns)
    _call(ctx, "b200_float8_rmsnorm", ptr(x), c_int64(x_stride), ptr(delta), c_int(DTYPE_CODES[delta.dtype] if delta is not None else 0), c_int64(delta_stride),
          ptr(weight), c_float(eps), ptr(stream), c_int64(stream_stride), ptr(out.values), c_int64(out.row_stride), ptr(out.scales), c_int(rows), c_int(columns))
    return out


def _product(ctx: StepContext, x: Float8Rows, weight: Float8Rows, out: torch.Tensor, width: int, bias, residual, kind: int, activation: str | None) -> torch.Tensor:
    _need_rows("x", x, ctx.device)
    _need_rows("weight", weight, ctx.device)
    (m, k), (n, inner) = x.shape, weight.shape
    _need(k == inner and k > 0, f"float8: x is {[m, k]} but weight is {[n, inner]}")
    _need_size(m, n, k)
    out_stride = _need_matrix("out", out, (m, width), _BOTH, ctx.device)
    _need(bias is None or (bias.dtype == torch.float32 and bias.shape == (n,) and bias.is_contiguous() and bias.device == ctx.device),
          f"float8: bias must be float32 [{n}]")
    residual_stride = _need_matrix("residual", residual, (m, n), _F32, ctx.device) if residual is not None else 0
    if m == 0 or n == 0:
        return out
    _call(ctx, "b200_float8_linear", ptr(x.values), c_int64(x.row_stride), ptr(x.scales), ptr(weight.values), c_int64(weight.row_stride), ptr(weight.scales),
          c_int(int(weight.constant)), ptr(out), c_int(DTYPE_CODES[out.dtype]), c_int64(out_stride), ptr(bias), ptr(residual), c_int64(residual_stride),
          c_int(m), c_int(n), c_int(k), c_int(kind), c_int(ACTIVATIONS[activation]), ptr(ctx.err))
    return out


def linear(ctx: StepContext, x: Float8Rows, weight: Float8Rows, out: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``out = act(x @ weight.T + bias) + residual`` in one kernel; ``weight`` is ``[out_features, in_features]``, ``out`` bfloat16 or float32 with
    contiguous rows, ``bias`` float32, ``activation`` None, ``"silu"``, ``"gelu"`` (tanh form) or ``"squared_relu"``, ``residual`` float32 (it may be
    ``out`` itself). Sums are 32-bit and rounded once on the way out."""
    _need(activation in ACTIVATIONS, f"float8: no activation {activation!r} (there are {', '.join(str(a) for a in ACTIVATIONS)})")
    return _product(ctx, x, weight, out, weight.shape[0], bias, residual, 0 if activation is None else 1, activation)


def linear_gated(ctx: StepContext, x: Float8Rows, weight: Float8Rows, out: torch.Tensor, activation: str = "silu", bias: torch.Tensor | None = None) -> torch.Tensor:
    """``out = act(gate) * up`` of ``x @ weight.T + bias`` with interleaved gate/up rows (row 2j is gate_j, row 2j + 1 up_j): both projections, the
    activation (``"silu"`` or ``"gelu"``) and the product in one kernel."""
    _need(activation in GATED_ACTIVATIONS, f"float8: no gated activation {activation!r} (there are {', '.join(GATED_ACTIVATIONS)})")
    n = weight.shape[0]
    _need(n % 2 == 0, f"float8: gate and up rows come in pairs, weight has {n} rows")
    return _product(ctx, x, weight, out, n // 2, bias, None, 2, activation)
