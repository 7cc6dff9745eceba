"""Matrices in 8 bits: rows of e4m3 numbers with a 32-bit scale each, and a decoder layer's operators over them.

``rmsnorm`` and ``quantize`` make rows in 8 bits, ``linear`` and ``linear_gated`` multiply them on the tensor cores at twice the rate and
half the bytes of bfloat16. Like the functions of :mod:`.ops` each checks its operands (:class:`KernelError`), launches on the current
stream of the step's device and writes into tensors that it is handed. The kernels are ``csrc/kernels/float8_rows.cu`` and
``gemm_float8*.cu``. There are no gradients: the engine does not train.
"""

from __future__ import annotations

from dataclasses import dataclass
from struct import Struct

import torch

from ..csrc.library import DTYPE_CODES, KernelError
from .context import StepContext

LARGEST = 448.0  # of e4m3
PER_LARGEST = 1.0 / LARGEST  # scales are products with it, rounded to 32 bits, on every device (the tensor library divides by a number in its own way on each)
SMALLEST_SCALE = 2.0**-126
ROW_BYTES = 16  # rows start on multiples of this
MOST = 2**30  # rows, columns

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
    """A weight matrix in 8 bits, laid out once, before any step: torch operations on the weight's own device, which have ended when this returns. The
    numbers are :func:`quantize`'s, a NaN in its place too."""
    if weight.dim() != 2:
        raise KernelError(f"float8: a matrix has two dimensions, not {weight.dim()}")
    out = empty_rows(*weight.shape, weight.device)
    for at in range(0, weight.shape[0], 4096):  # bounds the 32-bit copies
        rows = weight[at : at + 4096].detach().float()
        largest = torch.nan_to_num(rows.abs(), nan=0.0, posinf=torch.inf)  # a NaN counts for nothing beside a number
        scales = torch.clamp(largest.amax(1) * PER_LARGEST, min=SMALLEST_SCALE) if rows.shape[1] else torch.full_like(out.scales[at : at + 4096], SMALLEST_SCALE)
        out.scales[at : at + 4096] = scales
        out.values[at : at + 4096] = (rows / scales[:, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    if weight.is_cuda:
        torch.cuda.current_stream(weight.device).synchronize()
    out.constant = True
    return out


# Operands are checked with as few trips into the tensor library as it takes: a decode step makes a hundred of these calls, and one of
# them costs the device a few microseconds only.
_E4M3, _F32, _BF16 = torch.float8_e4m3fn, torch.float32, torch.bfloat16
_BOTH = {_F32: DTYPE_CODES[_F32], _BF16: DTYPE_CODES[_BF16]}
_ONLY_F32 = {_F32: DTYPE_CODES[_F32]}
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _device_index(ctx: StepContext) -> int:
    device = ctx.device
    if device.index is not None:
        return device.index
    return -1 if device.type == "cpu" else _current_device()


def _rows(name: str, m: Float8Rows, index: int) -> tuple[int, int, int, int, int]:
    """Checks rows in 8 bits; their address and pitch, the scales' address, rows and columns."""
    v, s = m.values, m.scales
    if v.dim() == 2 and s.dim() == 1:
        rows, columns = v.shape
        pitch, step = v.stride()
        if rows <= 1 or columns == 0:
            pitch = -(-columns // ROW_BYTES) * ROW_BYTES
        address = v.data_ptr()
        if (v.dtype is _E4M3 and (step == 1 or columns <= 1) and not (address | pitch) % ROW_BYTES and pitch >= columns and v.get_device() == index
                and s.dtype is _F32 and s.numel() == rows and s.is_contiguous() and s.get_device() == index and rows <= MOST and columns <= MOST):
            return address, pitch, s.data_ptr(), rows, columns
    raise KernelError(f"float8: {name} must be e4m3 [rows, columns] whose rows are contiguous on 16-byte boundaries, with float32 [rows] scales, at most 2**30 of each, on "
                      f"{_device_name(index)}; got {v.dtype} {list(v.shape)} (strides {list(v.stride())}, {v.device}) and {s.dtype} {list(s.shape)} ({s.device})")


def _matrix(name: str, t: torch.Tensor, rows: int, columns: int, dtypes: dict[torch.dtype, int], index: int) -> tuple[int, int, int]:
    """Checks a matrix whose rows are contiguous, some distance apart; its address, that distance and its type's code."""
    code = dtypes.get(t.dtype)
    if code is not None and t.shape == (rows, columns) and t.get_device() == index:
        pitch, step = t.stride()
        if rows <= 1:
            pitch = -(-columns // 8) * 8
        if (step == 1 or columns <= 1) and pitch >= columns:
            return t.data_ptr(), pitch, code
    raise KernelError(f"float8: {name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)} {[rows, columns]} with contiguous rows on "
                      f"{_device_name(index)}; got {t.dtype} {list(t.shape)} (strides {list(t.stride())}, {t.device})")


def _vector(name: str, t: torch.Tensor, count: int, index: int) -> int:
    if t.dtype is _F32 and t.dim() == 1 and t.numel() == count and t.is_contiguous() and t.get_device() == index:
        return t.data_ptr()
    raise KernelError(f"float8: {name} must be float32 [{count}] on {_device_name(index)}; got {t.dtype} {list(t.shape)} ({t.device})")


def _device_name(index: int) -> str:
    return "cpu" if index < 0 else f"cuda:{index}"


# A call's numbers travel as one block (the structs of the same names in csrc/kernels): one argument each took 4 us a product.
_pack_quantize = Struct("8q").pack
_pack_rmsnorm = Struct("13qd").pack
_pack_linear = Struct("19q").pack


def _refuse_host(index: int) -> None:
    if index < 0:
        raise KernelError("float8: the operands lie in host memory, and there are kernels for the GPU only")


def _call(ctx: StepContext, index: int, name: str, block: bytes) -> None:
    """Launches on the step's device, whichever is current."""
    if _current_device() == index:
        ctx.lib.call(name, block, ctx.stream)
    else:
        with torch.cuda.device(index):
            ctx.lib.call(name, block, ctx.stream)


def quantize(ctx: StepContext, x: torch.Tensor, out: Float8Rows) -> Float8Rows:
    """``out`` = the rows of ``x`` (float32 or bfloat16, rows contiguous) in 8 bits: ``scale = max(max |row| * (1 / 448), 2**-126)``, the quotients by it
    rounded to 32 bits and those to the nearest e4m3 number (ties to even): the numbers that elementary 32-bit operations make, and :func:`from_tensor`.
    NaN stays in its place; a row with an infinity has scale infinity, zeros and NaN."""
    index = _device_index(ctx)
    o, o_pitch, scales, rows, columns = _rows("out", out, index)
    if columns == 0:
        raise KernelError("float8: rows without numbers have no scale")
    x_at, x_pitch, code = _matrix("x", x, rows, columns, _BOTH, index)
    _refuse_host(index)
    _call(ctx, index, "b200_float8_quantize", _pack_quantize(x_at, code, x_pitch, o, o_pitch, scales, rows, columns))
    return out


def rmsnorm(ctx: StepContext, x: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float, out: Float8Rows,
            stream: torch.Tensor | None = None) -> Float8Rows:
    """``s = x + delta`` and ``out`` = the rows ``s * rsqrt(mean(s^2) + eps) * weight`` in 8 bits, nearest but for 32-bit rounding: a quotient within 2^-21 of
    the middle between two e4m3 numbers may go to either. ``s * weight`` has to be in the range of 32 bits. ``x`` is the 32-bit residual stream;
    the sum goes to ``stream``, by default back into ``x`` (with no ``delta`` nothing is written unless ``stream`` is given)."""
    index = _device_index(ctx)
    o, o_pitch, scales, rows, columns = _rows("out", out, index)
    if columns == 0:
        raise KernelError("float8: rows without numbers have no scale")
    x_at, x_pitch, _ = _matrix("x", x, rows, columns, _ONLY_F32, index)
    d_at, d_pitch, code = (0, 0, 0) if delta is None else _matrix("delta", delta, rows, columns, _BOTH, index)
    if stream is not None:
        s_at, s_pitch, _ = _matrix("stream", stream, rows, columns, _ONLY_F32, index)
    else:
        s_at, s_pitch = (0, 0) if delta is None else (x_at, x_pitch)
    w_at = _vector("the norm's weight", weight, columns, index)
    _refuse_host(index)
    _call(ctx, index, "b200_float8_rmsnorm", _pack_rmsnorm(x_at, x_pitch, d_at, code, d_pitch, w_at, s_at, s_pitch, o, o_pitch, scales, rows, columns, eps))
    return out


def _product(ctx: StepContext, x: Float8Rows, weight: Float8Rows, out: torch.Tensor, bias, residual, kind: int, activation: int) -> torch.Tensor:
    index = _device_index(ctx)
    x_at, x_pitch, x_scales, m, k = _rows("x", x, index)
    w_at, w_pitch, w_scales, n, inner = _rows("weight", weight, index)
    if k != inner or k == 0:
        raise KernelError(f"float8: x is {[m, k]} but weight is {[n, inner]}")
    if kind == _GATED and n % 2:
        raise KernelError(f"float8: gate and up rows come in pairs, weight has {n} rows")
    o, o_pitch, code = _matrix("out", out, m, n // 2 if kind == _GATED else n, _BOTH, index)
    b = 0 if bias is None else _vector("bias", bias, n, index)
    r, r_pitch, _ = (0, 0, 0) if residual is None else _matrix("residual", residual, m, n, _ONLY_F32, index)
    _refuse_host(index)
    if m and n:
        _call(ctx, index, "b200_float8_linear", _pack_linear(x_at, x_pitch, x_scales, w_at, w_pitch, w_scales, weight.constant, o, code, o_pitch, b, r, r_pitch,
                                                             m, n, k, kind, activation, ctx.err.data_ptr()))
    return out


_PLAIN, _ACTIVATED, _GATED = 0, 1, 2


def linear(ctx: StepContext, x: Float8Rows, weight: Float8Rows, out: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``out = act(x @ weight.T + bias) + residual`` in one kernel; ``weight`` is ``[out_features, in_features]``, ``out`` bfloat16 or float32 with
    contiguous rows, ``bias`` float32, ``activation`` None, ``"silu"``, ``"gelu"`` (tanh form) or ``"squared_relu"``, ``residual`` float32 (it may be
    ``out`` itself). Sums are 32-bit and rounded once on the way out. The tensor cores add toward zero, in chains that are bounded: a sum of terms of one sign
    comes out smaller by up to 4.5e-6 of itself in float32, by less than a hundredth of the output's own rounding in bfloat16; of both signs, by a tenth of that.
    The inner size is at most 2**28."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise KernelError(f"float8: no activation {activation!r} (there are {', '.join(str(a) for a in ACTIVATIONS)})")
    return _product(ctx, x, weight, out, bias, residual, _ACTIVATED if code else _PLAIN, code)


def linear_gated(ctx: StepContext, x: Float8Rows, weight: Float8Rows, out: torch.Tensor, activation: str = "silu", bias: torch.Tensor | None = None) -> torch.Tensor:
    """``out = act(gate) * up`` of ``x @ weight.T + bias`` with interleaved gate/up rows (row 2j is gate_j, row 2j + 1 up_j): both projections, the
    activation (``"silu"`` or ``"gelu"``) and the product in one kernel."""
    if activation not in GATED_ACTIVATIONS:
        raise KernelError(f"float8: no gated activation {activation!r} (there are {', '.join(GATED_ACTIVATIONS)})")
    return _product(ctx, x, weight, out, bias, None, _GATED, ACTIVATIONS[activation])
