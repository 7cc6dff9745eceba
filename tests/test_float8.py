"""The 8-bit operators against plain 64-bit forms, and their refusals.

Tolerances. A product of two e4m3 numbers is exact in 32 bits; sums on the tensor core drop what lies below the last bit of 32-bit numbers, so one
addition is off by at most 2^-23 of the sum of magnitudes A = sum |x w| that it belongs to, and the 32 products of an instruction by 32 half
steps of the largest of them; chains are counted from above. e4m3 rounds by at most 2^-4 of a number (half a step), which the tests take as the step itself where
they check that the nearest was taken."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from test_kernels import make_ctx
from llm_inference_b200.csrc.library import KernelError
from llm_inference_b200.parts import float8

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from llm_inference_b200.csrc.library import kernels

    return kernels()


def e4m3_step(u: torch.Tensor) -> torch.Tensor:
    """Distance of e4m3 numbers around u (64 bits)."""
    return torch.exp2(torch.clamp(torch.frexp(u).exponent - 1, min=-6).double() - 3.0)


def check_rows(out: float8.Float8Rows, v: torch.Tensor, scale_off: float, quotient_off: float) -> None:
    """``out`` holds the rows v (64 bits): scales to ``scale_off``, each number the nearest e4m3 one to v / scale, which itself may be off by
    ``quotient_off`` (both relative)."""
    scales = torch.clamp(v.abs().amax(1) / 448.0, min=2.0**-126)
    assert torch.all((out.scales.double() - scales).abs() <= scale_off * scales)
    u = v / scales[:, None]
    assert torch.all((out.values.double() - u).abs() <= e4m3_step(u) / 2 + quotient_off * u.abs())


# --- rows in 8 bits --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 16), (5, 1001), (1, 8192), (700, 64), (2500, 200), (4, 40000), (3, 9001), (320, 18944)])
def test_from_tensor_is_the_nearest(dtype, shape):
    torch.manual_seed(3)
    w = (torch.randn(shape) * 0.02).to(dtype)
    rows = float8.from_tensor(w)
    assert rows.constant and rows.shape == shape and rows.values.data_ptr() % 16 == 0 and (shape[0] == 1 or rows.values.stride(0) % 16 == 0)
    check_rows(rows, w.double(), 2.0**-23, 2.0**-22)
    torch.testing.assert_close(rows.dequantized().double(), w.double(), rtol=2.0**-4 + 2.0**-20, atol=float(w.abs().max()) * 2.0**-9 / 448)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(0, 64), (1, 1), (1, 3584), (3, 16), (5, 1001), (1, 8192), (700, 64), (2500, 200), (4, 40000), (3, 9001), (320, 18944)])
def test_quantize(lib, dtype, shape):
    torch.manual_seed(4)
    x = (torch.randn(shape, device="cuda") * torch.rand(shape[0], 1, device="cuda") * 5).to(dtype)
    if shape[0] > 2:
        x[1] = 0.0  # a padding row
    out = float8.empty_rows(*shape, "cuda:0")
    ctx = make_ctx(lib, positions=[0])
    assert float8.quantize(ctx, x, out) is out
    if shape[0]:
        check_rows(out, x.double(), 2.0**-23, 2.0**-22)
    if shape[0] > 2:
        assert torch.all(out.values[1].float() == 0) and float(out.scales[1]) == 2.0**-126


@gpu
def test_quantize_ends_of_the_range(lib):
    """Tiny, huge, infinite and missing numbers; the rows beside them are as always."""
    torch.manual_seed(5)
    x = torch.randn(8, 96, device="cuda")
    plain = x.clone()
    x[1] *= 1e-38  # amax / 448 is below the smallest scale
    x[2] = 1e-45
    x[3] *= 1e38 / float(x[3].abs().max())
    x[4, 7] = math.inf
    x[5, 9] = math.nan
    x[6, 3], x[6, 5] = math.inf, -math.inf
    out = float8.quantize(make_ctx(lib, positions=[0]), x, float8.empty_rows(8, 96, "cuda:0"))
    q, s = out.values.float(), out.scales
    pick = [0, 1, 2, 3, 7]
    check_rows(float8.Float8Rows(out.values[pick], s[pick]), x[pick].double(), 2.0**-23, 2.0**-21)
    assert torch.equal(x[[0, 7]], plain[[0, 7]])
    assert math.isinf(float(s[4])) and torch.isnan(q[4, 7]) and torch.all(q[4, :7] == 0) and torch.all(q[4, 8:] == 0)
    assert torch.isnan(q[5, 9]) and int(torch.isnan(q[5]).sum()) == 1 and math.isfinite(float(s[5]))
    assert torch.isnan(q[6, 3]) and torch.isnan(q[6, 5]) and int(torch.isnan(q[6]).sum()) == 2


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_odd_strides(lib, dtype):
    """Columns of a wider matrix, starting anywhere; what lies beside the output rows stays as it was."""
    torch.manual_seed(6)
    wide = torch.randn(40, 203, device="cuda").to(dtype)
    for first, count in ((0, 128), (1, 128), (8, 64), (3, 200)):
        x = wide[:, first : first + count]
        held = torch.full((42, 256), 0x55, dtype=torch.uint8, device="cuda")
        out = float8.Float8Rows(held.view(torch.float8_e4m3fn)[1:41, 16 : 16 + count], torch.empty(40, device="cuda"))
        float8.quantize(make_ctx(lib, positions=[0]), x, out)
        check_rows(out, x.double(), 2.0**-23, 2.0**-22)
        beside = held.clone()
        beside[1:41, 16 : 16 + count] = 0x55
        assert torch.all(beside == 0x55)


@gpu
@pytest.mark.parametrize("delta", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(0, 64), (1, 1), (1, 3584), (37, 1001), (5, 8200), (600, 96), (2500, 200), (3, 40000), (2, 9001)])
def test_rmsnorm(lib, delta, shape):
    torch.manual_seed(7)
    rows, columns = shape
    eps = 1e-6
    x = torch.randn(shape, device="cuda") * (1 + 30 * (torch.rand(columns, device="cuda") < 0.01))
    d = torch.randn(shape, device="cuda").to(delta) if delta is not None else None
    weight = 1 + 0.2 * torch.randn(columns, device="cuda")
    ctx = make_ctx(lib, positions=[0])
    out, before = float8.empty_rows(rows, columns, "cuda:0"), x.clone()
    apart = torch.empty_like(x)
    float8.rmsnorm(ctx, x, d, weight, eps, out, stream=apart)
    s = before if d is None else before + d.float()
    assert torch.equal(x, before) and torch.equal(apart, s)
    if rows == 0:
        return
    v = s.double()
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * weight.double()
    # Squares add up in chains of at most columns / 1,024 * 8 + 50 additions of 2^-24, half of which reaches the root; the root itself 2^-22.
    off = (columns / 128 + 50) * 2.0**-25 + 2.0**-21
    check_rows(out, v, off, 2.0**-21)
    again = float8.empty_rows(rows, columns, "cuda:0")
    float8.rmsnorm(ctx, x, d, weight, eps, again)  # into the stream itself
    assert torch.equal(x, s) and torch.equal(again.values.view(torch.uint8), out.values.view(torch.uint8)) and torch.equal(again.scales, out.scales)


@gpu
def test_rmsnorm_ends_of_the_range(lib):
    torch.manual_seed(8)
    x = torch.randn(7, 256, device="cuda")
    x[1] = 0.0
    x[2] *= 1e-30
    x[3, 5] = math.inf
    x[4, 5] = math.nan
    x[5] *= 1e15
    weight = torch.ones(256, device="cuda")
    out = float8.rmsnorm(make_ctx(lib, positions=[0]), x, None, weight, 1e-6, float8.empty_rows(7, 256, "cuda:0"))
    pick = [0, 1, 2, 5, 6]
    v = x[pick].double()
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)
    check_rows(float8.Float8Rows(out.values[pick], out.scales[pick]), v, 2.0**-18, 2.0**-20)
    assert torch.isnan(out.dequantized()[3]).any() and torch.isnan(out.dequantized()[4]).all()


# --- products --------------------------------------------------------------------------------------


def operand(rows: int, columns: int, std: float = 1.0) -> float8.Float8Rows:
    return float8.from_tensor(torch.randn(rows, columns, device="cuda") * std)


def wide_product(x: float8.Float8Rows, w: float8.Float8Rows) -> tuple[torch.Tensor, torch.Tensor]:
    """(x w^T, the same of magnitudes) in 64 bits."""
    a = x.values.double() * x.scales.double()[:, None]
    b = w.values.double() * w.scales.double()[:, None]
    return a @ b.t(), a.abs() @ b.abs().t()


def sum_off(k: int, magnitudes: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What a sum may be off by: additions of 32 products in a chain (cut where outputs are 32-bit, at 10,240 of K), of chains and of
    cluster members (16), of an instruction's products, and four roundings of scales and bias."""
    chain = math.ceil(k / 32) if dtype == torch.bfloat16 else min(math.ceil(k / 32), 320) + math.ceil(k / 10240)
    return magnitudes * 2.0**-23 * (chain + 16 + 16 + 4)


def wide_activation(v: torch.Tensor, name: str | None) -> torch.Tensor:
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))
    if name == "squared_relu":
        return torch.clamp(v, min=0) ** 2
    return v


def slope(v: torch.Tensor, off: torch.Tensor, name: str | None) -> torch.Tensor:
    """What an argument that is off by ``off`` does to an activation: its slope is at most 1.13 (silu and gelu), of the square 2 (|v| + off). The
    functions themselves are good to 2^-20 of their argument."""
    if name == "squared_relu":
        return 2 * (v.abs() + off) * off + (v * v) * 2.0**-22
    return off if name is None else 1.13 * off + v.abs() * 2.0**-20


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


SIZES = [
    (1, 1, 1), (1, 4608, 3584), (2, 130, 31), (3, 127, 129), (16, 2048, 1536), (17, 1001, 1001), (33, 5, 16), (64, 5120, 5120), (65, 384, 4096), (129, 640, 896),
    (200, 1536, 8960), (257, 1001, 640), (300, 2048, 1536), (513, 256, 128), (777, 2050, 2048), (1500, 896, 4864), (2048, 3584, 1024), (8, 1536, 18944),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(lib, dtype, m, n, k):
    torch.manual_seed(m * 7 + n + k)
    x, w = operand(m, k), operand(n, k, 0.05)
    ctx = make_ctx(lib, positions=[0])
    out = float8.linear(ctx, x, w, torch.full((m, n), math.nan, device="cuda", dtype=dtype))
    y, magnitudes = wide_product(x, w)
    assert torch.all((out.double() - y).abs() <= sum_off(k, magnitudes, dtype) + half_step(dtype) * 1.01 * y.abs())
    assert int(ctx.err.item()) == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "squared_relu"])
@pytest.mark.parametrize("m,n,k", [(1, 384, 640), (24, 1000, 512), (100, 257, 1024), (700, 1026, 256)])
def test_linear_epilogue(lib, dtype, activation, m, n, k):
    torch.manual_seed(11)
    x, w = operand(m, k), operand(n, k, 0.05)
    bias, residual = torch.randn(n, device="cuda"), torch.randn(m, n, device="cuda") * 3
    ctx = make_ctx(lib, positions=[0])
    y, magnitudes = wide_product(x, w)
    for b in (None, bias):
        for r in (None, residual):
            out = float8.linear(ctx, x, w, torch.empty(m, n, device="cuda", dtype=dtype), bias=b, activation=activation, residual=r)
            z = y if b is None else y + b.double()
            off = sum_off(k, magnitudes + (0 if b is None else b.double().abs()), dtype)
            want = wide_activation(z, activation) + (0 if r is None else r.double())
            off = slope(z, off, activation) + (0 if r is None else r.double().abs() * 2.0**-23)
            assert torch.all((out.double() - want).abs() <= off + half_step(dtype) * 1.01 * want.abs()), (b is None, r is None)
    into = residual.clone()  # the stream is its own residual and output
    assert float8.linear(ctx, x, w, into, residual=into) is into
    apart = float8.linear(ctx, x, w, torch.empty_like(into), residual=residual)
    assert torch.equal(into, apart)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("m,width,k", [(1, 1, 16), (1, 9472, 3584), (7, 65, 130), (48, 2240, 1536), (130, 320, 896), (500, 513, 1001), (1030, 1024, 512)])
def test_linear_gated(lib, dtype, activation, m, width, k):
    torch.manual_seed(12)
    x, w = operand(m, k), operand(2 * width, k, 0.05)
    ctx = make_ctx(lib, positions=[0])
    y, magnitudes = wide_product(x, w)
    for bias in (None, torch.randn(2 * width, device="cuda")):
        out = float8.linear_gated(ctx, x, w, torch.empty(m, width, device="cuda", dtype=dtype), activation, bias=bias)
        z = y if bias is None else y + bias.double()
        off = sum_off(k, magnitudes + (0 if bias is None else bias.double().abs()), dtype)
        g, u, og, ou = z[:, 0::2], z[:, 1::2], off[:, 0::2], off[:, 1::2]
        a, oa = wide_activation(g, activation), slope(g, og, activation)
        want = a * u
        limit = oa * (u.abs() + ou) + a.abs() * ou
        assert torch.all((out.double() - want).abs() <= limit + (half_step(dtype) * 1.01 + 2.0**-22) * want.abs())


@gpu
@pytest.mark.parametrize("m", [3, 40, 700])
def test_linear_strided_operands(lib, m):
    """Rows of wider matrices on every side; what lies beside the output stays as it was."""
    torch.manual_seed(13)
    n, k = 250, 200
    x, w = operand(m, k + 64), operand(n, k + 32, 0.05)
    x, w = float8.Float8Rows(x.values[:, 16 : 16 + k], x.scales), float8.Float8Rows(w.values[:, 32 : 32 + k], w.scales)
    y, magnitudes = wide_product(x, w)
    residual = torch.randn(m, n + 3, device="cuda")[:, 2 : 2 + n]
    for dtype in (torch.float32, torch.bfloat16):
        for first, columns in ((0, n + 7), (1, n + 8), (2, n + 2)):
            held = torch.full((m, columns), 7.0, device="cuda", dtype=dtype)
            out = float8.linear(make_ctx(lib, positions=[0]), x, w, held[:, first : first + n], residual=residual)
            want = y + residual.double()
            off = sum_off(k, magnitudes, dtype) + residual.double().abs() * 2.0**-23
            assert torch.all((out.double() - want).abs() <= off + half_step(dtype) * 1.01 * want.abs())
            held[:, first : first + n] = 7.0
            assert torch.all(held == 7.0)


@gpu
@pytest.mark.parametrize("m", [5, 70, 600])
def test_rows_that_are_not_finite_stay_by_themselves(lib, m):
    torch.manual_seed(14)
    x, w = operand(m, 256), operand(384, 256, 0.05)
    clean = float8.linear(make_ctx(lib, positions=[0]), x, w, torch.empty(m, 384, device="cuda"))
    x.values[2, 9] = math.nan
    x.scales[4] = math.inf
    w.scales[100] = math.inf
    out = float8.linear(make_ctx(lib, positions=[0]), x, w, torch.empty(m, 384, device="cuda"))
    assert torch.all(torch.isnan(out[2])) and not torch.any(torch.isfinite(out[4])) and not torch.any(torch.isfinite(out[:, 100]))
    rows = [i for i in range(m) if i not in (2, 4)]
    columns = [i for i in range(384) if i != 100]
    assert torch.equal(out[rows][:, columns], clean[rows][:, columns])


@gpu
@pytest.mark.parametrize("m", [1, 40, 700])
def test_calls_do_not_depend_on_what_runs_beside_or_before(lib, m):
    """The same call alone, on another stream beside itself, and captured and replayed: the same bits."""
    torch.manual_seed(15)
    x, w = torch.randn(m, 1024, device="cuda"), operand(2048, 1024, 0.05)
    weight = torch.ones(1024, device="cuda")

    def chain(ctx, rows, out):
        float8.rmsnorm(ctx, x, None, weight, 1e-6, rows)
        return float8.linear_gated(ctx, rows, w, out)

    # A context whose stream is looked up at each launch, as the engine's.
    def context():
        ctx = make_ctx(lib, positions=[0])

        class Current(SimpleNamespace):
            @property
            def stream(self):
                return torch.cuda.current_stream().cuda_stream

        fields = {k: v for k, v in vars(ctx).items() if k != "stream"}
        return Current(**fields)

    rooms = [(float8.empty_rows(m, 1024, "cuda:0"), torch.empty(m, 1024, device="cuda", dtype=torch.bfloat16)) for _ in range(3)]
    first = chain(context(), *rooms[0]).clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, room in zip(streams, rooms[1:]):
            with torch.cuda.stream(s):
                chain(context(), *room)
    torch.cuda.synchronize()
    assert torch.equal(rooms[1][1], first) and torch.equal(rooms[2][1], first)
    graph = torch.cuda.CUDAGraph()
    ctx = context()
    rooms[0][1].zero_()
    with torch.cuda.graph(graph):
        chain(ctx, *rooms[0])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(rooms[0][1], first) and int(ctx.err.item()) == 0


@gpu
def test_weights_made_on_the_same_stream_are_waited_for(lib):
    """Weights that are not promised constant may come out of the kernel right in front."""
    torch.manual_seed(16)
    ctx = make_ctx(lib, positions=[0])
    x = operand(4, 4096)
    sources = [torch.randn(4096, 4096, device="cuda") * 0.05 for _ in range(2)]
    want = [float8.linear(ctx, x, float8.quantize(ctx, s, float8.empty_rows(4096, 4096, "cuda:0")), torch.empty(4, 4096, device="cuda")) for s in sources]
    torch.cuda.synchronize()
    w = float8.empty_rows(4096, 4096, "cuda:0")
    for turn in range(20):
        float8.quantize(ctx, sources[turn % 2], w)
        out = float8.linear(ctx, x, w, torch.empty(4, 4096, device="cuda"))
        assert torch.equal(out, want[turn % 2])


@gpu
@pytest.mark.parametrize("constant", [True, False])
@pytest.mark.parametrize("m,n,k", [(3, 336, 1200), (50, 400, 2320), (40, 17936, 1040), (900, 1056, 720)])
def test_first_call_of_a_size_inside_a_capture(lib, m, n, k, constant):
    """Plans and attributes are made then; nothing of that is a stream's work."""
    torch.manual_seed(17)
    x, w = operand(m, k), operand(n, k, 0.05)
    w.constant = constant
    ctx = make_ctx(lib, positions=[0])
    out = torch.zeros(m, n, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.stream = torch.cuda.current_stream().cuda_stream
        float8.linear(ctx, x, w, out)
    graph.replay()
    torch.cuda.synchronize()
    y, magnitudes = wide_product(x, w)
    assert torch.all((out.double() - y).abs() <= sum_off(k, magnitudes, torch.float32) + half_step(torch.float32) * 1.01 * y.abs())


@gpu
def test_threads_of_one_process(lib):
    """Two threads, streams and sets of sizes at once."""
    import threading

    torch.manual_seed(18)
    cases = [[(m, operand(m, 640), operand(n, 640, 0.05)) for m, n in sizes] for sizes in (((1, 512), (40, 1024), (300, 768)), ((2, 528), (70, 1040), (600, 512)))]
    want = [[float8.linear(make_ctx(lib, positions=[0]), x, w, torch.empty(m, w.shape[0], device="cuda")) for m, x, w in case] for case in cases]
    torch.cuda.synchronize()
    wrong: list = []

    def work(case, expected):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            ctx = make_ctx(lib, positions=[0])
            for _ in range(30):
                got = [float8.linear(ctx, x, w, torch.empty(m, w.shape[0], device="cuda")) for m, x, w in case]
            stream.synchronize()
            wrong.extend(not torch.equal(a, b) for a, b in zip(got, expected))

    threads = [threading.Thread(target=work, args=pair) for pair in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(wrong) == 6 and not any(wrong)


@gpu
def test_offsets_past_32_bits(lib):
    """Rows whose numbers lie more than 2^31 elements behind the first: the last rows and columns of each are right."""
    torch.manual_seed(19)
    ctx = make_ctx(lib, positions=[0])
    rows, columns = 120000, 18944
    x = torch.empty(rows, columns, device="cuda", dtype=torch.bfloat16)
    x[-300:] = torch.randn(300, columns, device="cuda").bfloat16()
    x[:-300] = 0.5
    out = float8.quantize(ctx, x, float8.empty_rows(rows, columns, "cuda:0"))
    check_rows(float8.Float8Rows(out.values[-300:], out.scales[-300:]), x[-300:].double(), 2.0**-23, 2.0**-22)
    del x
    # That matrix as the weights of a few tokens, and as many tokens of a small product whose outputs pass 2^31 too.
    out.constant = True
    few = operand(3, columns)
    y = float8.linear(ctx, few, out, torch.empty(3, rows, device="cuda"))
    last = float8.Float8Rows(out.values[-300:], out.scales[-300:])
    want, magnitudes = wide_product(few, last)
    assert torch.all((y[:, -300:].double() - want).abs() <= sum_off(columns, magnitudes, torch.float32) + half_step(torch.float32) * 1.01 * want.abs())
    del out, y
    many, w = operand(70000, 64), operand(32000, 64, 0.05)
    y = float8.linear(ctx, many, w, torch.empty(70000, 32000, device="cuda", dtype=torch.bfloat16))
    want, magnitudes = wide_product(float8.Float8Rows(many.values[-200:], many.scales[-200:]), w)
    assert torch.all((y[-200:].double() - want).abs() <= sum_off(64, magnitudes, torch.bfloat16) + half_step(torch.bfloat16) * 1.01 * want.abs())
    del y
    # Rows that far apart, in the form that reads them without tensor maps.
    apart = torch.zeros(20 << 28, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).view(20, 1 << 28)
    spread = float8.Float8Rows(apart[:, :64], w.scales[:20].clone())
    spread.values.copy_(w.values[:20])
    got = float8.linear(ctx, few_rows := operand(2, 64), spread, torch.empty(2, 20, device="cuda"))
    want, magnitudes = wide_product(few_rows, float8.Float8Rows(w.values[:20], w.scales[:20]))
    assert torch.all((got.double() - want).abs() <= sum_off(64, magnitudes, torch.float32) + half_step(torch.float32) * 1.01 * want.abs())


# --- refusals, without a GPU ----------------------------------------------------------------------


def refuses(match: str, call) -> None:
    with pytest.raises(KernelError, match=match):
        call()


def test_refusals():
    cpu = torch.device("cpu")
    ctx = SimpleNamespace(device=cpu)
    rows = float8.empty_rows(4, 48, cpu)
    x = torch.zeros(4, 48)
    refuses("x must be", lambda: float8.quantize(ctx, x.half(), rows))
    refuses("x must be", lambda: float8.quantize(ctx, x[:, :40], rows))
    refuses("x must be", lambda: float8.quantize(ctx, torch.zeros(48, 4).t(), rows))
    refuses("x must be", lambda: float8.quantize(ctx, torch.zeros(1, 48).expand(4, 48), rows))
    refuses("out must be", lambda: float8.quantize(ctx, x, float8.Float8Rows(rows.values.view(torch.uint8), rows.scales)))
    refuses("out must be", lambda: float8.quantize(ctx, x, float8.Float8Rows(rows.values, rows.scales.double())))
    refuses("out must be", lambda: float8.quantize(ctx, x, float8.Float8Rows(rows.values, rows.scales[:3])))
    refuses("without numbers", lambda: float8.quantize(ctx, torch.zeros(4, 0), float8.empty_rows(4, 0, cpu)))
    odd = torch.empty(4, 50, dtype=torch.float8_e4m3fn)
    refuses("out must be", lambda: float8.quantize(ctx, x, float8.Float8Rows(odd[:, :48], rows.scales)))
    wide = torch.empty(4, 64, dtype=torch.float8_e4m3fn)
    refuses("out must be", lambda: float8.quantize(ctx, x, float8.Float8Rows(wide[:, 8:56], rows.scales)))
    weight = torch.ones(48)
    refuses("delta must be", lambda: float8.rmsnorm(ctx, x, x.half(), weight, 1e-6, rows))
    refuses("x must be", lambda: float8.rmsnorm(ctx, x.bfloat16(), None, weight, 1e-6, rows))
    refuses("weight must be", lambda: float8.rmsnorm(ctx, x, None, weight[:40], 1e-6, rows))
    refuses("stream must be", lambda: float8.rmsnorm(ctx, x, None, weight, 1e-6, rows, stream=x.bfloat16()))
    w, out = float8.empty_rows(6, 48, cpu), torch.zeros(4, 6)
    refuses("x is .* but weight is", lambda: float8.linear(ctx, rows, float8.empty_rows(6, 64, cpu), out))
    refuses("out must be", lambda: float8.linear(ctx, rows, w, out[:, :5]))
    refuses("out must be", lambda: float8.linear(ctx, rows, w, out.half()))
    refuses("out must be", lambda: float8.linear(ctx, rows, w, torch.zeros(6, 4).t()))
    refuses("bias must be", lambda: float8.linear(ctx, rows, w, out, bias=torch.zeros(6).bfloat16()))
    refuses("residual must be", lambda: float8.linear(ctx, rows, w, out, residual=out.bfloat16()))
    refuses("no activation", lambda: float8.linear(ctx, rows, w, out, activation="relu"))
    refuses("no gated activation", lambda: float8.linear_gated(ctx, rows, w, out[:, :3], activation="squared_relu"))
    refuses("come in pairs", lambda: float8.linear_gated(ctx, rows, float8.empty_rows(5, 48, cpu), out[:, :3]))
    refuses("out must be", lambda: float8.linear_gated(ctx, rows, w, out))
    refuses("two dimensions", lambda: float8.from_tensor(weight))
    elsewhere = SimpleNamespace(device=torch.device("cuda:0"))
    refuses("on cuda:0", lambda: float8.quantize(elsewhere, x, rows))
    refuses("on cuda:0", lambda: float8.linear(elsewhere, rows, w, out))


@gpu
def test_quantize_bfloat16_that_is_not_finite(lib):
    """Two at a time: a NaN beside a number, a pair of them, infinities of both signs."""
    torch.manual_seed(20)
    x = torch.randn(6, 512, device="cuda").bfloat16()
    clean = x.clone()
    x[1, 10] = math.nan
    x[2, 64:72] = math.nan
    x[3, 100], x[3, 101] = -math.inf, math.inf
    x[4, 500] = math.inf
    out = float8.quantize(make_ctx(lib, positions=[0]), x, float8.empty_rows(6, 512, "cuda:0"))
    q, s = out.values.float(), out.scales
    for row, places in ((1, [10]), (2, list(range(64, 72)))):
        others = [i for i in range(512) if i not in places]
        assert torch.isnan(q[row, places]).all() and math.isfinite(float(s[row]))
        check_rows(float8.Float8Rows(out.values[row : row + 1, others], s[row : row + 1]), clean[row : row + 1, others].double(), 2.0**-23, 2.0**-22)
    for row, places in ((3, [100, 101]), (4, [500])):
        others = [i for i in range(512) if i not in places]
        assert torch.isnan(q[row, places]).all() and math.isinf(float(s[row])) and torch.all(q[row, others] == 0)
    check_rows(float8.Float8Rows(out.values[[0, 5]], s[[0, 5]]), clean[[0, 5]].double(), 2.0**-23, 2.0**-22)


@gpu
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("columns", [1001, 4096, 20000])
def test_rmsnorm_with_a_weight_made_just_before(lib, rows, columns):
    """The kernel in front makes the weight, and lets its successor start before it has ended: the norm has to read what it wrote."""
    torch.manual_seed(31)
    ctx = make_ctx(lib, positions=[0])
    one, w = operand(1, 2048), operand(columns, 2048, 0.05)
    first, second = float8.Float8Rows(one.values, one.scales), float8.Float8Rows(one.values, one.scales * 3)
    x = torch.randn(rows, columns, device="cuda")
    want = []
    for source in (first, second):
        weight = float8.linear(ctx, source, w, torch.empty(1, columns, device="cuda"))
        torch.cuda.synchronize()
        want.append(float8.rmsnorm(ctx, x, None, weight[0], 1e-6, float8.empty_rows(rows, columns, "cuda:0")))
    torch.cuda.synchronize()
    weight, out = torch.empty(1, columns, device="cuda"), [float8.empty_rows(rows, columns, "cuda:0") for _ in range(40)]
    for i, o in enumerate(out):
        float8.linear(ctx, (first, second)[i % 2], w, weight)
        float8.rmsnorm(ctx, x, None, weight[0], 1e-6, o)
    for i, o in enumerate(out):
        assert torch.equal(o.values.view(torch.uint8), want[i % 2].values.view(torch.uint8)) and torch.equal(o.scales, want[i % 2].scales)


@gpu
@pytest.mark.parametrize("m", [9, 128, 500, 777])
@pytest.mark.parametrize("kind", ["plain", "squared_relu", "gated"])
def test_32_bit_outputs_of_long_rows(lib, kind, m):
    """Products are added toward zero: a chain of n additions loses 1.6e-9 n of a sum of both signs. Chains end after 320 (5.1e-7), after 160 under an
    activation (2.6e-7, which a square or a product of two sums doubles); the pieces, scales and the function are rounded as ever, each rounding 2^-24 at most, of
    which four at their worst add 2.4e-7, twice that through a square. Sum of both: 7.5e-7, and 9.9e-7."""
    torch.manual_seed(32)
    n, k = 37888 if m == 128 else 4096, 18944
    x, w = operand(m, k), operand(n, k, 0.02)
    ctx = make_ctx(lib, positions=[0])
    if kind == "gated":
        out = float8.linear_gated(ctx, x, w, torch.empty(m, n // 2, device="cuda"))
    else:
        out = float8.linear(ctx, x, w, torch.empty(m, n, device="cuda"), activation=None if kind == "plain" else kind)
    a = x.values.double() * x.scales.double()[:, None]
    y = torch.cat([a @ (w.values[at : at + 4096].double() * w.scales[at : at + 4096].double()[:, None]).t() for at in range(0, n, 4096)], dim=1)
    want = wide_activation(y[:, 0::2], "silu") * y[:, 1::2] if kind == "gated" else wide_activation(y, None if kind == "plain" else kind)
    off = float((out.double() - want).norm() / want.norm())
    assert off <= (7.5e-7 if kind == "plain" else 9.9e-7)
