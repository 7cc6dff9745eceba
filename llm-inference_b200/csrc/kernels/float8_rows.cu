// Rows of numbers to rows of e4m3 with a 32-bit scale each (float8.cuh), by themselves or as the output of an RMS norm with the residual's addition.
//
//   quantize:  scale = max(amax |v| / 448, 2^-126),  q = e4m3(v / scale)
//   rmsnorm:   s = x + delta (written out),  v = s * rsqrt(mean s^2 + eps) * w,  then the same
//
// One pass: a row is read once and stays in registers. The norm's 1 / rms is a factor of the whole row, so the largest |s w| is found together with the
// sum of squares (one meeting of the row's threads, not two), the factor drops out of q = s w / (amax |s w| / 448), and only the scale
// has it. Divisions by the scale are products with one reciprocal a row: 448 / amax is rounded once, v times it once, which moves a quotient by
// 2^-23 of itself at most; e4m3 rounds it by 2^-4.
// NaN stays NaN in its place (the largest magnitude is taken over the others); a row with an infinity has scale infinity, its finite numbers are
// zeros and its infinities NaN, so what is made of that row is NaN and no other row is touched.
//
// Memory bound. A row's threads each hold kItems packs of eight numbers (16 bytes of bfloat16, two times 16 of 32 bits; 8 bytes of e4m3 out); rows whose length,
// stride or base does not allow packs go a number at a time. A block takes as many rows as fit its threads, so short rows do not leave lanes
// idle. Rows too long for the registers are read twice (the second time out of L2).
#include <type_traits>

#include "float8.cuh"
#include "packs.cuh"

namespace float8 {
namespace {

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {  // lo in the lower byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight neighbouring numbers in packs, or one.
template <int W>
struct Group;
template <>
struct Group<8> {
  float v[8];
  template <typename T>
  __device__ __forceinline__ void load(const T* p) {
    const float4 a = load4<T>(p), b = load4<T>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void store_e4m3(uint8_t* p, float first, float second) const {
    uint2 r;
    r.x = to_e4m3x2(v[0] * first * second, v[1] * first * second) | to_e4m3x2(v[2] * first * second, v[3] * first * second) << 16;
    r.y = to_e4m3x2(v[4] * first * second, v[5] * first * second) | to_e4m3x2(v[6] * first * second, v[7] * first * second) << 16;
    *reinterpret_cast<uint2*>(p) = r;
  }
};
template <>
struct Group<1> {
  float v[1];
  template <typename T>
  __device__ __forceinline__ void load(const T* p) { v[0] = to_f32<T>(*p); }
  __device__ __forceinline__ void store(float* p) const { *p = v[0]; }
  __device__ __forceinline__ void store_e4m3(uint8_t* p, float first, float second) const { *p = static_cast<uint8_t>(to_e4m3x2(v[0] * first * second, 0.f)); }
};
template <>
__device__ __forceinline__ void Group<8>::load<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(words[i] << 16);
    v[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
  }
}

struct RowsParams {
  const void* x;       // quantize: T rows; norm: the 32-bit stream
  const void* delta;   // norm only: T rows or null
  const float* weight; // norm only
  float* stream;       // norm only: where s goes (null: nowhere)
  uint8_t* out;
  float* scales;
  int64_t x_stride, delta_stride, stream_stride, out_stride;
  int rows, columns;
  int row_threads;     // threads of a row, a multiple of 32
  float eps;
};

// Sum and maximum over a row's threads; `scratch` holds two floats a warp of the block.
__device__ __forceinline__ void meet(float& sum, float& most, float2* scratch, int row_threads) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if (row_threads == 32) return;
  const int warps = row_threads >> 5, first = warp / warps * warps;
  if (lane == 0) scratch[warp] = make_float2(sum, most);
  __syncthreads();
  const float2 part = lane < warps ? scratch[first + lane] : make_float2(0.f, 0.f);
  sum = part.x;
  most = part.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
}

// W: numbers a group; ITEMS: groups a thread holds (0: the row is read twice instead).
template <bool NORM, typename T, int W, int ITEMS>
__global__ void __launch_bounds__(1024)
float8_rows_kernel(const RowsParams p) {
  __shared__ float2 scratch[32];
  const int in_block = blockDim.x / p.row_threads;
  const int at_row = threadIdx.x / p.row_threads, t = threadIdx.x - at_row * p.row_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * in_block + at_row;
  const bool live = row < p.rows;
  const int groups = live ? p.columns / W : 0;
  using Source = typename std::conditional<NORM, float, T>::type;
  const Source* x = static_cast<const Source*>(p.x) + row * p.x_stride;
  const T* delta = NORM && p.delta != nullptr ? static_cast<const T*>(p.delta) + row * p.delta_stride : nullptr;
  float* stream = NORM && p.stream != nullptr ? p.stream + row * p.stream_stride : nullptr;
  uint8_t* out = p.out + row * p.out_stride;
  // The weight depends on nothing on the stream: it is asked for first.
  Group<W> weight[ITEMS > 0 ? ITEMS : 1];
  if constexpr (NORM && ITEMS > 0) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) weight[j].load(p.weight + (t + j * p.row_threads) * W);
  }
  wait_for_predecessor();
  let_successor_start();

  float sum = 0.f, most = 0.f;
  auto fetch = [&](Group<W>& g, Group<W>& d, int at) {
    g.load(x + at * W);
    if (NORM && delta != nullptr) d.load(delta + at * W);
  };
  auto take = [&](Group<W>& g, const Group<W>& d, const Group<W>& w, int at) {  // a group's part of the sum and of the maximum; times w
    if constexpr (NORM) {
      if (delta != nullptr) {
#pragma unroll
        for (int i = 0; i < W; ++i) g.v[i] += d.v[i];
      }
      if (stream != nullptr) g.store(stream + at * W);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        sum = fmaf(g.v[i], g.v[i], sum);
        g.v[i] *= w.v[i];
      }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) most = fmaxf(most, fabsf(g.v[i]));
  };
  Group<W> held[ITEMS > 0 ? ITEMS : 1], added[ITEMS > 0 ? ITEMS : 1];
  if constexpr (ITEMS > 0) {
    // All loads first: the sum's stores may be to where the next group lies, as far as the compiler knows.
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) fetch(held[j], added[j], t + j * p.row_threads);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) take(held[j], added[j], weight[j], t + j * p.row_threads);
  } else {
    for (int at = t; at < groups; at += p.row_threads) {
      if constexpr (NORM) weight[0].load(p.weight + at * W);
      fetch(held[0], added[0], at);
      take(held[0], added[0], weight[0], at);
    }
  }
  meet(sum, most, scratch, p.row_threads);
  if (!live) return;
  // What is held, times `first`, times `second`, is the quotient by the scale. Of a normed row 1 / rms cancels: 448 / most alone, unless the row is so
  // small that a factor would not be a normal number.
  const float rstd = NORM ? rsqrtf(sum / static_cast<float>(p.columns) + p.eps) : 1.f;
  const float largest = most * rstd;
  float scale = largest / kLargest, first = rstd, second = 1.f / kSmallestScale;
  if (scale >= kSmallestScale) {
    first = most >= 1e-30f ? kLargest / most : rstd;
    second = most >= 1e-30f ? 1.f : kLargest / largest;
  }
  if (scale < kSmallestScale) scale = kSmallestScale;
  if (t == 0) p.scales[row] = scale;
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) held[j].store_e4m3(out + (t + j * p.row_threads) * W, first, second);
  } else {
    // The second reading: of the sum where it was written out, else of its parts again.
    for (int at = t; at < groups; at += p.row_threads) {
      if (NORM && stream != nullptr) {
        held[0].load(stream + at * W);
      } else {
        held[0].load(x + at * W);
        if (delta != nullptr) {
          Group<W> d;
          d.load(delta + at * W);
#pragma unroll
          for (int i = 0; i < W; ++i) held[0].v[i] += d.v[i];
        }
      }
      if constexpr (NORM) {
        weight[0].load(p.weight + at * W);
#pragma unroll
        for (int i = 0; i < W; ++i) held[0].v[i] *= weight[0].v[i];
      }
      held[0].store_e4m3(out + at * W, first, second);
    }
  }
}

bool aligned(const void* p, int64_t stride_bytes, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0 && stride_bytes % to == 0; }

template <bool NORM, typename T, int W>
cudaError_t launch_rows_as(RowsParams p, cudaStream_t stream) {
  const int groups = p.columns / W;
  constexpr int kMost = W == 8 ? 4 : 8;  // groups a thread holds
  // Threads of a row: two groups each (one where rows are few, whose time is all latency), up to a block of 1,024.
  const int each = W == 8 ? (p.rows >= 2 * b200_sm_count_host() ? 2 : 1) : 4;
  int threads = ((groups + each - 1) / each + 31) / 32 * 32;
  threads = max(32, min(threads, 1024));
  int items = (groups + threads - 1) / threads;
  // Short rows share a block of up to 256 threads, if there are enough of them to go round.
  int in_block = 1;
  while (threads * in_block * 2 <= 256 && p.rows >= 2 * in_block * 4 * b200_sm_count_host()) in_block *= 2;
  p.row_threads = threads;
  const dim3 grid((p.rows + in_block - 1) / in_block), block(threads * in_block);
  if (items <= 1) return launch_kernel(float8_rows_kernel<NORM, T, W, 1>, grid, block, 0, stream, p);
  if (items <= 2) return launch_kernel(float8_rows_kernel<NORM, T, W, 2>, grid, block, 0, stream, p);
  if (items <= kMost) return launch_kernel(float8_rows_kernel<NORM, T, W, kMost>, grid, block, 0, stream, p);
  return launch_kernel(float8_rows_kernel<NORM, T, W, 0>, grid, block, 0, stream, p);
}

template <bool NORM>
int launch_rows(const RowsParams& p, bool packs, int dtype, cudaStream_t stream) {
  cudaError_t status;
  if (dtype == DTYPE_F32)
    status = packs ? launch_rows_as<NORM, float, 8>(p, stream) : launch_rows_as<NORM, float, 1>(p, stream);
  else
    status = packs ? launch_rows_as<NORM, __nv_bfloat16, 8>(p, stream) : launch_rows_as<NORM, __nv_bfloat16, 1>(p, stream);
  if (status != cudaSuccess) {
    cudaGetLastError();
    return b200_fail("float8 rows: %s", cudaGetErrorString(status));
  }
  return 0;
}

}  // namespace
}  // namespace float8

// The numbers of a call, in the order in which parts/float8.py packs them; pitches in elements.
struct Float8Quantize {
  const void* x;
  int64_t dtype, x_pitch;  // dtype: of x
  void* out;
  int64_t out_pitch;
  float* scales;
  int64_t rows, columns;
};
struct Float8RmsNorm {
  const float* x;
  int64_t x_pitch;
  const void* delta;
  int64_t dtype, delta_pitch;  // dtype: of delta (of nothing where there is none)
  const float* weight;
  float* stream;
  int64_t stream_pitch;
  void* out;
  int64_t out_pitch;
  float* scales;
  int64_t rows, columns;
  double eps;
};
static_assert(sizeof(Float8Quantize) == 8 * 8 && sizeof(Float8RmsNorm) == 14 * 8, "as packed by the caller");

static bool float8_sizes(int64_t rows, int64_t columns) { return rows > 0 && columns > 0 && rows < (int64_t(1) << 31) && columns < (int64_t(1) << 31); }

B200_API int b200_float8_quantize(const Float8Quantize* c, cudaStream_t stream) {
  using namespace float8;
  if (c->rows == 0) return 0;
  B200_REQUIRE(float8_sizes(c->rows, c->columns), "float8 quantize: bad sizes");
  B200_REQUIRE(c->dtype == DTYPE_F32 || c->dtype == DTYPE_BF16, "float8 quantize: unknown dtype %d", static_cast<int>(c->dtype));
  RowsParams p = {};
  p.x = c->x, p.x_stride = c->x_pitch, p.out = static_cast<uint8_t*>(c->out), p.out_stride = c->out_pitch, p.scales = c->scales;
  p.rows = static_cast<int>(c->rows), p.columns = static_cast<int>(c->columns);
  const int size = c->dtype == DTYPE_F32 ? 4 : 2;
  const bool packs = p.columns % 8 == 0 && aligned(c->x, c->x_pitch * size, 16) && aligned(c->out, c->out_pitch, 8);
  return launch_rows<false>(p, packs, static_cast<int>(c->dtype), stream);
}

B200_API int b200_float8_rmsnorm(const Float8RmsNorm* c, cudaStream_t stream) {
  using namespace float8;
  if (c->rows == 0) return 0;
  B200_REQUIRE(float8_sizes(c->rows, c->columns), "float8 rmsnorm: bad sizes");
  B200_REQUIRE(c->dtype == DTYPE_F32 || c->dtype == DTYPE_BF16, "float8 rmsnorm: unknown dtype %d", static_cast<int>(c->dtype));
  RowsParams p = {};
  p.x = c->x, p.x_stride = c->x_pitch, p.delta = c->delta, p.delta_stride = c->delta_pitch, p.weight = c->weight, p.eps = static_cast<float>(c->eps);
  p.stream = c->stream, p.stream_stride = c->stream_pitch;
  p.out = static_cast<uint8_t*>(c->out), p.out_stride = c->out_pitch, p.scales = c->scales;
  p.rows = static_cast<int>(c->rows), p.columns = static_cast<int>(c->columns);
  const int size = c->dtype == DTYPE_F32 ? 4 : 2;
  const bool packs = p.columns % 8 == 0 && aligned(c->x, c->x_pitch * 4, 16) && aligned(c->weight, 0, 16) && aligned(c->out, c->out_pitch, 8) &&
                     (c->delta == nullptr || aligned(c->delta, c->delta_pitch * size, 16)) &&
                     (c->stream == nullptr || aligned(c->stream, c->stream_pitch * 4, 16));
  return launch_rows<true>(p, packs, static_cast<int>(c->dtype), stream);
}
