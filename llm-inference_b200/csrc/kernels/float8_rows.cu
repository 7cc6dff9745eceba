// Rows of numbers to rows of e4m3 with a 32-bit scale each (float8.cuh), by themselves or as the output of an RMS norm with the residual's addition.
//
//   quantize:  scale = max(amax |v| * (1 / 448), 2^-126),  q = e4m3(v / scale), each step in 32 bits
//   rmsnorm:   s = x + delta (written out),  v = s * rsqrt(mean s^2 + eps) * w,  then the same
//
// One pass: a row is read once and stays in registers. The norm's 1 / rms is a factor of the whole row, so the largest |s w| is found together with the
// sum of squares (one meeting of the row's threads, not two), the factor drops out of q = s w / (amax |s w| / 448), and only the scale
// has it. The norm's divisions by the scale are products with one reciprocal a row: 448 / amax is rounded once, v times it once, which moves a quotient by
// 2^-23 of itself at most; e4m3 rounds it by 2^-4. quantize has to be exact: quotients of bfloat16 rows often lie on the middle between two e4m3 numbers, and one that
// is 2^-24 off goes to the other side (Quotient below).
// quantize: NaN stays NaN in its place (the largest magnitude is taken over the others); a row with an infinity has scale infinity, its finite numbers are
// zeros and its infinities NaN, so what is made of that row is NaN. rmsnorm: a NaN or an infinity makes the mean, and with it the row's scale, NaN. No
// other row is touched. s w is held in 32 bits before 1 / rms: weights for which it leaves their range while the normed number does not (below 1e-20, where eps is zero) are not
// provided for. A sum of squares beyond 32 bits (numbers of 1e19) counts as infinite: the row becomes zeros, as in the formula in 32 bits.
//
// Memory bound. A row's threads each hold a few groups of 16 bytes (of single numbers where a row's length, stride or base does not allow that), all
// asked for before the first is used. A block takes as many rows as fit its threads, so short rows do not leave lanes idle. Rows too long for
// the registers are read twice, the second time out of L2. Of what memory takes at its copy rate: 8,192 rows of 3,584 with a bfloat16 branch output
// 50.6 us of 49.3, 2,048 of 5,120 20.4 of 17.6; 2,048 rows of 18,944 bfloat16 to 8 bits 21.5 of 17.8 (64 registers a thread let
// three blocks onto an SM; instructions, some 90 for eight numbers, stand in the way with two).
#include "float8.cuh"
#include "packs.cuh"

namespace float8 {
namespace {

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {  // lo in the lower byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The larger magnitudes of two pairs of bfloat16 numbers (a NaN counts for nothing beside a number).
__device__ __forceinline__ uint32_t max_abs(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
  return r;
}

// W neighbouring numbers as they lie in memory, and as 32-bit ones.
template <typename T, int W>
struct Raw;
template <>
struct Raw<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ float largest() const { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }  // NaN counts for nothing
  __device__ __forceinline__ void widen(float (&f)[4]) const { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
};
template <>
struct Raw<__nv_bfloat16, 4> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void widen(float (&f)[4]) const {
    f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u), f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
};
template <>
struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ float largest() const {  // two at a time
    uint32_t m = max_abs(max_abs(v.x, v.y), max_abs(v.z, v.w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  __device__ __forceinline__ void widen(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ float largest() const { return fabsf(to_f32<T>(v)); }
  __device__ __forceinline__ void widen(float (&f)[1]) const { f[0] = to_f32<T>(v); }
};
__device__ __forceinline__ void store_f32(float* p, const float (&f)[4]) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
__device__ __forceinline__ void store_f32(float* p, const float (&f)[1]) { *p = f[0]; }
__device__ __forceinline__ uint32_t four(float2 lo, float2 hi) { return to_e4m3x2(lo.x, lo.y) | to_e4m3x2(hi.x, hi.y) << 16; }
__device__ __forceinline__ uint32_t four(const float* f, float factor) {
  const float2 both = make_float2(factor, factor);
  return four(mul_2(make_float2(f[0], f[1]), both), mul_2(make_float2(f[2], f[3]), both));
}
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[8], float factor) { *reinterpret_cast<uint2*>(p) = make_uint2(four(f, factor), four(f + 4, factor)); }
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[4], float factor) { *reinterpret_cast<uint32_t*>(p) = four(f, factor); }
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[1], float factor) { *p = static_cast<uint8_t>(to_e4m3x2(f[0] * factor, 0.f)); }
// The same of a row that may need two factors (RowScale).
template <int W>
__device__ __forceinline__ void store_e4m3(uint8_t* p, float (&f)[W], float first, float second) {
  if (second != 1.f) {
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] *= first;
    first = second;
  }
  store_e4m3(p, f, first);
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

// Largest of numbers that are not negative (their bits are ordered as they are), and the sum too, over a row's threads; `scratch` holds a number a
// warp of the block, each.
__device__ __forceinline__ float warp_largest(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }
__device__ __forceinline__ float row_largest(float most, float* scratch, int row_threads) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  most = warp_largest(most);
  if (row_threads == 32) return most;
  const int warps = row_threads >> 5, first = warp / warps * warps;
  if (lane == 0) scratch[warp] = most;
  __syncthreads();
  return warp_largest(lane < warps ? scratch[first + lane] : 0.f);
}
__device__ __forceinline__ void row_sum_and_largest(float& sum, float& most, float2* scratch, int row_threads) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  sum = warp_sum(sum);
  most = warp_largest(most);
  if (row_threads == 32) return;
  const int warps = row_threads >> 5, first = warp / warps * warps;
  if (lane == 0) scratch[warp] = make_float2(sum, most);
  __syncthreads();
  const float2 part = lane < warps ? scratch[first + lane] : make_float2(0.f, 0.f);
  sum = warp_sum(part.x);
  most = warp_largest(part.y);
}

constexpr unsigned kPrefetchBlocks = 148;  // as many as SMs
constexpr float kSmallestAmax = kLargest * kSmallestScale;  // rows below it have the smallest scale
constexpr float kPerLargest = 1.f / kLargest;

// A row's scale and its numbers' quotients by it, as elementary operations have them: rounded to 32 bits (to nearest even) before they are rounded to e4m3.
// 1 / scale is held in two words, 1 / scale = hi + lo but for 2^-48 of itself, and the quotient is v lo + v hi, rounded twice, the first time far below the last
// bit. With `lo` rounded upward no quotient comes to lie on another side of a middle between two e4m3 numbers than the rounded one (or beside a middle that
// it should be on): tried for all 2^23 mantissas of a scale and, next to each middle, 13 numbers v, whose exponents do not matter while nothing leaves the
// range. Numbers and scale are therefore made smaller where `lo` would be too small to have all its bits. A scale of infinity has quotients 0 and, of infinities, NaN.
// (2,048 rows of 18,944 bfloat16 numbers 21.5 us; with the product by `hi` alone 20.2.)
struct Quotient {
  float scale, hi, lo, down;
  __device__ __forceinline__ explicit Quotient(float most) {
    scale = fmaxf(most * kPerLargest, kSmallestScale);
    down = scale > 0x1p64f ? 0x1p-64f : 1.f;  // a normal number is left of all quotients above 2^-10
    const float by = scale * down;
    hi = 1.f / by;
    lo = isinf(scale) ? 0.f : __fmul_ru(fmaf(-hi, by, 1.f), hi);
  }
  __device__ __forceinline__ float2 two(float a, float b) const {
    const float2 v = make_float2(a, b);
    return fma_2(v, make_float2(hi, hi), mul_2(v, make_float2(lo, lo)));
  }
  __device__ __forceinline__ float one(float v) const { return fmaf(v, hi, v * lo); }
};
__device__ __forceinline__ uint32_t four(const float* f, const Quotient& q) { return four(q.two(f[0], f[1]), q.two(f[2], f[3])); }
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[8], const Quotient& q) { *reinterpret_cast<uint2*>(p) = make_uint2(four(f, q), four(f + 4, q)); }
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[4], const Quotient& q) { *reinterpret_cast<uint32_t*>(p) = four(f, q); }
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[1], const Quotient& q) { *p = static_cast<uint8_t>(to_e4m3x2(q.one(f[0]), 0.f)); }

// The factors of a normed row: what is held (before 1 / rms), times `first`, times `second`, is the quotient by the scale. 1 / rms cancels, 448 / most alone is
// left, unless the row is so small that a factor would not be a normal number.
struct RowScale {
  float scale, first, second;
  __device__ __forceinline__ RowScale(float most, float rstd) {
    const float largest = most * rstd;
    scale = largest < kSmallestAmax ? kSmallestScale : largest / kLargest;
    if (most >= 1e-30f && largest >= kSmallestAmax) first = kLargest / most, second = 1.f;
    else first = rstd, second = largest >= kSmallestAmax ? kLargest / largest : 1.f / kSmallestScale;
  }
};

// W: numbers a group; ITEMS: groups a thread holds (0: the row is read twice instead); THREADS: of a block at most.
template <typename T, int W, int ITEMS, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS <= 512 ? 2 : 1)
float8_quantize_kernel(const RowsParams p) {
  __shared__ float scratch[32];
  const int in_block = blockDim.x / p.row_threads;
  const int at_row = threadIdx.x / p.row_threads, t = threadIdx.x - at_row * p.row_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * in_block + at_row;
  const bool live = row < p.rows;
  const int groups = live ? p.columns / W : 0;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  uint8_t* out = p.out + row * p.out_stride;
  wait_for_predecessor();
  let_successor_start();
  float most = 0.f;
  Raw<T, W> held[ITEMS > 0 ? ITEMS : 1];
  auto look = [&](const Raw<T, W>& g) { most = fmaxf(most, g.largest()); };
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) held[j].load(x + (t + j * p.row_threads) * W);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) look(held[j]);
  } else {
    for (int at = t; at < groups; at += p.row_threads) {
      held[0].load(x + at * W);
      look(held[0]);
    }
  }
  most = row_largest(most, scratch, p.row_threads);
  if (!live) return;
  const Quotient quotient(most);
  if (t == 0) p.scales[row] = quotient.scale;
  auto put = [&](const Raw<T, W>& g, int at) {
    float f[W];
    g.widen(f);
    if (quotient.down != 1.f) {
#pragma unroll
      for (int i = 0; i < W; ++i) f[i] *= quotient.down;
    }
    store_e4m3(out + at * W, f, quotient);
  };
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) put(held[j], t + j * p.row_threads);
  } else {
    for (int at = t; at < groups; at += p.row_threads) {
      held[0].load(x + at * W);
      put(held[0], at);
    }
  }
}

template <typename T, int W, int ITEMS, int THREADS>
__global__ void __launch_bounds__(THREADS)
float8_rmsnorm_kernel(const RowsParams p) {
  __shared__ float2 scratch[32];
  const int in_block = blockDim.x / p.row_threads;
  const int at_row = threadIdx.x / p.row_threads, t = threadIdx.x - at_row * p.row_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * in_block + at_row;
  const bool live = row < p.rows;
  const int groups = live ? p.columns / W : 0;
  const float* x = static_cast<const float*>(p.x) + row * p.x_stride;
  const T* delta = p.delta != nullptr ? static_cast<const T*>(p.delta) + row * p.delta_stride : nullptr;
  float* stream = p.stream != nullptr ? p.stream + row * p.stream_stride : nullptr;
  uint8_t* out = p.out + row * p.out_stride;
  constexpr int kHeld = ITEMS > 0 ? ITEMS : 1;
  // The weight is brought into L2 ahead, by the first blocks, and read only behind the wait: the kernel in front may be what makes it. (By all blocks: 2,048
  // rows of 5,120 15.0 us against 14.3; read ahead of the wait, which would go wrong then, 14.2, and one row of 3,584 1.75 against 1.82.)
  Raw<float, W> weight[kHeld];
  if constexpr (ITEMS > 0) {
    constexpr int kLine = 32 / W;  // groups of 128 bytes
    if (blockIdx.x < kPrefetchBlocks && t % kLine == 0) {
#pragma unroll
      for (int j = 0; j < ITEMS; ++j)
        if (t + j * p.row_threads < groups) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.weight + (t + j * p.row_threads) * W));
    }
  }
  wait_for_predecessor();
  let_successor_start();
  float sum = 0.f, most = 0.f;
  float held[kHeld][W];  // s w
  Raw<float, W> from[kHeld];
  Raw<T, W> added[kHeld];
  auto fetch = [&](int j, int at) {
    from[j].load(x + at * W);
    if (delta != nullptr) added[j].load(delta + at * W);
  };
  auto take = [&](int j, int at, bool counts) {
    float w[W];
    from[j].widen(held[j]);
    weight[j].widen(w);
    if (delta != nullptr) {
      float d[W];
      added[j].widen(d);
#pragma unroll
      for (int i = 0; i < W; ++i) held[j][i] += d[i];
    }
    if (counts && stream != nullptr) store_f32(stream + at * W, held[j]);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      sum = fmaf(held[j][i], held[j][i], sum);
      held[j][i] *= w[i];
      most = fmaxf(most, fabsf(held[j][i]));
    }
  };
  if constexpr (ITEMS > 0) {
    // All loads first: the sum's stores may be to where the next group lies, as far as the compiler knows.
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) fetch(j, t + j * p.row_threads);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) weight[j].load(p.weight + (t + j * p.row_threads) * W);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) take(j, t + j * p.row_threads, true);
  } else {
    for (int at = t; at < groups; at += p.row_threads) {
      fetch(0, at);
      weight[0].load(p.weight + at * W);
      take(0, at, true);
    }
  }
  row_sum_and_largest(sum, most, scratch, p.row_threads);
  if (!live) return;
  const RowScale s(most, rsqrtf(sum / static_cast<float>(p.columns) + p.eps));
  if (t == 0) p.scales[row] = s.scale;
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (t + j * p.row_threads < groups) store_e4m3<W>(out + (t + j * p.row_threads) * W, held[j], s.first, s.second);
  } else {
    // The second reading: of the sum where it was written (which may be where x was), else of its parts again.
    if (stream != nullptr) x = stream, delta = nullptr;
    for (int at = t; at < groups; at += p.row_threads) {
      fetch(0, at);
      weight[0].load(p.weight + at * W);
      take(0, at, false);
      store_e4m3<W>(out + at * W, held[0], s.first, s.second);
    }
  }
}

bool aligned(const void* p, int64_t stride_bytes, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0 && stride_bytes % to == 0; }

struct RowsShape {
  int threads, in_block, items;
};
// Threads of a row, `each` groups a thread, up to a block of `most`. Short rows share a block of up to 256 threads, if there are enough of them to go round.
RowsShape rows_shape(int rows, int groups, int each, int most) {
  RowsShape s;
  s.threads = max(32, min(most, ((groups + each - 1) / each + 31) / 32 * 32));
  s.items = (groups + s.threads - 1) / s.threads;
  s.in_block = 1;
  while (s.threads * s.in_block * 2 <= 256 && rows >= 8 * s.in_block * b200_sm_count_host()) s.in_block *= 2;
  return s;
}

template <typename Kernel>
cudaError_t launch_shape(Kernel kernel, RowsParams p, const RowsShape& s, cudaStream_t stream) {
  p.row_threads = s.threads;
  return launch_kernel(kernel, dim3((p.rows + s.in_block - 1) / s.in_block), dim3(s.threads * s.in_block), 0, stream, p);
}

// Groups a thread: two where rows are few and all is latency (64 rows of 5,120: the norm with one group 3.1 us, with two 2.7); else four, of
// eight bfloat16 numbers or of one number eight, so that what every thread does once a row counts less (the norm of 1,777 rows of 1,001 with a
// 32-bit branch output, out of L2: 256 threads 7.6 us, 128 threads 6.9; out of memory 8.0 and 7.8). Longer rows are read twice (2,048 of 18,944 in 32 bits: 384 threads 39 us, 256 45).
template <typename T, int W>
cudaError_t launch_quantize(const RowsParams& p, cudaStream_t stream) {
  const bool few = p.rows < 2 * b200_sm_count_host();
  const RowsShape s = rows_shape(p.rows, p.columns / W, few && W > 1 ? 2 : W == 4 ? 4 : 8, few ? 1024 : 512);
  if (s.items <= 1) return launch_shape(float8_quantize_kernel<T, W, 1, 1024>, p, s, stream);
  if (s.items <= 2) return launch_shape(float8_quantize_kernel<T, W, 2, 1024>, p, s, stream);
  if (s.items <= 4) return launch_shape(float8_quantize_kernel<T, W, 4, 1024>, p, s, stream);
  if (s.items <= 8 && s.threads <= 512) return launch_shape(float8_quantize_kernel<T, W, 8, 512>, p, s, stream);
  return launch_shape(float8_quantize_kernel<T, W, 0, 1024>, p, rows_shape(p.rows, p.columns / W, 1, few ? 1024 : 384), stream);
}

template <typename T, int W>
cudaError_t launch_rmsnorm(const RowsParams& p, cudaStream_t stream) {
  const bool few = p.rows < 2 * b200_sm_count_host();
  const RowsShape s = rows_shape(p.rows, p.columns / W, W == 1 ? 8 : few ? 2 : 4, few ? 1024 : 512);
  if (s.items <= 1) return launch_shape(float8_rmsnorm_kernel<T, W, 1, 1024>, p, s, stream);
  if (s.items <= 2) return launch_shape(float8_rmsnorm_kernel<T, W, 2, 1024>, p, s, stream);
  if (s.items <= 4 && s.threads <= 512) return launch_shape(float8_rmsnorm_kernel<T, W, 4, 512>, p, s, stream);
  if (s.items <= 8 && s.threads <= 512) return launch_shape(float8_rmsnorm_kernel<T, W, 8, 512>, p, s, stream);
  return launch_shape(float8_rmsnorm_kernel<T, W, 0, 1024>, p, s, stream);
}

int launched(cudaError_t status) {
  if (status == cudaSuccess) return 0;
  cudaGetLastError();
  return b200_fail("float8 rows: %s", cudaGetErrorString(status));
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

static bool float8_sizes(int64_t rows, int64_t columns) { return rows > 0 && columns > 0 && rows <= (int64_t(1) << 30) && columns <= (int64_t(1) << 30); }

B200_API int b200_float8_quantize(const Float8Quantize* c, cudaStream_t stream) {
  using namespace float8;
  if (c->rows == 0) return 0;
  B200_REQUIRE(float8_sizes(c->rows, c->columns), "float8 quantize: bad sizes");
  B200_REQUIRE(c->dtype == DTYPE_F32 || c->dtype == DTYPE_BF16, "float8 quantize: unknown dtype %d", static_cast<int>(c->dtype));
  RowsParams p = {};
  p.x = c->x, p.x_stride = c->x_pitch, p.out = static_cast<uint8_t*>(c->out), p.out_stride = c->out_pitch, p.scales = c->scales;
  p.rows = static_cast<int>(c->rows), p.columns = static_cast<int>(c->columns);
  const int size = c->dtype == DTYPE_F32 ? 4 : 2;
  const int w = 16 / size;  // numbers of 16 bytes
  const bool packs = p.columns % w == 0 && aligned(c->x, c->x_pitch * size, 16) && aligned(c->out, c->out_pitch, w);
  if (c->dtype == DTYPE_F32) return launched(packs ? launch_quantize<float, 4>(p, stream) : launch_quantize<float, 1>(p, stream));
  return launched(packs ? launch_quantize<__nv_bfloat16, 8>(p, stream) : launch_quantize<__nv_bfloat16, 1>(p, stream));
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
  const bool packs = p.columns % 4 == 0 && aligned(c->x, c->x_pitch * 4, 16) && aligned(c->weight, 0, 16) && aligned(c->out, c->out_pitch, 4) &&
                     (c->delta == nullptr || aligned(c->delta, c->delta_pitch * size, 4 * size)) &&
                     (c->stream == nullptr || aligned(c->stream, c->stream_pitch * 4, 16));
  if (c->dtype == DTYPE_F32) return launched(packs ? launch_rmsnorm<float, 4>(p, stream) : launch_rmsnorm<float, 1>(p, stream));
  return launched(packs ? launch_rmsnorm<__nv_bfloat16, 4>(p, stream) : launch_rmsnorm<__nv_bfloat16, 1>(p, stream));
}
