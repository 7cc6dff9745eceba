// Product of 8-bit rows for up to 16 tokens and matrices whose stream is short: latency, not bandwidth, is what they cost.
//   y[m][n] = act((sum_k x[m][k] w[n][k]) xs[m] ws[n] + bias[n]) + residual[m][n],  or act(gate) * up over pairs of W's rows.
//
// A block has 16 rows of W (the 16-row operand of `mma.sync` m16n8k32, e4m3) and all tokens (its 8 columns, once or twice); its warps cut K among
// them. A lane takes 16 bytes of two rows of W straight from memory into registers, kSlabs times 64 k at once, and the same of the tokens; the
// order of k inside a slab is the same for both, which a sum does not notice. The warps' sums meet in shared memory and are added in warp
// order. Between the first byte of X and the last store lie two trips to L2 and one meeting of the block, where the streaming form
// (gemm_float8_stream.cu) has TMEM to take, copies and products to wait for and a cluster to meet.
//
// Weights are asked for before the kernel in front has ended where the caller says that nothing still writes them.
#include "float8.cuh"

namespace float8 {
namespace {

constexpr int kRows = 16;        // rows of W a block
constexpr int kSlabK = 64;       // k of a slab: 16 bytes a lane and row
constexpr int kMostWarps = 16;

struct SkinnyParams {
  Epilogue e;
  const uint8_t* x;
  const uint8_t* w;
  int64_t x_stride, w_stride;
  int K;
  int w_constant;
};

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// What is left of a row from k on, fewer than 16 bytes, with zeros behind it.
__device__ __noinline__ uint4 row_end(const uint8_t* row, int k, int K) {
  uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (k + i < K) words[i >> 2] |= static_cast<uint32_t>(row[k + i]) << (8 * (i & 3));
  return make_uint4(words[0], words[1], words[2], words[3]);
}

// MT: tokens / 8. SLABS: slabs of a set; a lane has two sets, one on its way while the other is used.
template <int KIND, typename T, int MT, int SLABS>
__global__ void __launch_bounds__(kMostWarps * 32)
float8_skinny_kernel(const SkinnyParams p) {
  __shared__ __align__(16) float partial[kMostWarps][MT * 8][kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kRows;
  const int whole = p.K & ~15;  // what is behind it is the last warp's, at the end
  const int slabs = (whole + kSlabK - 1) / kSlabK;
  const int begin = static_cast<int>(static_cast<int64_t>(slabs) * warp / warps), end = static_cast<int>(static_cast<int64_t>(slabs) * (warp + 1) / warps);
  const int limit = min(whole, end * kSlabK);
  const int limit_a = n0 + g < p.e.N ? limit : 0, limit_b = n0 + g + 8 < p.e.N ? limit : 0;
  const uint8_t* wa = p.w + (n0 + g < p.e.N ? n0 + g : 0) * p.w_stride;
  const uint8_t* wb = p.w + (n0 + g + 8 < p.e.N ? n0 + g + 8 : 0) * p.w_stride;

  struct Set {
    uint4 a[SLABS], b[SLABS], x[MT][SLABS];
  } sets[2];
  const uint4 zeros = make_uint4(0, 0, 0, 0);
  auto fetch_w = [&](Set& set, int first) {
#pragma unroll
    for (int s = 0; s < SLABS; ++s) {
      const int k = (first + s) * kSlabK + t * 16;
      set.a[s] = k < limit_a ? *reinterpret_cast<const uint4*>(wa + k) : zeros;
      set.b[s] = k < limit_b ? *reinterpret_cast<const uint4*>(wb + k) : zeros;
    }
  };
  auto fetch_x = [&](Set& set, int first) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = i * 8 + g, limit_x = m < p.e.M ? limit : 0;
      const uint8_t* row = p.x + (m < p.e.M ? m : 0) * p.x_stride;
#pragma unroll
      for (int s = 0; s < SLABS; ++s) {
        const int k = (first + s) * kSlabK + t * 16;
        set.x[i][s] = k < limit_x ? *reinterpret_cast<const uint4*>(row + k) : zeros;
      }
    }
  };
  float acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  auto use = [&](const Set& set) {
#pragma unroll
    for (int s = 0; s < SLABS; ++s) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        mma_e4m3(acc[i], set.a[s].x, set.b[s].x, set.a[s].y, set.b[s].y, set.x[i][s].x, set.x[i][s].y);
        mma_e4m3(acc[i], set.a[s].z, set.b[s].z, set.a[s].w, set.b[s].w, set.x[i][s].z, set.x[i][s].w);
      }
    }
  };

  if (!p.w_constant) wait_for_predecessor();
  fetch_w(sets[0], begin);
  fetch_w(sets[1], begin + SLABS);
  wait_for_predecessor();
  let_successor_start();
  fetch_x(sets[0], begin);
  fetch_x(sets[1], begin + SLABS);
  for (int first = begin; first < end; first += 2 * SLABS) {
    use(sets[0]);
    if (first + 2 * SLABS < end) {
      fetch_w(sets[0], first + 2 * SLABS);
      fetch_x(sets[0], first + 2 * SLABS);
    }
    if (first + SLABS < end) use(sets[1]);
    if (first + 3 * SLABS < end) {
      fetch_w(sets[1], first + 3 * SLABS);
      fetch_x(sets[1], first + 3 * SLABS);
    }
  }
  if (whole < p.K && warp == warps - 1) {
    const uint4 a = t == 0 && n0 + g < p.e.N ? row_end(wa, whole, p.K) : zeros;
    const uint4 b = t == 0 && n0 + g + 8 < p.e.N ? row_end(wb, whole, p.K) : zeros;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = i * 8 + g;
      const uint4 x = t == 0 && m < p.e.M ? row_end(p.x + m * p.x_stride, whole, p.K) : zeros;
      mma_e4m3(acc[i], a.x, b.x, a.y, b.y, x.x, x.y);
      mma_e4m3(acc[i], a.z, b.z, a.w, b.w, x.z, x.w);
    }
  }
  // This warp's sums: rows g and g + 8, tokens 8 i + 2 t and the next.
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    partial[warp][i * 8 + 2 * t][g] = acc[i][0];
    partial[warp][i * 8 + 2 * t + 1][g] = acc[i][1];
    partial[warp][i * 8 + 2 * t][g + 8] = acc[i][2];
    partial[warp][i * 8 + 2 * t + 1][g + 8] = acc[i][3];
  }
  // An item is four neighbouring rows of one token; what it needs from memory is asked for before the block meets.
  const int m = threadIdx.x >> 2, j = (threadIdx.x & 3) * 4, n = n0 + j;
  const bool mine = m < p.e.M && n < p.e.N;
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f), ws = r, bias = r;
  float xs = 0.f;
  if (mine) {
    const int last = p.e.N - 1;
    xs = p.e.x_scale[m];
    ws = make_float4(p.e.w_scale[n], p.e.w_scale[min(n + 1, last)], p.e.w_scale[min(n + 2, last)], p.e.w_scale[min(n + 3, last)]);
    if (p.e.bias != nullptr) bias = make_float4(p.e.bias[n], p.e.bias[min(n + 1, last)], p.e.bias[min(n + 2, last)], p.e.bias[min(n + 3, last)]);
    if (KIND != GATED && p.e.residual != nullptr) r = residual_quad(p.e, m, n);
  }
  __syncthreads();
  if (!mine) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < warps; ++w) sum = add_each(sum, *reinterpret_cast<const float4*>(&partial[w][m][j]));
  float4 v = make_float4(fmaf(sum.x * xs, ws.x, bias.x), fmaf(sum.y * xs, ws.y, bias.y), fmaf(sum.z * xs, ws.z, bias.z), fmaf(sum.w * xs, ws.w, bias.w));
  if constexpr (KIND == ACTIVATED) v = activate_quad(v, p.e.activation);
  if constexpr (KIND != GATED) v = add_each(v, r);
  T* to = static_cast<T*>(p.e.out) + m * p.e.out_stride + (KIND == GATED ? n >> 1 : n);
  if (p.e.vector && n + 3 < p.e.N) store_whole<KIND, T>(to, v, p.e.activation);
  else store_some<KIND, T>(to, n, p.e.N, v, p.e.activation);
}

template <typename T, int MT, int SLABS>
cudaError_t launch_kind(const SkinnyParams& p, int kind, dim3 grid, dim3 block, cudaStream_t stream) {
  if (kind == GATED) return launch_kernel(float8_skinny_kernel<GATED, T, MT, SLABS>, grid, block, 0, stream, p);
  if (kind == ACTIVATED) return launch_kernel(float8_skinny_kernel<ACTIVATED, T, MT, SLABS>, grid, block, 0, stream, p);
  return launch_kernel(float8_skinny_kernel<PLAIN, T, MT, SLABS>, grid, block, 0, stream, p);
}

}  // namespace

// All blocks run at once, 16 warps an SM (their registers), each warp with three slabs at least.
static int skinny_warps(int N, int K) {
  const int blocks = (N + kRows - 1) / kRows, slabs = (K + kSlabK - 1) / kSlabK, sms = b200_sm_count_host();
  return max(1, min(kMostWarps / ((blocks + sms - 1) / sms), (slabs + 2) / 3));
}

// Streams that are short for a warp. Up to 8 tokens (us, this form and the streaming one): 2,048 x 1,536 2.3 and 4.3, 3,584 x 3,584 4.2 and 5.1, 4,608 x
// 3,584 4.9 and 5.7 (7 slabs a warp), 5,120 x 5,120 8.2 and 7.2 (16). Up to 16, where a block takes as much of X as of W out of L2: 2,048 x 1,536
// 2.9 and 4.3 (3 slabs), 896 x 4,864 4.5 and 5.5 (5), 3,584 x 3,584 6.3 and 5.5 (7).
bool skinny_takes(int M, int N, int K) {
  if (M > 16) return false;
  const int blocks = (N + kRows - 1) / kRows, sms = b200_sm_count_host();
  if (blocks > kMostWarps * sms) return false;
  const int slabs = (K + kSlabK - 1) / kSlabK, warps = skinny_warps(N, K);
  return (slabs + warps - 1) / warps <= (M <= 8 ? 9 : 5);
}

int launch_skinny(const Product& product, cudaStream_t stream) {
  SkinnyParams p;
  p.e = product.e;
  p.x = static_cast<const uint8_t*>(product.x);
  p.w = static_cast<const uint8_t*>(product.w);
  p.x_stride = product.x_stride;
  p.w_stride = product.w_stride;
  p.K = product.K;
  p.w_constant = product.w_constant;
  const dim3 grid((p.e.N + kRows - 1) / kRows), block(32 * max(2, skinny_warps(p.e.N, p.K)));  // two: 64 threads finish
  cudaError_t status;
  if (p.e.M <= 8)
    status = product.out_f32 ? launch_kind<float, 1, 4>(p, product.kind, grid, block, stream) : launch_kind<__nv_bfloat16, 1, 4>(p, product.kind, grid, block, stream);
  else
    status = product.out_f32 ? launch_kind<float, 2, 3>(p, product.kind, grid, block, stream) : launch_kind<__nv_bfloat16, 2, 3>(p, product.kind, grid, block, stream);
  if (status != cudaSuccess) {
    cudaGetLastError();
    return b200_fail("float8 product: %s", cudaGetErrorString(status));
  }
  return 0;
}

}  // namespace float8
