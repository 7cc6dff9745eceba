// What the kernels over 8-bit rows share: the e4m3 format, the epilogue of their products and the tcgen05 / TMA pieces.
//
// A matrix in 8 bits is a `Float8Rows` (parts/float8.py): e4m3 numbers q[row][k], rows a multiple of 16 bytes apart, and one 32-bit scale a
// row; the number at (row, k) is q * scale. A product of two such matrices has both scales in front of the sum:
//   y[m][n] = (sum_k x[m][k] w[n][k]) * xs[m] * ws[n].
// A product of two e4m3 numbers has 8 bits, so every product is exact; sums are 32-bit. `tcgen05.mma` drops the bits below the last when it
// adds (toward zero), the products' too, so a sum loses the more an addition the longer its chain is. Measured, 32 k an addition: of numbers of both signs 1.6e-9 of
// itself an addition (5e-7 in 320), of one sign 1.1e-8 in chains of 160, 1.4e-8 in 320 (4.5e-6), 3.9e-8 in 4,096 (1.6e-4), 6.8e-8 in 16,384 (1.1e-3), 1.1e-7 in 65,536
// (7.4e-3). Chains are therefore cut after chain_limit k-blocks and the pieces added in registers with ordinary rounding. 32-bit outputs: 320 additions (K of
// 10,240), half of that under an activation, since a square or a product of two sums has twice the error of one (inner size 18,944, squared: 1.2e-6 with
// 320, 4.9e-7 with 160, and 777 x 4,096 57.3 -> 58.9 us). More cuts cost more than they give: reading the sums takes the products' time in TMEM, about a
// microsecond (2,048 x 5,120 x 5,120 into a 32-bit stream: cut after 64 additions 64 us, after 128 60, uncut 52). bfloat16 outputs: 1,024 additions (K of
// 32,768, so that a layer's products run uncut), which take less than a hundredth of what the output's own rounding does (2^-9 to 2^-8).
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "packs.cuh"

namespace float8 {

constexpr float kLargest = 448.f;             // of e4m3
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126: a row of zeros has this scale and no quotient overflows
constexpr int kRowsW = 128;                   // rows of W a block holds: TMEM lanes
constexpr int kBlockK = 128;                  // k per stage: 128 bytes, one swizzle row
constexpr int kMmaK = 32;
constexpr long long kWaitCycles = 4000000000LL;  // about two seconds
constexpr int ERRBIT_TIMEOUT = 8;

// KIND of a product's epilogue; ACTIVATED and GATED take their function from Epilogue::activation.
enum : int { PLAIN = 0, ACTIVATED = 1, GATED = 2 };
// k-blocks a chain of products runs over at most.
constexpr int chain_limit(int kind, bool out_f32) { return !out_f32 ? 256 : kind == PLAIN ? 80 : 40; }
enum : int { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU = 2, ACT_SQUARED_RELU = 3 };

struct Epilogue {
  void* out;
  const float* x_scale;   // [M]
  const float* w_scale;   // [N]
  const float* bias;      // [N] or null
  const float* residual;  // [M, N] or null (may be `out` itself)
  int64_t out_stride;     // elements from row to row
  int64_t residual_stride;
  int M, N;
  int activation;
  int vector;  // four neighbouring outputs of a row can be written (and residuals read) at once: strides and bases allow it
};

__device__ __forceinline__ float activate(float v, int activation) {
  if (activation == ACT_SILU) return gated_unit<false>(v, 1.f);
  if (activation == ACT_GELU) return gated_unit<true>(v, 1.f);
  const float r = v < 0.f ? 0.f : v;  // NaN stays
  return r * r;
}

// Four neighbouring outputs (n a multiple of four, rows of W beyond the last left out): the residual's, and from four sums with their scales and bias.
__device__ __forceinline__ float4 residual_quad(const Epilogue& e, int m, int n) {
  const float* from = e.residual + m * e.residual_stride + n;
  if (e.vector && n + 3 < e.N) return *reinterpret_cast<const float4*>(from);
  return make_float4(n < e.N ? from[0] : 0.f, n + 1 < e.N ? from[1] : 0.f, n + 2 < e.N ? from[2] : 0.f, n + 3 < e.N ? from[3] : 0.f);
}
__device__ __forceinline__ float4 activate_quad(float4 v, int activation) {
  return make_float4(activate(v.x, activation), activate(v.y, activation), activate(v.z, activation), activate(v.w, activation));
}
__device__ __forceinline__ float2 gated_pair(float4 v, int activation) {  // gate, up, gate, up
  return activation == ACT_GELU ? make_float2(gated_unit<true>(v.x, v.y), gated_unit<true>(v.z, v.w))
                                : make_float2(gated_unit<false>(v.x, v.y), gated_unit<false>(v.z, v.w));
}
// Four finished numbers (gated: still gates and up values) to their place: all of them on an aligned place, or those that belong to rows of W.
template <int KIND, typename T>
__device__ __forceinline__ void store_whole(T* to, float4 v, int activation) {
  if constexpr (KIND == GATED) {
    const float2 y = gated_pair(v, activation);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(to) = y;
    else *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(y.x, y.y);
  } else {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(to) = v;
    } else {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(to) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
}
template <int KIND, typename T>
__device__ __noinline__ void store_some(T* to, int n, int N, float4 v, int activation) {
  if constexpr (KIND == GATED) {
    const float2 y = gated_pair(v, activation);
    if (n < N) to[0] = from_f32<T>(y.x);
    if (n + 2 < N) to[1] = from_f32<T>(y.y);
  } else {
    if (n < N) to[0] = from_f32<T>(v.x);
    if (n + 1 < N) to[1] = from_f32<T>(v.y);
    if (n + 2 < N) to[2] = from_f32<T>(v.z);
    if (n + 3 < N) to[3] = from_f32<T>(v.w);
  }
}

// Two 32-bit numbers at once.
__device__ __forceinline__ float2 mul_2(float2 a, float2 b) {
  float2 r;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 z, x, y;\nmov.b64 {%0, %1}, z;\n}\n" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma_2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// A warp's way out of TMEM: 32 neighbouring rows of W, one a lane (n0: lane 0's, a multiple of 32), for tokens m0, m0 + 1, ..., eight at a time. The
// numbers pass through `stage`, 1 KB of shared memory of the warp's own, so that a lane goes on with four neighbouring rows of one token: a
// quarter of the stores, addresses and conditions, and gates beside their up values. (Neighbours that trade numbers by shuffles took 13
// instructions an output and 3.6 us for the 128 x 256 sums of an SM, eight warps; this takes under five.) Where rows of the output start anywhere, and at its
// edges, each lane stores its own row's numbers one by one, 32 neighbours of an output row a warp (774 tokens of 27,055 x 5,056 into 32 bits 107 us; with quads
// stored one by one 123). The whole warp calls this.
constexpr int kStageFloats = 8 * 32;
template <int KIND, typename T>
class WayOut {
 public:
  // apart: tokens from one eight to the next.
  __device__ __forceinline__ WayOut(const Epilogue& e, int m0, int n0, float* stage, int apart = 8) : e_(e), stage_(stage), apart_(apart), m_(m0), n0_(n0) {
    const int lane = threadIdx.x & 31;
    ws_ = b_ = 0.f;
    if (n0 + lane < e.N) {
      ws_ = e.w_scale[n0 + lane];
      if (e.bias != nullptr) b_ = e.bias[n0 + lane];
    }
    whole_ = e.vector && n0 + 31 < e.N;
    const int m = m0 + (lane >> 3), n = n0 + (lane & 7) * 4;  // this lane's tokens: m, m + 4 of each eight
    to_ = static_cast<T*>(e.out) + m * e.out_stride + (KIND == GATED ? n >> 1 : n);
    from_ = e.residual != nullptr ? e.residual + m * e.residual_stride + n : nullptr;
    ask();
  }

  // The next eight tokens; `v`: sums without scales, `xs`: the tokens' scales (16-byte aligned).
  __device__ __forceinline__ void take(const float* xs, const float (&v)[8]) {
    const int lane = threadIdx.x & 31;
    const int m = m_, left = e_.M - m;
    const bool whole = whole_ && left >= 8;
    const bool add = KIND != GATED && e_.residual != nullptr;
    float r[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = residual_[i];
    m_ += apart_;
    if (add) {
      from_ += apart_ * e_.residual_stride;
      ask();
    }
    const float2 ws = make_float2(ws_, ws_), b = make_float2(b_, b_);
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 s = *reinterpret_cast<const float4*>(xs + i);
      const float2 lo = fma_2(mul_2(make_float2(v[i], v[i + 1]), make_float2(s.x, s.y)), ws, b);
      const float2 hi = fma_2(mul_2(make_float2(v[i + 2], v[i + 3]), make_float2(s.z, s.w)), ws, b);
      y[i] = lo.x, y[i + 1] = lo.y, y[i + 2] = hi.x, y[i + 3] = hi.y;
    }
    if (whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) stage_[i * 32 + lane] = y[i];
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float4 mine = *reinterpret_cast<const float4*>(stage_ + (q * 4 + (lane >> 3)) * 32 + (lane & 7) * 4);
        if constexpr (KIND == ACTIVATED) mine = activate_quad(mine, e_.activation);
        if (add) mine = add_each(mine, make_float4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]));
        store_whole<KIND, T>(to_ + q * 4 * e_.out_stride, mine, e_.activation);
      }
      __syncwarp();
    } else {
      const int n = n0_ + lane;
      if constexpr (KIND == GATED) {
        // Neighbours trade one of two tokens: an even lane has the gate and up value of the first, the odd one beside it those of the second.
        const bool odd = lane & 1;
        T* to = static_cast<T*>(e_.out) + (m + odd) * e_.out_stride + (n >> 1);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float other = __shfl_xor_sync(0xffffffffu, odd ? y[i] : y[i + 1], 1);
          const float gate = odd ? other : y[i], up = odd ? y[i + 1] : other;
          if (n < e_.N && i + odd < left) to[i * e_.out_stride] = from_f32<T>(e_.activation == ACT_GELU ? gated_unit<true>(gate, up) : gated_unit<false>(gate, up));
        }
      } else {
        T* to = static_cast<T*>(e_.out) + m * e_.out_stride + n;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (KIND == ACTIVATED) y[i] = activate(y[i], e_.activation);
          if (n < e_.N && i < left) to[i * e_.out_stride] = from_f32<T>(add ? y[i] + r[i] : y[i]);
        }
      }
    }
    to_ += apart_ * e_.out_stride;
  }

 private:
  // The residual's numbers for the next eight tokens, before anything waits for them: as this lane's quads have them, or its own row's.
  __device__ __forceinline__ void ask() {
    if (KIND == GATED || e_.residual == nullptr) return;
    const int lane = threadIdx.x & 31, left = e_.M - m_;
    if (whole_ && left >= 8) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float4 f = *reinterpret_cast<const float4*>(from_ + q * 4 * e_.residual_stride);
        residual_[4 * q] = f.x, residual_[4 * q + 1] = f.y, residual_[4 * q + 2] = f.z, residual_[4 * q + 3] = f.w;
      }
    } else {
      const float* from = e_.residual + m_ * e_.residual_stride + n0_ + lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) residual_[i] = n0_ + lane < e_.N && i < left ? from[i * e_.residual_stride] : 0.f;
    }
  }

  const Epilogue& e_;
  float* stage_;
  int apart_, m_, n0_;
  float ws_, b_;
  bool whole_;
  T* to_;
  const float* from_;
  float residual_[8];
};

// --- shared memory, TMA, tcgen05 -------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// Bounded wait for the phase with the given parity to complete.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_addr(bar);
  const long long start = clock64();
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if (clock64() - start > kWaitCycles) return false;
  }
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_addr(dst)),
               "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y)
               : "memory");
}

// Shared-memory matrix descriptor of a K-major tile with 128-byte rows and 128-byte swizzle: groups of 8 rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);  // start address
  desc |= static_cast<uint64_t>(1) << 16;                 // leading byte offset (unused for swizzled K-major)
  desc |= static_cast<uint64_t>(1024 >> 4) << 32;         // stride byte offset
  desc |= static_cast<uint64_t>(1) << 46;                 // descriptor version (sm_100)
  desc |= static_cast<uint64_t>(2) << 61;                 // SWIZZLE_128B
  return desc;
}
// Instruction descriptor: e4m3 x e4m3 (format 0 of kind::f8f6f4) -> fp32, both operands K-major.
__device__ __forceinline__ uint32_t instr_desc(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(chosen));
  return chosen != 0;
}
// Eight columns of this warp's 32 TMEM lanes, a lane per thread: asked for, and there once tmem_wait has returned.
__device__ __forceinline__ void tmem_ask(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait(float (&v)[8]) {  // the numbers go through it, so that none is used before
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t taddr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The same eight columns of `chains` accumulators, `apart` columns from one to the next, added in order; and of two places at once.
__device__ __forceinline__ void tmem_sums(uint32_t taddr, int chains, int apart, float (&v)[8]) {
  tmem_ask(taddr, v);
  tmem_wait(v);
  for (int c = 1; c < chains; ++c) {
    float more[8];
    tmem_ask(taddr + c * apart, more);
    tmem_wait(more);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += more[i];
  }
}
__device__ __forceinline__ void tmem_sums(uint32_t first, uint32_t second, int chains, int apart, float (&v)[2][8]) {
  tmem_ask(first, v[0]);
  tmem_ask(second, v[1]);
  tmem_wait(v[0]);
  tmem_wait(v[1]);
  for (int c = 1; c < chains; ++c) {
    float more[2][8];
    tmem_ask(first + c * apart, more[0]);
    tmem_ask(second + c * apart, more[1]);
    tmem_wait(more[0]);
    tmem_wait(more[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[h][i] += more[h][i];
  }
}

// --- host ------------------------------------------------------------------------------------------

// A [rows, K] matrix of bytes, rows `stride` bytes apart, as a 2-D tensor map with boxes of 128 k x box_rows rows; zeros beyond its edges.
int make_map(CUtensorMap* map, const void* base, int rows, int K, int64_t stride, int box_rows);

// The work of one call, the same for both kernels.
struct Product {
  const void* x;
  const void* w;
  int64_t x_stride, w_stride;  // bytes from row to row
  int K;
  int kind, out_f32;
  int w_constant;  // nothing on the stream still writes W or its scales: they may be fetched before the kernel in front has ended
  Epilogue e;
  int* err;
};

// csrc/kernels/gemm_float8_skinny.cu: up to 16 tokens and a short stream of weights.
bool skinny_takes(int M, int N, int K);
int launch_skinny(const Product& p, cudaStream_t stream);
// csrc/kernels/gemm_float8_stream.cu: weights streamed past few tokens, K split inside clusters.
constexpr float kNever = 1e30f;
float stream_time(const Product& p);
int launch_stream(const Product& p, cudaStream_t stream);
// csrc/kernels/gemm_float8_tiles.cu: pairs of SMs on tiles of 256 rows of W by `tile` tokens (64 to 256, a multiple of 32).
float tiles_time(const Product& p, int tile);
int launch_tiles(const Product& p, int tile, cudaStream_t stream);

}  // namespace float8
