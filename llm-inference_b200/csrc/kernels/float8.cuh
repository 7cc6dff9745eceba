// What the kernels over 8-bit rows share: the e4m3 format, the epilogue of their products and the tcgen05 / TMA pieces.
//
// A matrix in 8 bits is a `Float8Rows` (parts/float8.py): e4m3 numbers q[row][k], rows a multiple of 16 bytes apart, and one 32-bit scale a
// row; the number at (row, k) is q * scale. A product of two such matrices has both scales in front of the sum:
//   y[m][n] = (sum_k x[m][k] w[n][k]) * xs[m] * ws[n].
// A product of two e4m3 numbers has 8 bits, so every product is exact; sums are 32-bit. `tcgen05.mma` drops the bits below the last when it
// adds (toward zero), which over a chain of n additions makes a sum smaller by about n 2^-25 of itself: 1e-5 after the 592 additions of
// K = 18,944. Where outputs are 32-bit the chains are therefore cut (kChainBlocks) and the pieces added in registers with ordinary
// rounding; a bfloat16 output's own rounding (2^-9) is a hundred times what an uncut chain loses.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace float8 {

constexpr float kLargest = 448.f;             // of e4m3
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126: a row of zeros has this scale and no quotient overflows
constexpr int kRowsW = 128;                   // rows of W a block holds: TMEM lanes
constexpr int kBlockK = 128;                  // k per stage: 128 bytes, one swizzle row
constexpr int kMmaK = 32;
constexpr int kChainBlocks = 4;               // 32-bit outputs: k-blocks a chain runs over (16 additions: 5e-7 of a sum at most)
constexpr long long kWaitCycles = 4000000000LL;  // about two seconds
constexpr int ERRBIT_TIMEOUT = 8;

// KIND of a product's epilogue; ACTIVATED and GATED take their function from Epilogue::activation.
enum : int { PLAIN = 0, ACTIVATED = 1, GATED = 2 };
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
  int pairs;  // rows can be written two numbers at a time: N and the stride even, the base on two numbers' boundary
};

__device__ __forceinline__ float activate(float v, int activation) {
  if (activation == ACT_SILU) return gated_unit<false>(v, 1.f);
  if (activation == ACT_GELU) return gated_unit<true>(v, 1.f);
  const float r = v < 0.f ? 0.f : v;  // NaN stays
  return r * r;
}
// `COUNT` sums with their scales and bias through the activation; the choice is the call's, so it is made once.
template <int COUNT>
__device__ __forceinline__ void activate_all(float (&v)[COUNT], int activation) {
  if (activation == ACT_SQUARED_RELU) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = activate(v[i], ACT_SQUARED_RELU);
  } else if (activation == ACT_SILU) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = activate(v[i], ACT_SILU);
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = activate(v[i], ACT_GELU);
  }
}

// COUNT tokens from m0 on, one per entry of `v` (sums without scales), for the row of W that this lane holds (n; 32 neighbouring rows a
// warp, even for lane 0). `xs` are the tokens' scales (16-byte aligned), ws and b the row's own. Rows are features, so a warp's store covers 32
// neighbours of one output row. bfloat16 neighbours trade one of two tokens with the lane beside them, and each then stores 4 bytes instead of two
// times 2; in gated products the same trade brings a gate and its up value together. All of it is straight-line code, the residual asked for
// first: with a branch per pair of tokens, and each residual number loaded where it is added, a tile of 128 x 256 took 8 us instead of 2.
// The whole warp calls this.
template <int KIND, typename T, int COUNT>
__device__ __forceinline__ void finish_columns(const Epilogue& e, const float* xs, float ws, float b, int m0, int n, float (&v)[COUNT]) {
  const bool odd = threadIdx.x & 1, live = n < e.N;
  const int count = min(COUNT, e.M - m0);  // tokens there are
  float r[COUNT];
  const bool add = KIND != GATED && e.residual != nullptr;
  if (add) {
    const float* from = e.residual + m0 * e.residual_stride + n;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) r[i] = live && i < count ? from[i * e.residual_stride] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < COUNT; i += 4) {
    const float4 s = *reinterpret_cast<const float4*>(xs + i);
    v[i] = fmaf(v[i] * s.x, ws, b);
    v[i + 1] = fmaf(v[i + 1] * s.y, ws, b);
    v[i + 2] = fmaf(v[i + 2] * s.z, ws, b);
    v[i + 3] = fmaf(v[i + 3] * s.w, ws, b);
  }
  if constexpr (KIND == ACTIVATED) activate_all<COUNT>(v, e.activation);
  if (add) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] += r[i];
  }
  T* to = static_cast<T*>(e.out) + m0 * e.out_stride;
  if constexpr (KIND == GATED) {
    float y[COUNT / 2];  // this lane's gate-and-up pairs: tokens 2 i + odd
#pragma unroll
    for (int i = 0; i < COUNT; i += 2) {
      const float other = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[i + 1], 1);
      const float gate = odd ? other : v[i], up = odd ? v[i + 1] : other;
      v[i] = gate;
      v[i + 1] = up;
    }
    if (e.activation == ACT_GELU) {
#pragma unroll
      for (int i = 0; i < COUNT / 2; ++i) y[i] = gated_unit<true>(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < COUNT / 2; ++i) y[i] = gated_unit<false>(v[2 * i], v[2 * i + 1]);
    }
    to += odd * e.out_stride + (n >> 1);
#pragma unroll
    for (int i = 0; i < COUNT / 2; ++i)
      if (live && 2 * i + odd < count) to[2 * i * e.out_stride] = from_f32<T>(y[i]);
  } else if (sizeof(T) == 2 && e.pairs) {
    __nv_bfloat16* at = reinterpret_cast<__nv_bfloat16*>(to) + odd * e.out_stride + (n & ~1);
#pragma unroll
    for (int i = 0; i < COUNT; i += 2) {
      const float other = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[i + 1], 1);
      if (live && i + odd < count)
        *reinterpret_cast<__nv_bfloat162*>(at + i * e.out_stride) = odd ? __floats2bfloat162_rn(other, v[i + 1]) : __floats2bfloat162_rn(v[i], other);
    }
  } else {
    to += n;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      if (live && i < count) to[i * e.out_stride] = from_f32<T>(v[i]);
  }
}

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
// 16 columns of this warp's 32 TMEM lanes, a lane per thread: asked for, and there once tmem_wait has returned.
__device__ __forceinline__ void tmem_ask_16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait(float (&v)[16]) {  // the numbers go through it, so that none is used before
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}
// The same 16 columns of `chains` accumulators, `apart` columns from one to the next, added in order.
__device__ __forceinline__ void tmem_sums_16(uint32_t taddr, int chains, int apart, float (&v)[16]) {
  tmem_ask_16(taddr, v);
  tmem_wait(v);
  for (int c = 1; c < chains; ++c) {
    float more[16];
    tmem_ask_16(taddr + c * apart, more);
    tmem_wait(more);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += more[i];
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

// csrc/kernels/gemm_float8_stream.cu: weights streamed past few tokens, K split inside clusters.
int launch_stream(const Product& p, cudaStream_t stream);
// csrc/kernels/gemm_float8_tiles.cu: pairs of SMs on tiles of 256 rows of W by up to 256 tokens.
int launch_tiles(const Product& p, int tile, cudaStream_t stream);

}  // namespace float8
