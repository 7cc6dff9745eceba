// Product of 8-bit rows for many tokens: pairs of SMs on tiles of 256 rows of W by up to 256 tokens.
//   y[m][n] = act((sum_k x[m][k] w[n][k]) xs[m] ws[n] + bias[n]) + residual[m][n],  or act(gate) * up over pairs of W's rows.
//
// The two blocks of a cluster are one `tcgen05.mma.cta_group::2` (kind::f8f6f4): each holds 128 of the tile's rows of W and half of its tokens in
// shared memory and 128 rows of the sums in TMEM, so what an SM takes out of L2 for 128 k is 16 KB of W and 16 KB of X for 128 x 256 sums, where a
// block by itself would need 48. Persistent: a cluster per two SMs walks over the tiles. In each block one thread fills a ring of stages by TMA
// (both blocks' copies are counted on the leader's barriers), in the leader one thread issues the products, and sixteen warps per block read the
// sums of one tile while the next is made in the other half of TMEM. A lane has one row of W and a quarter of the tile's tokens: scales and bias of
// the row are the lane's own; on their way out the numbers change places inside a warp (WayOut in float8.cuh).
//
// After each chain of k-blocks (chain_limit in float8.cuh) the warps add the sums to registers and the products go on in the other half. bfloat16 outputs have
// a form without that, for rows of one chain.
//
// Tiles are taken in strips of a few token tiles across all rows of W, so that at any time the clusters share a few rows of both operands in L2.
// TMEM, all of it, is taken before the kernel in front has ended: shared memory leaves no room for a block of it that still wants some. Every wait is bounded: a role that
// gives up sets the timeout bit and leaves its loop; copies in flight are waited for, and both blocks meet before either leaves. (Asking for the first
// tile's weights before the kernel in front has ended gains nothing here: 2,048 tokens of 4,608 x 3,584 behind a norm 34.0 us with it, 33.7 without.)
#include "float8.cuh"

namespace float8 {
namespace {

constexpr int kPairRows = 2 * kRowsW;     // rows of W of a tile: MMA M
constexpr int kMostTokens = 256;          // tokens of a tile: MMA N, a multiple of 32
constexpr int kSumWarps = 16;                   // four a quarter of the TMEM lanes
constexpr int kThreads = (2 + kSumWarps) * 32;  // warp 0: TMA, warp 1: MMA, 2-17: sums
constexpr int kMaxStages = 10;
constexpr int kStrip = 8;                 // token tiles of a strip
constexpr size_t kRingBytes = 6 * 32 * 1024;

struct TileParams {
  Epilogue e;
  int* err;
  int K;
  int stages;
  int tile;          // tokens
  int chain_blocks;  // k-blocks between two readings of the sums
};

__device__ __forceinline__ uint32_t of_leader(const void* p) { return peer_address(p, 0); }

// A copy into this block's shared memory, counted on the leader's barrier.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t leader_bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                   smem_addr(dst)),
               "l"(map), "r"(leader_bar), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
// Arrives on the barrier of both blocks once all products issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
// What it says is that TMEM has been read (tcgen05.wait::ld has returned); with release it would wait for all stores of the warp, 1,000 cycles.
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// Tile `at` of the order described above: its token tile and its rows-of-W tile.
__device__ __forceinline__ void locate(int at, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int strip = at / (kStrip * tiles_n), first = strip * kStrip;
  const int height = min(kStrip, tiles_m - first);
  const int in = at - strip * kStrip * tiles_n;
  tn = in / height;
  tm = first + in - tn * height;
}

template <int KIND, typename T, bool CHAINED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
float8_tiles_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const TileParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t w_bytes = kRowsW * kBlockK;
  const uint32_t x_bytes = static_cast<uint32_t>(p.tile / 2) * kBlockK;
  const uint32_t stage_bytes = w_bytes + ((x_bytes + 1023u) & ~1023u);
  unsigned char* tiles = smem_raw + (-smem_addr(smem_raw) & 1023u);
  __shared__ __align__(8) uint64_t full_bar[kMaxStages];
  __shared__ __align__(8) uint64_t empty_bar[kMaxStages];
  __shared__ __align__(8) uint64_t sums_full[2];
  __shared__ __align__(8) uint64_t sums_empty[2];
  __shared__ uint32_t tmem_base_shared;
  __shared__ __align__(16) float x_scales[2][kMostTokens];
  __shared__ __align__(16) float stages_out[kSumWarps * kStageFloats];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  const int stages = p.stages;
  const int tiles_m = (p.e.M + p.tile - 1) / p.tile, tiles_n = (p.e.N + kPairRows - 1) / kPairRows;
  const int total = tiles_m * tiles_n;
  const int k_blocks = (p.K + kBlockK - 1) / kBlockK;
  const int links = CHAINED ? (k_blocks + p.chain_blocks - 1) / p.chain_blocks : 1;  // readings of a tile's sums

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sums_full[b], 1);
      mbar_init(&sums_empty[b], 2 * kSumWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_base_shared)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync_all();  // the other block's barriers are there
  wait_for_predecessor();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  let_successor_start();
  const uint32_t tmem_base = tmem_base_shared;

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t leader_full = of_leader(full_bar);
      int s = 0, phase = 0;
      int64_t sent = 0;
      bool alive = true;
      for (int at = cluster; at < total && alive; at += clusters) {
        int tm, tn;
        locate(at, tiles_m, tiles_n, tm, tn);
        const int wy = tn * kPairRows + rank * kRowsW, xy = tm * p.tile + rank * (p.tile / 2);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty_bar[s], phase ^ 1)) {  // passes at once the first time round
            atomicOr(p.err, ERRBIT_TIMEOUT);
            alive = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * (w_bytes + x_bytes));
          unsigned char* stage = tiles + s * stage_bytes;
          tma_load_pair(stage, &w_map, leader_full + s * 8, kb * kBlockK, wy);
          tma_load_pair(stage + w_bytes, &x_map, leader_full + s * 8, kb * kBlockK, xy);
          ++sent;
          if (++s == stages) s = 0, phase ^= 1;
        }
      }
      if (alive) {  // the last products have read their stages and said so
        for (int i = 0; i < stages; ++i) {
          if (!mbar_wait(&empty_bar[s], phase ^ 1)) break;
          if (++s == stages) s = 0, phase ^= 1;
        }
      } else if (rank == 0) {  // both blocks' copies in flight
        for (int64_t i = max(int64_t(0), sent - stages); i < sent; ++i) mbar_wait(&full_bar[i % stages], (i / stages) & 1);
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool chosen = elect_one();
      const uint32_t idesc = instr_desc(kPairRows, p.tile);
      const uint64_t a_first = smem_desc(smem_addr(tiles)), b_first = smem_desc(smem_addr(tiles) + w_bytes);
      int s = 0, phase = 0, item = 0;
      bool alive = true;
      for (int at = cluster; at < total && alive; at += clusters) {
        for (int link = 0, kb = 0; link < links && alive; ++link, ++item) {
          const int half = item & 1;
          if (!mbar_wait(&sums_empty[half], ((item >> 1) & 1) ^ 1)) {
            alive = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sums = tmem_base + half * kMostTokens;
          const int end = CHAINED ? min(k_blocks, kb + p.chain_blocks) : k_blocks;
          for (const int begin = kb; kb < end; ++kb) {
            if (!mbar_wait(&full_bar[s], phase)) {
              alive = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t stage_units = static_cast<uint64_t>(s) * (stage_bytes >> 4);
#pragma unroll
            for (int k = 0; k < kBlockK / kMmaK; ++k) {
              const uint64_t step = stage_units + static_cast<uint64_t>(k * (kMmaK >> 4));
              if (chosen) umma_pair(sums, a_first + step, b_first + step, idesc, kb > begin || k > 0);
            }
            if (chosen) umma_commit_pair(&empty_bar[s]);
            __syncwarp();
            if (++s == stages) s = 0, phase ^= 1;
          }
          if (chosen) umma_commit_pair(&sums_full[half]);
          __syncwarp();
        }
      }
      if (!alive && chosen) atomicOr(p.err, ERRBIT_TIMEOUT);
    }
  } else {
    const int quarter = warp & 3;             // TMEM lanes 32 * quarter .. + 31 belong to this warp
    const int side = (warp - 2) >> 2;         // which quarter of the tokens
    const int width = p.tile / 4;             // a multiple of 8
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + side * width;
    const uint32_t leader_empty = of_leader(sums_empty);
    const int tid = threadIdx.x - 64;
    float* stage = stages_out + (warp - 2) * kStageFloats;
    int item = 0;
    bool alive = true;
    for (int at = cluster, turn = 0; at < total; at += clusters, turn ^= 1) {  // to the end even after giving up: the warps meet once a tile
      int tm, tn;
      locate(at, tiles_m, tiles_n, tm, tn);
      const int m0 = tm * p.tile;
      const int n0 = tn * kPairRows + rank * kRowsW + quarter * 32;
      // The tile's token scales, for all warps; the copy of two tiles ago is read by nobody any more (a warp meets the others once a tile).
      if (tid < p.tile) x_scales[turn][tid] = m0 + tid < p.e.M ? p.e.x_scale[m0 + tid] : 0.f;
      const float* xs = x_scales[turn] + side * width;
      // The residual's lines of the tile, a token each: they come from memory while the products run.
      if (KIND != GATED && p.e.residual != nullptr && n0 < p.e.N)
        for (int i = lane; i < width; i += 32)
          if (m0 + side * width + i < p.e.M) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.e.residual + (m0 + side * width + i) * p.e.residual_stride + n0));
      // Waits for a tile's (or a chain's) sums and says where in TMEM they are.
      auto sums_of = [&](int which) {
        alive = alive && mbar_wait(&sums_full[which & 1], (which >> 1) & 1);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        return lanes + (which & 1) * kMostTokens;
      };
      auto sums_read = [&](int which) {  // they are in registers: the products after next may go there
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive_at(leader_empty + (which & 1) * 8);
      };
      auto finish = [&](WayOut<KIND, T>& way, uint32_t from) {
        for (int c = 0; c < width; c += 8) {
          float v[8];
          tmem_ask(from + c, v);
          tmem_wait(v);
          if (c + 8 >= width) sums_read(item);
          way.take(xs + c, v);
        }
      };
      if constexpr (!CHAINED) {
        WayOut<KIND, T> way(p.e, m0 + side * width, n0, stage);
        asm volatile("bar.sync 1, 512;" ::: "memory");
        const uint32_t from = sums_of(item);
        if (alive) finish(way, from);
        ++item;
      } else {
        asm volatile("bar.sync 1, 512;" ::: "memory");
        uint32_t from = lanes;
        if (links > 1) {  // the chains in registers; with the last one back to where that lies
          float acc[kMostTokens / 32][8];
          for (int link = 0; link < links; ++link) {
            from = sums_of(item + link);
            if (!alive) break;
#pragma unroll
            for (int g = 0; g < kMostTokens / 32; ++g) {
              if (g * 8 < width) {
                float v[8];
                tmem_ask(from + g * 8, v);
                tmem_wait(v);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[g][i] = link > 0 ? acc[g][i] + v[i] : v[i];
                if (link == links - 1) tmem_store(from + g * 8, acc[g]);
              }
            }
            if (link < links - 1) sums_read(item + link);
          }
          tmem_stored();
          item += links - 1;
        } else {
          from = sums_of(item);
        }
        WayOut<KIND, T> way(p.e, m0 + side * width, n0, stage);
        if (alive) finish(way, from);
        ++item;
      }
    }
    if (!alive && lane == 0) atomicOr(p.err, ERRBIT_TIMEOUT);
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync_all();  // nothing of the other block's still arrives here
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

using TileKernel = void (*)(const CUtensorMap, const CUtensorMap, const TileParams);

template <typename T, bool CHAINED>
TileKernel pick_kind(int kind) {
  return kind == GATED       ? float8_tiles_kernel<GATED, T, CHAINED>
         : kind == ACTIVATED ? float8_tiles_kernel<ACTIVATED, T, CHAINED>
                             : float8_tiles_kernel<PLAIN, T, CHAINED>;
}

}  // namespace

// Microseconds, roughly, with tiles of `tile` tokens: a launch, k-blocks one after the other (or what all clusters take out of L2 at 8.5 TB/s) and a
// tile's way out, the last one's in full; fitted to 17 to 4,096 tokens of eleven matrices.
float tiles_time(const Product& p, int tile) {
  const int k_blocks = (p.K + kBlockK - 1) / kBlockK, clusters = b200_sm_count_host() / 2;
  const int64_t tiles = static_cast<int64_t>((p.e.M + tile - 1) / tile) * ((p.e.N + kPairRows - 1) / kPairRows);
  const float way_out = p.out_f32 ? 1.5f + tile * 0.0145f : 0.5f + tile * 0.0085f;
  const int limit = chain_limit(p.kind, p.out_f32 != 0);
  const float links = k_blocks > limit ? 1.f + 4.f / limit : 1.f;
  const float turns = static_cast<float>((tiles + clusters - 1) / clusters) * max(k_blocks * (0.21f + 0.0004f * tile) * links, way_out);
  const float all = static_cast<float>(tiles) * k_blocks * (kPairRows + tile) * kBlockK / 8.5e6f * links;
  return 3.3f + max(turns, all) + way_out;
}

int launch_tiles(const Product& product, int tile, cudaStream_t stream) {
  const Epilogue& e = product.e;
  TileParams p;
  p.e = e;
  p.err = product.err;
  p.K = product.K;
  p.tile = tile;
  const int k_blocks = (product.K + kBlockK - 1) / kBlockK, limit = chain_limit(product.kind, product.out_f32 != 0), chains = (k_blocks + limit - 1) / limit;
  p.chain_blocks = (k_blocks + chains - 1) / chains;
  const int stage = kRowsW * kBlockK + ((tile / 2 * kBlockK + 1023) & ~1023);
  p.stages = min(kMaxStages, static_cast<int>(kRingBytes / stage));
  CUtensorMap w_map, x_map;
  if (make_map(&w_map, product.w, e.N, product.K, product.w_stride, kRowsW) != 0) return -1;
  if (make_map(&x_map, product.x, e.M, product.K, product.x_stride, tile / 2) != 0) return -1;
  const int form = product.out_f32 ? 0 : chains > 1 ? 1 : 2;
  const TileKernel kernel = form == 0   ? pick_kind<float, true>(product.kind)
                            : form == 1 ? pick_kind<__nv_bfloat16, true>(product.kind)
                                        : pick_kind<__nv_bfloat16, false>(product.kind);
  constexpr size_t smem = kRingBytes + 1024;
  static OncePerDevice prepared[9];
  if (!prepared[product.kind * 3 + form](
          [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) == cudaSuccess; }))
    return b200_fail("float8 product: the kernel's attributes could not be set");
  const int tiles = (e.M + tile - 1) / tile * ((e.N + kPairRows - 1) / kPairRows);
  const int clusters = min(tiles, b200_sm_count_host() / 2);
  const cudaError_t status = launch_kernel(kernel, dim3(2 * clusters), dim3(kThreads), smem, stream, w_map, x_map, p);
  if (status != cudaSuccess) {
    cudaGetLastError();
    return b200_fail("float8 product: %s", cudaGetErrorString(status));
  }
  return 0;
}

}  // namespace float8
