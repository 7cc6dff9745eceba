// Product of 8-bit rows for few tokens: the weights stream past the tensor cores once, K split inside thread-block clusters.
//   y[m][n] = act((sum_k x[m][k] w[n][k]) xs[m] ws[n] + bias[n]) + residual[m][n],  or act(gate) * up over pairs of W's rows.
//
// W is the wide operand: a block owns 128 rows of W (the MMA's M) and a tile of up to 128 tokens (its N, a multiple of 16). One thread fills a ring
// of stages by TMA (128 rows x 128 bytes of W, tokens x 128 bytes of X, 128-byte swizzle), one issues `tcgen05.mma` (kind::f8f6f4, 32 k an
// instruction) into TMEM, eight warps read the sums back, a lane per row of W. Where W has too few rows to give every SM work, the blocks of a
// cluster share rows and split K: each sends its partial sums to the members that finish those rows, a slice each, and the owners add in member
// order, so a sum does not depend on timing. A block puts its sums where its ring was, one bulk copy per owner takes them to an inbox behind the
// owner's ring, and the owner waits for the bytes: nobody waits for a member that has nothing to do with its rows, and the cluster meets only to
// know that barriers are there and, on leaving, that copies have been read. (64 tokens of 4,608 x 3,584: 11.1 us with the cluster meeting
// three times and single stores into neighbours' memory, 7.8 so.)
//
// Chains of k-blocks (chain_limit in float8.cuh) have an accumulator each, as far as a block's share of TMEM goes (128 columns, 256 where it
// has an SM to itself; the tile's tokens each), added up as they are read. Where that is not far enough the call is the tile form's.
//
// The first stages' weights are asked for before the kernel in front has ended where the caller says that nothing still writes them. TMEM is
// taken first thing: an SM starts no second block that takes TMEM before the first has given up the permit to (measured: with the wait for the kernel in
// front before it, the second block of every SM began 2.7 us late, with it in front 1.1 us). A block takes no larger a share of an SM's TMEM than of its
// shared memory, so a resident block never waits for another's. Every wait is bounded: a block that gives up sets the timeout bit, waits for its
// copies in flight, frees its TMEM and leaves.
#include <map>
#include <mutex>
#include <tuple>
#include <vector>

#include "float8.cuh"

namespace float8 {
namespace {

constexpr int kSumWarps = 8;       // two a quarter of the TMEM lanes
constexpr int kThreads = (2 + kSumWarps) * 32;  // warp 0: TMA, warp 1: MMA, warps 2-9: sums
constexpr int kMaxStages = 12;
constexpr int kMaxMembers = 16;
constexpr int kMaxTokens = 128;    // a block's

struct StreamParams {
  Epilogue e;
  int* err;
  int K;
  int stages;
  int tile;          // tokens of a block, a multiple of 16
  int chain_blocks;  // k-blocks per accumulator
  int tmem_cols;
  int w_constant;
  int inbox_at;      // bytes from the ring's start
};

// Rows of a block that one member of a cluster finishes: whole 32-byte pieces of 32-bit output rows (the last members may have none).
__host__ __device__ constexpr int slice_rows(int members) { return ((kRowsW + members - 1) / members + 7) & ~7; }

__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// `bytes` (a multiple of 16) from here to the same place of block `rank`, counted on that block's barrier.
__device__ __forceinline__ void copy_to_peer(float* dst, const float* src, uint32_t bytes, uint64_t* bar, int rank) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(peer_address(dst, rank)), "r"(smem_addr(src)),
               "r"(bytes), "r"(peer_address(bar, rank))
               : "memory");
}

// What one member finishes: `rows` rows of W from n0 on, the members' partial sums ([members][tokens][slice]) added in member order; `scales` and
// `bias` are those rows'. An item is four neighbouring rows of one token; a thread takes kItems of them at a time, and asks for the next ones'
// residual before it adds (the first ones' before the partial sums have come: `wait` is called then, by every thread).
template <int KIND, typename T, typename Wait>
__device__ __forceinline__ void finish_slice(const Epilogue& e, const float* inbox, const float* x_scales, const float* scales, const float* bias, int m0, int tokens,
                                             int n0, int rows, int slice, int members, int tid, Wait wait) {
  constexpr int kItems = 2, kFinishThreads = kSumWarps * 32;
  const int quads = max(0, (min(rows, e.N - n0) + 3) / 4);  // with rows of W left
  const int total = quads * tokens, plane = tokens * slice;
  int m[kItems], j[kItems];
  float4 r[kItems];
  auto ask = [&](int base) {
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int item = base + u * kFinishThreads;
      m[u] = j[u] = 0;
      r[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (item >= total) continue;
      m[u] = item / quads;
      j[u] = 4 * (item - m[u] * quads);
      if (KIND != GATED && e.residual != nullptr) r[u] = residual_quad(e, m0 + m[u], n0 + j[u]);
    }
  };
  ask(tid);
  wait();
  for (int base = tid; base < total; base += kFinishThreads * kItems) {
    float4 sum[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u) sum[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int member = 0; member < members; ++member) {
#pragma unroll
      for (int u = 0; u < kItems; ++u) sum[u] = add_each(sum[u], *reinterpret_cast<const float4*>(inbox + member * plane + m[u] * slice + j[u]));
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      if (base + u * kFinishThreads >= total) break;
      const float4 ws = *reinterpret_cast<const float4*>(scales + j[u]), b = *reinterpret_cast<const float4*>(bias + j[u]);
      float4 v = fma_each(scale_each(sum[u], x_scales[m[u]]), ws, b);
      if constexpr (KIND == ACTIVATED) v = activate_quad(v, e.activation);
      if constexpr (KIND != GATED) v = add_each(v, r[u]);
      const int n = n0 + j[u];
      T* to = static_cast<T*>(e.out) + (m0 + m[u]) * e.out_stride + (KIND == GATED ? n >> 1 : n);
      if (e.vector && n + 3 < e.N) store_whole<KIND, T>(to, v, e.activation);
      else store_some<KIND, T>(to, n, e.N, v, e.activation);
    }
    ask(base + kFinishThreads * kItems);
  }
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
// Without waiting for this thread's stores to be seen: what it says is that copies have come.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A form carries no code that it does not take: a block runs its epilogue once, from a cold instruction cache (measured in gemm_tcgen05.cu).
template <int KIND, typename T, bool CLUSTERED>
__global__ void __launch_bounds__(kThreads)
float8_stream_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const StreamParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t w_bytes = kRowsW * kBlockK;
  const uint32_t x_bytes = static_cast<uint32_t>(p.tile) * kBlockK;
  const uint32_t stage_bytes = w_bytes + ((x_bytes + 1023u) & ~1023u);
  unsigned char* tiles = smem_raw + (-smem_addr(smem_raw) & 1023u);
  __shared__ __align__(8) uint64_t full_bar[kMaxStages];
  __shared__ __align__(8) uint64_t empty_bar[kMaxStages];
  __shared__ __align__(8) uint64_t accum_bar;
  __shared__ __align__(8) uint64_t inbox_bar;
  __shared__ uint32_t tmem_base_shared;
  __shared__ __align__(16) float x_scales[kMaxTokens];
  // Clustered: the scales and bias of the rows that this member finishes. Otherwise the warps' way out of TMEM.
  __shared__ __align__(16) float rows_out[CLUSTERED ? 2 * kRowsW : kSumWarps * kStageFloats];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = p.stages;
  const int n0 = blockIdx.x * kRowsW;
  const int m0 = blockIdx.z * p.tile;
  const int members = gridDim.y, rank = blockIdx.y;
  const int k_blocks = (p.K + kBlockK - 1) / kBlockK;
  const int kb_begin = static_cast<int>(static_cast<int64_t>(k_blocks) * rank / members);
  const int num_kb = static_cast<int>(static_cast<int64_t>(k_blocks) * (rank + 1) / members) - kb_begin;  // at least one: members <= k_blocks
  const int first = min(num_kb, stages);

  auto load_w = [&](int i) { tma_load_2d(tiles + (i % stages) * stage_bytes, &w_map, &full_bar[i % stages], (kb_begin + i) * kBlockK, n0); };
  auto load_x = [&](int i) { tma_load_2d(tiles + (i % stages) * stage_bytes + w_bytes, &x_map, &full_bar[i % stages], (kb_begin + i) * kBlockK, m0); };

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base_shared)),
                 "r"(static_cast<uint32_t>(p.tmem_cols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&accum_bar, 1);
    mbar_init(&inbox_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // The thread that made the barriers also loads: the first weights are on their way before the block has met.
    if (p.w_constant)
      for (int i = 0; i < first; ++i) {
        mbar_expect_tx(&full_bar[i], w_bytes + x_bytes);
        load_w(i);
      }
  }
  if constexpr (CLUSTERED) {
    __syncwarp();
    cluster_arrive();  // this block's barriers are there
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_shared;

  if (warp == 0) {
    if (lane == 0) {
      wait_for_predecessor();
      for (int i = 0; i < first; ++i) {
        if (!p.w_constant) {
          mbar_expect_tx(&full_bar[i], w_bytes + x_bytes);
          load_w(i);
        }
        load_x(i);
      }
      int sent = first;
      for (; sent < num_kb; ++sent) {
        const int s = sent % stages;
        if (!mbar_wait(&empty_bar[s], ((sent / stages) - 1) & 1)) {
          atomicOr(p.err, ERRBIT_TIMEOUT);
          for (int i = max(0, sent - stages); i < sent; ++i) mbar_wait(&full_bar[i % stages], (i / stages) & 1);  // copies in flight
          break;
        }
        mbar_expect_tx(&full_bar[s], w_bytes + x_bytes);
        load_w(sent);
        load_x(sent);
      }
    }
  } else if (warp == 1) {
    // The whole warp walks the loop and one elected lane issues, so that descriptors stay in uniform registers.
    wait_for_predecessor();  // its limit does not run while the kernel in front does
    const bool leader = elect_one();
    const uint32_t idesc = instr_desc(kRowsW, p.tile);
    const uint64_t a_first = smem_desc(smem_addr(tiles)), b_first = smem_desc(smem_addr(tiles) + w_bytes);
    int s = 0, phase = 0, link = 0;
    uint32_t accumulator = tmem_base;
    for (int i = 0; i < num_kb; ++i) {
      if (!mbar_wait(&full_bar[s], phase)) {
        if (leader) atomicOr(p.err, ERRBIT_TIMEOUT);
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t stage_units = static_cast<uint64_t>(s) * (stage_bytes >> 4);
#pragma unroll
      for (int k = 0; k < kBlockK / kMmaK; ++k) {
        const uint64_t step = stage_units + static_cast<uint64_t>(k * (kMmaK >> 4));
        if (leader) umma(accumulator, a_first + step, b_first + step, idesc, link > 0 || k > 0);
      }
      if (leader) umma_commit(&empty_bar[s]);
      __syncwarp();
      if (++s == stages) s = 0, phase ^= 1;
      if (++link == p.chain_blocks) link = 0, accumulator += p.tile;
    }
    if (leader) umma_commit(&accum_bar);
  }
  __syncwarp();

  const int tokens = min(p.tile, p.e.M - m0);
  const int chains = (num_kb + p.chain_blocks - 1) / p.chain_blocks;
  const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31 belong to this warp, every other eight tokens too
  const int side = (warp - 2) >> 2;
  const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  const int tid = threadIdx.x - 64;  // among the warps that finish
  wait_for_predecessor();
  let_successor_start();
  if constexpr (!CLUSTERED) {
    if (warp >= 2) {
      WayOut<KIND, T> way(p.e, m0 + side * 8, n0 + quarter * 32, rows_out + (warp - 2) * kStageFloats, 16);
      if (tid < p.tile) x_scales[tid] = m0 + tid < p.e.M ? p.e.x_scale[m0 + tid] : 0.f;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const bool have = mbar_wait(&accum_bar, 0);
      if (!have && lane == 0) atomicOr(p.err, ERRBIT_TIMEOUT);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (int c0 = side * 8; have && c0 < tokens; c0 += 16) {
        float v[8];
        tmem_sums(lanes + c0, chains, p.tile, v);
        way.take(x_scales + c0, v);
      }
    }
  } else {
    cluster_wait();  // the other members' barriers are there
    const int slice = slice_rows(members);
    const int mine = rank * slice, rows = max(0, min(kRowsW - mine, slice));  // the rows this member finishes, from n0 + mine on
    float* outbox = reinterpret_cast<float*>(tiles);  // [owners][tokens][slice], where the ring was
    float* inbox = reinterpret_cast<float*>(tiles + p.inbox_at);  // [members][tokens][slice]
    const int plane = tokens * slice;
    if (warp >= 2) {
      // While the weights stream: what the finish will want.
      if (tid < p.tile) x_scales[tid] = tid < tokens ? p.e.x_scale[m0 + tid] : 0.f;
      if (tid < rows) {
        const int n = n0 + mine + tid;
        rows_out[tid] = n < p.e.N ? p.e.w_scale[n] : 0.f;
        rows_out[kRowsW + tid] = p.e.bias != nullptr && n < p.e.N ? p.e.bias[n] : 0.f;
      }
      if (KIND != GATED && p.e.residual != nullptr && tid < tokens && n0 + mine < p.e.N)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.e.residual + (m0 + tid) * p.e.residual_stride + n0 + mine));
      if (!mbar_wait(&accum_bar, 0) && lane == 0) atomicOr(p.err, ERRBIT_TIMEOUT);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int row = quarter * 32 + lane, owner = row / slice;
      float* to = outbox + owner * plane + (row - owner * slice);
      for (int c0 = side * 8; c0 < tokens; c0 += 32) {  // twice eight tokens at a time
        float v[2][8];
        const bool second = c0 + 16 < p.tile;
        tmem_sums(lanes + c0, second ? lanes + c0 + 16 : lanes + c0, chains, p.tile, v);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c0 + h * 16 + i < tokens) to[(c0 + h * 16 + i) * slice] = v[h][i];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const uint32_t bytes = static_cast<uint32_t>(plane) * sizeof(float);
      if (tid == 0 && rows > 0) mbar_expect_tx(&inbox_bar, members * bytes);
      if (tid < members && tid * slice < kRowsW) copy_to_peer(inbox + rank * plane, outbox + tid * plane, bytes, &inbox_bar, tid);  // a thread per owner
    }
    auto inbox_filled = [&] {
      __syncwarp();
      if (rows > 0 && !mbar_wait(&inbox_bar, 0) && lane == 0) atomicOr(p.err, ERRBIT_TIMEOUT);
      __syncwarp();
      cluster_arrive_relaxed();  // what was sent here has come
    };
    if (warp >= 2)
      finish_slice<KIND, T>(p.e, inbox, x_scales, rows_out, rows_out + kRowsW, m0, tokens, n0 + mine, rows, slice, members, tid, inbox_filled);
    else
      inbox_filled();
    __syncwarp();
    cluster_wait();  // what was sent from here has been read
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(static_cast<uint32_t>(p.tmem_cols)) : "memory");
  }
}

using StreamKernel = void (*)(const CUtensorMap, const CUtensorMap, const StreamParams);

template <typename T, bool CLUSTERED>
StreamKernel pick_kind(int kind) {
  return kind == GATED ? float8_stream_kernel<GATED, T, CLUSTERED>
         : kind == ACTIVATED ? float8_stream_kernel<ACTIVATED, T, CLUSTERED>
                             : float8_stream_kernel<PLAIN, T, CLUSTERED>;
}
StreamKernel pick_kernel(int kind, bool f32, bool clustered) {
  if (f32) return clustered ? pick_kind<float, true>(kind) : pick_kind<float, false>(kind);
  return clustered ? pick_kind<__nv_bfloat16, true>(kind) : pick_kind<__nv_bfloat16, false>(kind);
}

constexpr size_t kMaxDynamicSmem = 200 * 1024;

// An instantiation's opt-ins, once per device.
bool prepare_kernel(StreamKernel kernel) {
  struct Ready { StreamKernel kernel; int device; };
  static std::mutex guard;
  static std::vector<Ready> ready;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  std::lock_guard<std::mutex> lock(guard);
  for (const Ready& r : ready)
    if (r.kernel == kernel && r.device == device) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxDynamicSmem)) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  ready.push_back({kernel, device});
  return true;
}

struct StreamPlan {
  int blocks, members, tiles, tile, stages, chain_blocks, tmem_cols;
  size_t smem;
  int inbox_at;
  bool cut;  // chains are as short as they have to be
};

// How many clusters of `members` blocks run at once with one block an SM (clusters do not straddle GPCs); 0 if it cannot be told.
int clusters_one_per_sm(int members) {
  const StreamKernel kernel = pick_kernel(PLAIN, false, true);
  if (!prepare_kernel(kernel)) return 0;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(1, members * 64);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = 120 * 1024;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = 1;
  attribute.val.clusterDim.y = members;
  attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return clusters;
}

// `limit`: k-blocks of a chain; `budget`: bytes of shared memory that a block means to take.
void size_ring(StreamPlan& plan, int k_blocks, int limit, size_t budget) {
  const size_t stage = kRowsW * kBlockK + ((static_cast<size_t>(plan.tile) * kBlockK + 1023) & ~size_t(1023));
  const int per_block = (k_blocks + plan.members - 1) / plan.members;
  size_t inbox = 0, outbox = 0;
  if (plan.members > 1) {
    const int slice = slice_rows(plan.members), owners = (kRowsW + slice - 1) / slice;
    outbox = static_cast<size_t>(owners) * slice * plan.tile * sizeof(float);  // takes the ring's place
    inbox = static_cast<size_t>(plan.members) * slice * plan.tile * sizeof(float);
  }
  const size_t for_ring = budget > inbox ? budget - inbox : 0;
  plan.stages = max(2, min(min(static_cast<int>(for_ring / stage), kMaxStages), per_block));
  const size_t ring = max(plan.stages * stage, outbox);
  plan.inbox_at = static_cast<int>(ring);
  plan.smem = ring + inbox + 1024;
  // Accumulators: one per chain, as many as the block's share of TMEM holds.
  const int wanted = (per_block + limit - 1) / limit;
  const int most = budget > 114 * 1024 ? 256 : 128;
  const int accumulators = max(1, min(wanted, most / plan.tile));
  plan.chain_blocks = (per_block + accumulators - 1) / accumulators;
  plan.cut = accumulators == wanted;
  plan.tmem_cols = 32;
  while (plan.tmem_cols < accumulators * plan.tile) plan.tmem_cols *= 2;
  plan.smem = max(plan.smem, max(static_cast<size_t>(plan.tmem_cols) * 227 * 1024 / 512, static_cast<size_t>(48 * 1024)));  // see the head of the file
}

// Members share rows where there are too few blocks of 128 rows to give every SM one, as long as each keeps six or seven k-blocks to stream: below
// that the sums cost more to bring together than the stream to share (48 tokens of 2,048 x 1,536: one member 4.7 us, four 5.6).
// With more than 16 tokens a block has an SM to itself, and as many stages as that gives: two an SM hold fewer bytes in flight beside their inboxes (64
// tokens of 17,920 x 1,536: 140 blocks 7.3 us, 280 of half the size 12.1; of 4,608 x 3,584: 108 blocks 8.4 us, 216 9.8). Up to 16 tokens
// half again as many blocks as SMs (one of 4,608 x 3,584: 144 blocks 5.7 us, 216 6.2). All clusters should run at once: one that has to wait for a place
// starts when the others are done, so clusters are narrowed until they do.
StreamPlan plan_uncached(int M, int N, int K, int limit) {
  StreamPlan plan;
  plan.blocks = (N + kRowsW - 1) / kRowsW;
  plan.tiles = (M + kMaxTokens - 1) / kMaxTokens;
  plan.tile = (((M + plan.tiles - 1) / plan.tiles) + 15) / 16 * 16;
  const int k_blocks = (K + kBlockK - 1) / kBlockK;
  const int sms = b200_sm_count_host();
  const int columns = plan.blocks * plan.tiles;
  const bool alone = plan.tile > 16 && columns <= sms;
  auto fit = [&](int members, int per_sm) {  // a lower bound: s blocks an SM take clusters of m as one block an SM takes clusters of m / s
    if (members == 1) return columns <= per_sm * sms;
    const int room = clusters_one_per_sm((members + per_sm - 1) / per_sm);
    return room == 0 || columns <= room;
  };
  plan.members = max(1, min(min(kMaxMembers, k_blocks / (plan.tile > 16 ? 7 : 6)), (alone ? sms : sms + sms / 2) / columns));
  while (plan.members > 1 && !fit(plan.members, alone ? 1 : 2)) --plan.members;
  const bool one = alone || fit(plan.members, 1);
  size_ring(plan, k_blocks, limit, (one ? (alone ? 190 : 150) : columns * plan.members <= 2 * sms ? 100 : 66) * 1024);
  return plan;
}

// Plans are remembered: the occupancy question costs more than a launch. A plan goes by N, K, the padded tokens and the chains' limit only.
StreamPlan plan_stream(const Product& p) {
  static std::mutex guard;
  static std::map<std::tuple<int, int, int, int, int>, StreamPlan> known;
  int device = 0;
  cudaGetDevice(&device);
  const int rows = (p.e.M + 15) / 16 * 16, limit = chain_limit(p.kind, p.out_f32 != 0);
  const auto key = std::make_tuple(p.e.N, p.K, rows, limit, device);
  std::lock_guard<std::mutex> lock(guard);
  const auto found = known.find(key);
  if (found != known.end()) return found->second;
  if (known.size() >= 8192) known.clear();
  return known[key] = plan_uncached(rows, p.e.N, p.K, limit);
}

}  // namespace

// Microseconds, roughly: a launch, bringing sums together, and the stream (a block's k-blocks one after the other, or what all of them take out of
// L2 at 10 to 8 TB/s and out of memory at 6.5); fitted to 17 to 512 tokens of ten matrices. kNever where
// chains would be too long.
float stream_time(const Product& p) {
  const StreamPlan plan = plan_stream(p);
  if (!plan.cut) return kNever;
  const int k_blocks = (p.K + kBlockK - 1) / kBlockK, sms = b200_sm_count_host();
  const int columns = plan.blocks * plan.tiles;
  const int turns = (columns * plan.members + sms - 1) / sms;
  const float one = static_cast<float>((k_blocks + plan.members - 1) / plan.members) * turns * (0.1f + 0.001f * plan.tile);
  const float all = static_cast<float>(columns) * k_blocks * (kRowsW + plan.tile) * kBlockK / (10.5e6f - 2e4f * plan.tile);
  const float memory = static_cast<float>(p.e.N) * p.K / 6.5e6f;
  return max((plan.members > 1 ? 4.5f + 0.028f * plan.tile : 3.6f) + max(one, all), 2.5f + memory);
}

int launch_stream(const Product& product, cudaStream_t stream) {
  const Epilogue& e = product.e;
  const bool f32 = product.out_f32 != 0;
  const StreamPlan plan = plan_stream(product);
  B200_REQUIRE(plan.smem <= kMaxDynamicSmem, "float8 product: the plan wants %zu bytes of shared memory", plan.smem);
  StreamParams p;
  p.e = e;
  p.err = product.err;
  p.K = product.K;
  p.stages = plan.stages;
  p.tile = plan.tile;
  p.chain_blocks = plan.chain_blocks;
  p.tmem_cols = plan.tmem_cols;
  p.w_constant = product.w_constant;
  p.inbox_at = plan.inbox_at;
  CUtensorMap w_map, x_map;
  if (make_map(&w_map, product.w, e.N, product.K, product.w_stride, kRowsW) != 0) return -1;
  if (make_map(&x_map, product.x, e.M, product.K, product.x_stride, plan.tile) != 0) return -1;
  const StreamKernel kernel = pick_kernel(product.kind, f32, plan.members > 1);
  if (!prepare_kernel(kernel)) return b200_fail("float8 product: the kernel's attributes could not be set");
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(plan.blocks, plan.members, plan.tiles);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = plan.smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  int count = 0;
  if (plan.members > 1) {
    attributes[count].id = cudaLaunchAttributeClusterDimension;
    attributes[count].val.clusterDim.x = 1;
    attributes[count].val.clusterDim.y = plan.members;
    attributes[count].val.clusterDim.z = 1;
    ++count;
  }
  if (b200_overlap_enabled()) {
    attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[count].val.programmaticStreamSerializationAllowed = 1;
    ++count;
  }
  config.attrs = attributes;
  config.numAttrs = count;
  const cudaError_t status = cudaLaunchKernelEx(&config, kernel, w_map, x_map, p);
  if (status != cudaSuccess) {
    cudaGetLastError();
    return b200_fail("float8 product: %s", cudaGetErrorString(status));
  }
  return 0;
}

}  // namespace float8
