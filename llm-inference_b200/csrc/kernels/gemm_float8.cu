// The product of 8-bit rows (float8.cuh): the call's checks, its tensor maps, and which kernel takes it.
#include "float8.cuh"

namespace float8 {

namespace {
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult status;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &status) != cudaSuccess || status != cudaDriverEntryPointSuccess)
      return EncodeTiled(nullptr);
    return reinterpret_cast<EncodeTiled>(ptr);
  }();
  return fn;
}
}  // namespace

int make_map(CUtensorMap* map, const void* base, int rows, int K, int64_t stride, int box_rows) {
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return b200_fail("float8 product: the driver does not provide cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {kBlockK, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult status = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (status != CUDA_SUCCESS) return b200_fail("float8 product: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(status));
  return 0;
}

// Which kernel. Up to 16 tokens weights are all there is to read: the form for short streams, else the streaming one. With more the faster one by the
// kernels' own estimates of their time, and the tile form's width with it: tiles fill whole turns of all clusters at different widths (777 tokens
// of 8,192 x 2,048: 224 tokens 19.9 us, 256 21.3, 160 22.6; 2,048 of 4,608 x 3,584: 256 27.6, 224 33.7).
static int launch_chosen(const Product& p, cudaStream_t stream) {
  if (skinny_takes(p.e.M, p.e.N, p.K)) return launch_skinny(p, stream);
  int best = 0;
  float least = p.e.M <= 512 ? stream_time(p) : kNever;
  if (p.e.M <= 16 && least < kNever) return launch_stream(p, stream);
  for (int tile = 64; tile <= 256 && (tile == 64 || tile < p.e.M + 32); tile += 32) {
    const float time = tiles_time(p, tile);
    if (time < least) least = time, best = tile;
  }
  return best == 0 ? launch_stream(p, stream) : launch_tiles(p, best, stream);
}

}  // namespace float8

// The numbers of a call, in the order in which parts/float8.py packs them: y = epilogue(x w^T), x [M, K] and w [N, K] in e4m3 (pitches in bytes, multiples
// of 16), scales a row each. kind: 0 plain, 1 activated, 2 gated (W's rows in pairs; out has N / 2 columns, no residual). out and residual pitches in elements.
struct Float8Linear {
  const void* x;
  int64_t x_pitch;
  const float* x_scales;
  const void* w;
  int64_t w_pitch;
  const float* w_scales;
  int64_t w_constant;
  void* out;
  int64_t out_dtype, out_pitch;
  const float* bias;
  const float* residual;
  int64_t residual_pitch, M, N, K, kind, activation;
  int* err;
};
static_assert(sizeof(Float8Linear) == 19 * 8, "as packed by the caller");

B200_API int b200_float8_linear(const Float8Linear* c, cudaStream_t stream) {
  using namespace float8;
  if (c->M == 0 || c->N == 0) return 0;
  constexpr int64_t kMost = int64_t(1) << 30;  // counts and coordinates are 32-bit
  constexpr int64_t kMostK = int64_t(1) << 28;  // a tile's products then take half a second: no wait inside a kernel runs out
  B200_REQUIRE(c->M > 0 && c->N > 0 && c->K > 0 && c->M <= kMost && c->N <= kMost && c->K <= kMostK, "float8 product: rows, features and inner size are at most 2^30, 2^30 and 2^28");
  Product p;
  p.x = c->x, p.w = c->w, p.x_stride = c->x_pitch, p.w_stride = c->w_pitch, p.K = static_cast<int>(c->K);
  p.kind = static_cast<int>(c->kind), p.out_f32 = c->out_dtype == DTYPE_F32, p.w_constant = c->w_constant != 0, p.err = c->err;
  Epilogue& e = p.e;
  e.out = c->out, e.x_scale = c->x_scales, e.w_scale = c->w_scales, e.bias = c->bias, e.residual = c->residual;
  e.out_stride = c->out_pitch, e.residual_stride = c->residual_pitch, e.M = static_cast<int>(c->M), e.N = static_cast<int>(c->N);
  e.activation = static_cast<int>(c->activation);
  B200_REQUIRE(p.kind >= PLAIN && p.kind <= GATED, "float8 product: unknown kind %d", p.kind);
  B200_REQUIRE(e.activation >= ACT_NONE && e.activation <= ACT_SQUARED_RELU && (p.kind == PLAIN) == (e.activation == ACT_NONE),
               "float8 product: unknown activation %d", e.activation);
  B200_REQUIRE(p.kind != GATED || (e.N % 2 == 0 && e.activation != ACT_SQUARED_RELU && e.residual == nullptr),
               "float8 product: the gated form takes pairs of rows, silu or gelu, no residual");
  B200_REQUIRE(c->out_dtype == DTYPE_F32 || c->out_dtype == DTYPE_BF16, "float8 product: unknown dtype %d", static_cast<int>(c->out_dtype));
  B200_REQUIRE(reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0 && p.x_stride % 16 == 0 && p.w_stride % 16 == 0 &&
                   p.x_stride >= p.K && p.w_stride >= p.K,
               "float8 product: operands' rows start on 16-byte boundaries");
  const int size = p.out_f32 ? 4 : 2, at_once = p.kind == GATED ? 2 : 4;  // outputs from four rows of W
  e.vector = e.out_stride % at_once == 0 && reinterpret_cast<uintptr_t>(e.out) % (at_once * size) == 0 &&
             (e.residual == nullptr || (e.residual_stride % 4 == 0 && reinterpret_cast<uintptr_t>(e.residual) % 16 == 0));
  try {
    return launch_chosen(p, stream);
  } catch (...) {  // plans are kept in containers
    return b200_fail("float8 product: out of memory on the host");
  }
}
