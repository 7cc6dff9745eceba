// The product of 8-bit rows (float8.cuh): the call's checks, its tensor maps, and which kernel takes it.
#include "float8.cuh"

namespace float8 {

int g_tile = 0;
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

}  // namespace float8

// y = epilogue(x w^T): x [M, K] and w [N, K] in e4m3 (strides in bytes, multiples of 16), scales a row each. kind: 0 plain, 1 activated, 2 gated
// (W's rows in pairs; out has N / 2 columns, no residual). out and residual strides in elements.
B200_API int b200_float8_linear(const void* x, int64_t x_stride, const float* x_scale, const void* w, int64_t w_stride, const float* w_scale, int w_constant,
                                void* out, int out_dtype, int64_t out_stride, const float* bias, const float* residual, int64_t residual_stride, int M, int N,
                                int K, int kind, int activation, int* err, cudaStream_t stream) {
  using namespace float8;
  if (M == 0 || N == 0) return 0;
  B200_REQUIRE(M > 0 && N > 0 && K > 0, "float8 product: bad sizes %d x %d x %d", M, N, K);
  B200_REQUIRE(kind >= PLAIN && kind <= GATED, "float8 product: unknown kind %d", kind);
  B200_REQUIRE(activation >= ACT_NONE && activation <= ACT_SQUARED_RELU && (kind == PLAIN) == (activation == ACT_NONE), "float8 product: unknown activation %d",
               activation);
  B200_REQUIRE(kind != GATED || (N % 2 == 0 && activation != ACT_SQUARED_RELU && residual == nullptr), "float8 product: the gated form takes pairs of rows, silu or gelu, no residual");
  B200_REQUIRE(out_dtype == DTYPE_F32 || out_dtype == DTYPE_BF16, "float8 product: unknown dtype %d", out_dtype);
  B200_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 && x_stride % 16 == 0 && w_stride % 16 == 0 && x_stride >= K &&
                   w_stride >= K,
               "float8 product: operands' rows start on 16-byte boundaries");
  Product p;
  p.x = x, p.w = w, p.x_stride = x_stride, p.w_stride = w_stride, p.K = K, p.kind = kind, p.out_f32 = out_dtype == DTYPE_F32, p.w_constant = w_constant, p.err = err;
  p.e.out = out, p.e.x_scale = x_scale, p.e.w_scale = w_scale, p.e.bias = bias, p.e.residual = residual;
  p.e.out_stride = out_stride, p.e.residual_stride = residual_stride, p.e.M = M, p.e.N = N, p.e.activation = activation;
  const int size = out_dtype == DTYPE_F32 ? 4 : 2, at_once = kind == GATED ? 2 : 4;  // outputs from four rows of W
  p.e.vector = out_stride % at_once == 0 && reinterpret_cast<uintptr_t>(out) % (at_once * size) == 0 &&
               (residual == nullptr || (residual_stride % 4 == 0 && reinterpret_cast<uintptr_t>(residual) % 16 == 0));
  if (float8::g_tile > 0) return launch_tiles(p, float8::g_tile, stream);
  return launch_stream(p, stream);
}
B200_API void b200_float8_tile_override(int tile) { float8::g_tile = tile; }
