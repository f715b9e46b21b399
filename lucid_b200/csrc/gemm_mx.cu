// Product of two MXFP4 matrices.
//   out[m, n] = sum_k a[m, k] * w[n, k] (+ bias[n]) (ReLU), float32 accumulation.
#include "microscale.cuh"

namespace lq {
namespace {

__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One output per thread, block by block: sum over a block of the element products (exact: at most
// 32 * 36 in steps of 1/4), times the two scales.
template <typename T>
__global__ void __launch_bounds__(128)
mx_matmul_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ sa, size_t M, const uint8_t* __restrict__ w,
                 const uint8_t* __restrict__ sw, size_t N, size_t K, const float* __restrict__ bias, int relu,
                 T* __restrict__ out, size_t ldo) {
  const size_t n = (size_t)blockIdx.x * 128 + threadIdx.x;
  if (n >= N) return;
  const size_t col_tiles = (K + mx::kTileCols - 1) / mx::kTileCols;
  for (size_t m = blockIdx.y; m < M; m += gridDim.y) {
    float acc = 0.0f;
    for (size_t b = 0; b < K / mx::kBlock; ++b) {
      float dot = 0.0f;
      for (int q = 0; q < 4; ++q) {
        float va[8], vw[8];
        mx::decode8(__ldg(reinterpret_cast<const uint32_t*>(a + m * (K / 2) + b * 16) + q), va);
        mx::decode8(__ldg(reinterpret_cast<const uint32_t*>(w + n * (K / 2) + b * 16) + q), vw);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot = fmaf(va[i], vw[i], dot);
      }
      const float fa = mx::scale_value(sa[(m / 128 * col_tiles + b / 8) * mx::kTileBytes + mx::tile_offset((int)(m % 128), (int)(b % 8))]);
      const float fw = mx::scale_value(sw[(n / 128 * col_tiles + b / 8) * mx::kTileBytes + mx::tile_offset((int)(n % 128), (int)(b % 8))]);
      acc = fmaf(dot * fa, fw, acc);
    }
    if (bias) acc += __ldg(bias + n);
    if (relu) acc = acc < 0.0f ? 0.0f : acc;
    store1(out + m * ldo + n, acc);
  }
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_mx_linear_workspace_bytes(size_t M, size_t K) {
  return (M * (K / 2) + 1023) / 1024 * 1024 + lq_mx_scale_bytes(M, K);
}

extern "C" int lq_mx_matmul(const uint8_t* a_codes, const uint8_t* a_scales, size_t M, const uint8_t* w_codes,
                            const uint8_t* w_scales, size_t N, size_t K, const float* bias, int relu, void* out,
                            int out_dtype, size_t ldo, int32_t* status, void* stream) {
  if (M == 0 || N == 0) return LQ_OK;
  if (!a_codes || !a_scales || !w_codes || !w_scales || !out) return fail(LQ_ERR_DEVICE, "lq_mx_matmul: null pointer");
  if (out_dtype != LQ_F32 && out_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_matmul: out must be f32|bf16");
  if (K == 0 || K % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, "lq_mx_matmul: K must be a multiple of 32");
  if (M >= ((size_t)1 << 30) || N >= ((size_t)1 << 30) || K >= ((size_t)1 << 30)) return fail(LQ_ERR_SHAPE, "lq_mx_matmul: extents must be below 2^30");
  if (ldo < N) return fail(LQ_ERR_SHAPE, "lq_mx_matmul: output row stride shorter than a row");
  if (!aligned16(a_codes) || !aligned16(a_scales) || !aligned16(w_codes) || !aligned16(w_scales))
    return fail(LQ_ERR_ALIGNMENT, "lq_mx_matmul: codes and scales must be 16-byte aligned");
  (void)status;
  const dim3 grid((unsigned)((N + 127) / 128), (unsigned)(M < 4096 ? M : 4096));
  cudaStream_t st = (cudaStream_t)stream;
  if (out_dtype == LQ_F32)
    mx_matmul_kernel<float><<<grid, 128, 0, st>>>(a_codes, a_scales, M, w_codes, w_scales, N, K, bias, relu, (float*)out, ldo);
  else
    mx_matmul_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a_codes, a_scales, M, w_codes, w_scales, N, K, bias, relu, (__nv_bfloat16*)out, ldo);
  return check_cuda(cudaGetLastError(), "lq_mx_matmul launch");
}

extern "C" int lq_mx_linear(const void* x, int in_dtype, size_t M, size_t ldx, const uint8_t* w_codes, const uint8_t* w_scales,
                            size_t N, size_t K, const float* bias, int relu, void* out, int out_dtype, size_t ldo,
                            uint8_t* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  if (M == 0 || N == 0) return LQ_OK;
  if (!workspace) return fail(LQ_ERR_DEVICE, "lq_mx_linear: null workspace");
  if (K % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, "lq_mx_linear: K must be a multiple of 32");
  if (workspace_bytes < lq_mx_linear_workspace_bytes(M, K)) return fail(LQ_ERR_WORKSPACE, "lq_mx_linear: workspace too small");
  uint8_t* a_scales = workspace + (M * (K / 2) + 1023) / 1024 * 1024;
  if (int rc = lq_mx_quantize(x, in_dtype, M, K, ldx, workspace, a_scales, stream)) return rc;
  return lq_mx_matmul(workspace, a_scales, M, w_codes, w_scales, N, K, bias, relu, out, out_dtype, ldo, status, stream);
}
