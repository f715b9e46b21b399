// MXFP4 streams: encode, decode, and the fake quantization of quantization-aware training.
//
// All of them are bound by HBM: encode reads 2 or 4 bytes and writes 17/32 of a byte per value, decode the
// reverse, the fake quantization reads and writes a value and keeps one bit.  A warp takes 256
// consecutive values of a row (eight per lane, one 16-byte load for bf16): four lanes hold a block, so
// its largest magnitude is two shuffles away, and the warp's eight scale bytes are one column of a scale
// tile.
#include <cuda_fp16.h>

#include "microscale.cuh"

namespace lq {
namespace {

using mx::Chunk;

constexpr int kThreads = 256;

// Rows of a unit: a warp takes the same 256 columns of four consecutive rows, all loads first (one row at a
// time left the loads too far apart to fill HBM: 119 us against 1NEW us for an 8192 x 8192 float32 round trip).
constexpr int kUnitRows = 4;

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_quantize_kernel(const T* __restrict__ x, size_t rows, size_t K, size_t ldx, uint32_t col_tiles, size_t units, int wide,
                   uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  pdl_wait();
  pdl_launch_dependents();
  const size_t unit = ((size_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  if (unit >= units) return;
  const int lane = threadIdx.x & 31;
  const size_t group = unit / col_tiles;
  const size_t ct = unit - group * col_tiles;
  const size_t row0 = group * kUnitRows, k0 = ct * mx::kTileCols + lane * 8;
  const bool in_k = k0 < K;
  Chunk<T> c[kUnitRows];
#pragma unroll
  for (int r = 0; r < kUnitRows; ++r) {
    if (!(in_k && row0 + r < rows)) c[r].clear();
    else if (wide) c[r].load_wide(x + (row0 + r) * ldx + k0);
    else c[r].load(x + (row0 + r) * ldx + k0);
  }
  uint8_t* tile = scales + ((row0 / mx::kTileRows) * col_tiles + ct) * mx::kTileBytes;
#pragma unroll
  for (int r = 0; r < kUnitRows; ++r) {
    uint32_t amax = c[r].amax_bits();
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t byte = mx::scale_byte(amax);
    if (in_k && row0 + r < rows) {
      float v[8];
      c[r].values(v);
      const float inv = mx::inverse_scale(byte);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], inv);
      *reinterpret_cast<uint32_t*>(codes + (row0 + r) * (K / 2) + k0 / 2) = byte == 255u ? 0u : mx::encode8(v);
    }
    // four blocks (16 lanes) share a scale word; lanes past K and rows past the end hold zeros and so byte 0
    uint32_t word = byte << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if ((lane & 15) == 0)
      *reinterpret_cast<uint32_t*>(tile + mx::tile_offset((int)((row0 + r) % mx::kTileRows), 0) + (lane >> 4) * 512) = word;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, size_t rows, size_t K,
                     uint32_t col_tiles, size_t units, int wide, T* __restrict__ out) {
  const size_t unit = ((size_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  if (unit >= units) return;
  const int lane = threadIdx.x & 31;
  const size_t group = unit / col_tiles;
  const size_t ct = unit - group * col_tiles;
  const size_t row0 = group * kUnitRows, k0 = ct * mx::kTileCols + lane * 8;
  if (k0 >= K) return;
  const uint8_t* tile = scales + ((row0 / mx::kTileRows) * col_tiles + ct) * mx::kTileBytes;
  uint32_t code[kUnitRows], byte[kUnitRows];
#pragma unroll
  for (int r = 0; r < kUnitRows; ++r)
    if (row0 + r < rows) {
      code[r] = __ldg(reinterpret_cast<const uint32_t*>(codes + (row0 + r) * (K / 2) + k0 / 2));
      byte[r] = __ldg(tile + mx::tile_offset((int)((row0 + r) % mx::kTileRows), lane >> 2));
    }
#pragma unroll
  for (int r = 0; r < kUnitRows; ++r)
    if (row0 + r < rows) {
      float v[8];
      mx::decode8(code[r], v);
      const float s = mx::scale_value(byte[r]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], s);
      mx::store8(out + (row0 + r) * K + k0, v, wide);
    }
}

// y = decode(encode(x)); bit i of mask byte j says that value 8j + i passes its gradient: it was rounded
// inside the grid, i.e. |x| / scale < 7 (7 is the midpoint of 6 and the 8 that the clamp removes).
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_fake_quantize_kernel(const T* __restrict__ x, size_t n, int wide, T* __restrict__ out, uint8_t* __restrict__ mask) {
  const size_t i0 = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  const bool valid = i0 < n;
  Chunk<T> c;
  if (!valid) c.clear();
  else if (wide) c.load_wide(x + i0);
  else c.load(x + i0);
  uint32_t amax = c.amax_bits();
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  if (!valid) return;
  const uint32_t byte = mx::scale_byte(amax);
  const float inv = mx::inverse_scale(byte), s = mx::scale_value(byte);
  float v[8];
  c.values(v);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = __fmul_rn(v[i], inv);
    if (fabsf(t) < 7.0f) bits |= 1u << i;
    v[i] = __fmul_rn(mx::round_element(t), s);
  }
  if (mask) mask[i0 / 8] = byte == 255u ? 0 : (uint8_t)bits;
  mx::store8(out + i0, v, wide);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_fake_quantize_grad_kernel(const T* __restrict__ grad, const uint8_t* __restrict__ mask, size_t n, int wide, T* __restrict__ out) {
  const size_t i0 = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  if (i0 >= n) return;
  Chunk<T> c;
  if (wide) c.load_wide(grad + i0);
  else c.load(grad + i0);
  const uint32_t bits = __ldg(mask + i0 / 8);
  float v[8];
  c.values(v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (bits >> i) & 1u ? v[i] : 0.0f;
  mx::store8(out + i0, v, wide);
}

int check_matrix(const char* who, size_t rows, size_t K) {
  if (K == 0 || K % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, std::string(who) + ": the last axis must be a multiple of 32");
  if (rows >= ((size_t)1 << 40) || K >= ((size_t)1 << 31)) return fail(LQ_ERR_SHAPE, std::string(who) + ": matrix too large");
  return LQ_OK;
}
int check_grid(const char* who, size_t blocks) {
  if (blocks > 0x7fffffffu) return fail(LQ_ERR_SHAPE, std::string(who) + ": too many values for one launch");
  return LQ_OK;
}
uint32_t col_tiles_of(size_t K) { return (uint32_t)((K + mx::kTileCols - 1) / mx::kTileCols); }

}  // namespace
}  // namespace lq

using namespace lq;
using bf16 = __nv_bfloat16;

extern "C" size_t lq_mx_scale_bytes(size_t rows, size_t K) {
  return (rows + mx::kTileRows - 1) / mx::kTileRows * col_tiles_of(K) * mx::kTileBytes;
}

extern "C" int lq_mx_quantize(const void* x, int in_dtype, size_t rows, size_t K, size_t ldx, uint8_t* codes,
                              uint8_t* scales, void* stream) {
  if (rows == 0) return LQ_OK;
  if (!x || !codes || !scales) return fail(LQ_ERR_DEVICE, "lq_mx_quantize: null pointer");
  if (in_dtype != LQ_F32 && in_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_quantize: x must be f32|bf16");
  if (int rc = check_matrix("lq_mx_quantize", rows, K)) return rc;
  const size_t esz = in_dtype == LQ_F32 ? 4 : 2;
  if (ldx < K) return fail(LQ_ERR_SHAPE, "lq_mx_quantize: row stride shorter than a row");
  if (!aligned16(x) || !aligned16(codes) || !aligned16(scales) || (ldx * esz) % 16 != 0)
    return fail(LQ_ERR_ALIGNMENT, "lq_mx_quantize: rows, codes and scales must be 16-byte aligned");
  const uint32_t ct = col_tiles_of(K);
  const size_t units = (rows + mx::kTileRows - 1) / mx::kTileRows * (mx::kTileRows / kUnitRows) * ct;
  const size_t grid = (units * 32 + kThreads - 1) / kThreads;
  const int wide = reinterpret_cast<uintptr_t>(x) % 32 == 0 && (ldx * esz) % 32 == 0;
  if (int rc = check_grid("lq_mx_quantize", grid)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (in_dtype == LQ_F32) return check_cuda(launch_pdl(mx_quantize_kernel<float>, dim3((unsigned)grid), dim3(kThreads), 0, st, (const float*)x, rows, K, ldx, ct, units, wide, codes, scales), "lq_mx_quantize launch");
  return check_cuda(launch_pdl(mx_quantize_kernel<bf16>, dim3((unsigned)grid), dim3(kThreads), 0, st, (const bf16*)x, rows, K, ldx, ct, units, wide, codes, scales), "lq_mx_quantize launch");
}

extern "C" int lq_mx_dequantize(const uint8_t* codes, const uint8_t* scales, size_t rows, size_t K, void* out,
                                int out_dtype, void* stream) {
  if (rows == 0) return LQ_OK;
  if (!out || !codes || !scales) return fail(LQ_ERR_DEVICE, "lq_mx_dequantize: null pointer");
  if (out_dtype != LQ_F32 && out_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_dequantize: out must be f32|bf16");
  if (int rc = check_matrix("lq_mx_dequantize", rows, K)) return rc;
  if (!aligned16(out) || !aligned16(codes) || !aligned16(scales))
    return fail(LQ_ERR_ALIGNMENT, "lq_mx_dequantize: out, codes and scales must be 16-byte aligned");
  const uint32_t ct = col_tiles_of(K);
  const size_t units = (rows + kUnitRows - 1) / kUnitRows * ct;
  const size_t grid = (units * 32 + kThreads - 1) / kThreads;
  const int wide = reinterpret_cast<uintptr_t>(out) % 32 == 0;
  if (int rc = check_grid("lq_mx_dequantize", grid)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (out_dtype == LQ_F32) mx_dequantize_kernel<float><<<(unsigned)grid, kThreads, 0, st>>>(codes, scales, rows, K, ct, units, wide, (float*)out);
  else mx_dequantize_kernel<bf16><<<(unsigned)grid, kThreads, 0, st>>>(codes, scales, rows, K, ct, units, wide, (bf16*)out);
  return check_cuda(cudaGetLastError(), "lq_mx_dequantize launch");
}

extern "C" int lq_mx_fake_quantize(const void* x, int dtype, size_t n, void* out, uint8_t* mask, void* stream) {
  if (n == 0) return LQ_OK;
  if (!x || !out) return fail(LQ_ERR_DEVICE, "lq_mx_fake_quantize: null pointer");
  if (dtype != LQ_F32 && dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_fake_quantize: x must be f32|bf16");
  if (n % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, "lq_mx_fake_quantize: the count must be a multiple of 32");
  if (!aligned16(x) || !aligned16(out)) return fail(LQ_ERR_ALIGNMENT, "lq_mx_fake_quantize: x and out must be 16-byte aligned");
  const size_t grid = (n / 8 + kThreads - 1) / kThreads;
  if (int rc = check_grid("lq_mx_fake_quantize", grid)) return rc;
  const int wide = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % 32 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == LQ_F32) mx_fake_quantize_kernel<float><<<(unsigned)grid, kThreads, 0, st>>>((const float*)x, n, wide, (float*)out, mask);
  else mx_fake_quantize_kernel<bf16><<<(unsigned)grid, kThreads, 0, st>>>((const bf16*)x, n, wide, (bf16*)out, mask);
  return check_cuda(cudaGetLastError(), "lq_mx_fake_quantize launch");
}

extern "C" int lq_mx_fake_quantize_grad(const void* grad, int dtype, const uint8_t* mask, size_t n, void* out, void* stream) {
  if (n == 0) return LQ_OK;
  if (!grad || !mask || !out) return fail(LQ_ERR_DEVICE, "lq_mx_fake_quantize_grad: null pointer");
  if (dtype != LQ_F32 && dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_fake_quantize_grad: the gradient must be f32|bf16");
  if (n % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, "lq_mx_fake_quantize_grad: the count must be a multiple of 32");
  if (!aligned16(grad) || !aligned16(out)) return fail(LQ_ERR_ALIGNMENT, "lq_mx_fake_quantize_grad: the gradients must be 16-byte aligned");
  const size_t grid = (n / 8 + kThreads - 1) / kThreads;
  if (int rc = check_grid("lq_mx_fake_quantize_grad", grid)) return rc;
  const int wide = (reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(out)) % 32 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == LQ_F32) mx_fake_quantize_grad_kernel<float><<<(unsigned)grid, kThreads, 0, st>>>((const float*)grad, mask, n, wide, (float*)out);
  else mx_fake_quantize_grad_kernel<bf16><<<(unsigned)grid, kThreads, 0, st>>>((const bf16*)grad, mask, n, wide, (bf16*)out);
  return check_cuda(cudaGetLastError(), "lq_mx_fake_quantize_grad launch");
}
