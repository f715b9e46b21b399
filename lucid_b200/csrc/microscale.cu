// MXFP4 streams: encode, decode, and the fake quantization of quantization-aware training.
//
// All of them are bound by HBM: encode reads 2 or 4 bytes and writes 17/32 of a byte per value, decode the
// reverse, the fake quantization reads and writes a value and keeps one bit.  A warp takes 512 consecutive
// values of a row, sixteen per lane (32 bytes of bf16 in one load): two lanes hold a block, one shuffle
// gives its largest magnitude, and the warp's sixteen scale bytes are one row of two scale tiles.  Eight values
// per lane spent twice the instructions on bookkeeping and were bound by issue in bf16: 50 us against 27 for
// an encode of 8192 x 8192.
#include "microscale.cuh"

namespace lq {
namespace {

using mx::Chunk;

constexpr int kThreads = 256;

constexpr int kSpan = 512;  // columns of a warp

// Rows of a unit: a warp takes the same columns of two (float32) or four (bf16) consecutive rows, all loads
// first, 128 bytes a lane in flight.
template <typename T>
constexpr int kUnitRows = 8 / (int)sizeof(T);

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_quantize_kernel(const T* __restrict__ x, size_t rows, size_t K, size_t ldx, uint32_t spans, uint32_t units, int wide,
                   uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int kRows = kUnitRows<T>;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t unit = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int lane = threadIdx.x & 31;
  const uint32_t group = unit / spans, span = unit - group * spans;
  const size_t row0 = (size_t)group * kRows, k0 = (size_t)span * kSpan + lane * 16;
  const bool in_k = k0 < K;
  Chunk<T> c[kRows];
  const T* src = x + row0 * ldx + k0;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (in_k && row0 + r < rows) c[r].load(src + r * ldx, wide);
    else c[r].clear();
  }
  // lane l holds half of block l / 2; lanes 0, 8, 16, 24 write the words of four blocks: their tile (two to a
  // span; the second may lie past the last), half tile and row
  const uint32_t col_tiles = (uint32_t)((K + mx::kTileCols - 1) / mx::kTileCols), ct = span * 2 + (lane >> 4);
  const bool writer = (lane & 7) == 0 && ct < col_tiles;
  const uint32_t in_tile = (uint32_t)row0 % mx::kTileRows;
  uint8_t* word_at = scales + (row0 / mx::kTileRows * col_tiles + ct) * mx::kTileBytes + mx::tile_offset((int)in_tile, 0) + ((lane >> 3) & 1) * 512;
  uint8_t* code_at = codes + row0 * (K / 2) + k0 / 2;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const uint32_t byte = mx::block_byte<T>(c[r]);
    const uint2 q = mx::encode16<T>(c[r], byte);
    if (in_k && row0 + r < rows) *reinterpret_cast<uint2*>(code_at + r * (K / 2)) = q;
    // lanes past K and rows past the end hold zeros and so byte 0
    uint32_t word = byte << (8 * ((lane >> 1) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    if (writer) *reinterpret_cast<uint32_t*>(word_at + 16 * r) = word;  // the rows of a unit share a row group
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, size_t rows, size_t K,
                     uint32_t spans, uint32_t units, int wide, T* __restrict__ out) {
  constexpr int kRows = 4;
  const uint32_t unit = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int lane = threadIdx.x & 31;
  const uint32_t group = unit / spans, span = unit - group * spans;
  const size_t row0 = (size_t)group * kRows, k0 = (size_t)span * kSpan + lane * 16;
  if (k0 >= K) return;
  const uint32_t col_tiles = (uint32_t)((K + mx::kTileCols - 1) / mx::kTileCols), ct = span * 2 + (lane >> 4);
  const uint8_t* byte_at = scales + (row0 / mx::kTileRows * col_tiles + ct) * mx::kTileBytes +
                           mx::tile_offset((int)((uint32_t)row0 % mx::kTileRows), (lane >> 1) & 7);
  const uint8_t* code_at = codes + row0 * (K / 2) + k0 / 2;
  uint2 code[kRows];
  uint32_t byte[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (row0 + r < rows) code[r] = __ldg(reinterpret_cast<const uint2*>(code_at + r * (K / 2))), byte[r] = __ldg(byte_at + 16 * r);
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (row0 + r < rows) {
      float lo[8], hi[8];
      mx::decode8(code[r].x, lo);
      mx::decode8(code[r].y, hi);
      const float s = mx::scale_value(byte[r]);
#pragma unroll
      for (int i = 0; i < 8; ++i) lo[i] = __fmul_rn(lo[i], s), hi[i] = __fmul_rn(hi[i], s);
      mx::store16(out + (row0 + r) * K + k0, lo, hi, wide);
    }
}

// y = decode(encode(x)); bit i of mask byte j says that value 8j + i passes its gradient: it was rounded
// inside the grid, i.e. |x| / scale < 7 (7 is the midpoint of 6 and the 8 that the clamp removes).  The test is
// a saturating multiply-add, exact because neighbours of 7 lie 2^-21 apart, and a sum of powers of two: the
// comparison unit is the busiest one here.  `zero` is 0: a value the compiler does not know between encode8
// and decode8, which come out as zeros when it can join them.
template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_fake_quantize_kernel(const T* __restrict__ x, size_t n, int wide, uint32_t zero, T* __restrict__ out, uint8_t* __restrict__ mask) {
  const size_t i0 = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 16;
  const bool valid = i0 < n;
  Chunk<T> c;
  if (valid) c.load(x + i0, wide);
  else c.clear();
  const uint32_t byte = mx::block_byte<T>(c);
  if (!valid) return;
  const float inv = mx::inverse_scale(byte), s = mx::scale_value(byte);
  float y[2][8];
  uint32_t bits = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[8], sum = 0.0f;
    c.values(h, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = __fmul_rn(v[i], inv);
      sum = __fmaf_rn(__saturatef(__fmaf_rn(-2097152.0f, fabsf(v[i]), 14680064.0f)), (float)(1 << i), sum);
    }
    bits |= (uint32_t)sum << (8 * h);
    mx::decode8(mx::encode8(v) + zero, y[h]);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[h][i] = __fmul_rn(y[h][i], s);
  }
  if (mask) *reinterpret_cast<uint16_t*>(mask + i0 / 8) = byte == 255u ? 0 : (uint16_t)bits;
  mx::store16(out + i0, y[0], y[1], wide);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
mx_fake_quantize_grad_kernel(const T* __restrict__ grad, const uint8_t* __restrict__ mask, size_t n, int wide, T* __restrict__ out) {
  const size_t i0 = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 16;
  if (i0 >= n) return;
  Chunk<T> c;
  c.load(grad + i0, wide);
  const uint32_t bits = __ldg(reinterpret_cast<const uint16_t*>(mask + i0 / 8));
  float v[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    c.values(h, v[h]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[h][i] = (bits >> (8 * h + i)) & 1u ? v[h][i] : 0.0f;
  }
  mx::store16(out + i0, v[0], v[1], wide);
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
size_t col_tiles_of(size_t K) { return (K + mx::kTileCols - 1) / mx::kTileCols; }
uint32_t spans_of(size_t K) { return (uint32_t)((K + kSpan - 1) / kSpan); }

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
  const uint32_t spans = spans_of(K);
  const int unit_rows = in_dtype == LQ_F32 ? kUnitRows<float> : kUnitRows<bf16>;
  const size_t units = (rows + mx::kTileRows - 1) / mx::kTileRows * (mx::kTileRows / unit_rows) * spans;
  const size_t grid = (units * 32 + kThreads - 1) / kThreads;
  const int wide = reinterpret_cast<uintptr_t>(x) % 32 == 0 && (ldx * esz) % 32 == 0;
  if (int rc = check_grid("lq_mx_quantize", units / 2)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (in_dtype == LQ_F32) return check_cuda(launch_pdl(mx_quantize_kernel<float>, dim3((unsigned)grid), dim3(kThreads), 0, st, (const float*)x, rows, K, ldx, spans, (uint32_t)units, wide, codes, scales), "lq_mx_quantize launch");
  return check_cuda(launch_pdl(mx_quantize_kernel<bf16>, dim3((unsigned)grid), dim3(kThreads), 0, st, (const bf16*)x, rows, K, ldx, spans, (uint32_t)units, wide, codes, scales), "lq_mx_quantize launch");
}

extern "C" int lq_mx_dequantize(const uint8_t* codes, const uint8_t* scales, size_t rows, size_t K, void* out,
                                int out_dtype, void* stream) {
  if (rows == 0) return LQ_OK;
  if (!out || !codes || !scales) return fail(LQ_ERR_DEVICE, "lq_mx_dequantize: null pointer");
  if (out_dtype != LQ_F32 && out_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_dequantize: out must be f32|bf16");
  if (int rc = check_matrix("lq_mx_dequantize", rows, K)) return rc;
  if (!aligned16(out) || !aligned16(codes) || !aligned16(scales))
    return fail(LQ_ERR_ALIGNMENT, "lq_mx_dequantize: out, codes and scales must be 16-byte aligned");
  const uint32_t spans = spans_of(K);
  const size_t units = (rows + 3) / 4 * spans;
  const size_t grid = (units * 32 + kThreads - 1) / kThreads;
  const int wide = reinterpret_cast<uintptr_t>(out) % 32 == 0;
  if (int rc = check_grid("lq_mx_dequantize", units / 2)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (out_dtype == LQ_F32) mx_dequantize_kernel<float><<<(unsigned)grid, kThreads, 0, st>>>(codes, scales, rows, K, spans, (uint32_t)units, wide, (float*)out);
  else mx_dequantize_kernel<bf16><<<(unsigned)grid, kThreads, 0, st>>>(codes, scales, rows, K, spans, (uint32_t)units, wide, (bf16*)out);
  return check_cuda(cudaGetLastError(), "lq_mx_dequantize launch");
}

extern "C" int lq_mx_fake_quantize(const void* x, int dtype, size_t n, void* out, uint8_t* mask, void* stream) {
  if (n == 0) return LQ_OK;
  if (!x || !out) return fail(LQ_ERR_DEVICE, "lq_mx_fake_quantize: null pointer");
  if (dtype != LQ_F32 && dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_fake_quantize: x must be f32|bf16");
  if (n % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, "lq_mx_fake_quantize: the count must be a multiple of 32");
  if (!aligned16(x) || !aligned16(out) || reinterpret_cast<uintptr_t>(mask) % 2) return fail(LQ_ERR_ALIGNMENT, "lq_mx_fake_quantize: x and out must be 16-byte, the mask 2-byte aligned");
  const size_t grid = (n / 16 + kThreads - 1) / kThreads;
  if (int rc = check_grid("lq_mx_fake_quantize", grid)) return rc;
  const int wide = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % 32 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == LQ_F32) mx_fake_quantize_kernel<float><<<(unsigned)grid, kThreads, 0, st>>>((const float*)x, n, wide, 0u, (float*)out, mask);
  else mx_fake_quantize_kernel<bf16><<<(unsigned)grid, kThreads, 0, st>>>((const bf16*)x, n, wide, 0u, (bf16*)out, mask);
  return check_cuda(cudaGetLastError(), "lq_mx_fake_quantize launch");
}

extern "C" int lq_mx_fake_quantize_grad(const void* grad, int dtype, const uint8_t* mask, size_t n, void* out, void* stream) {
  if (n == 0) return LQ_OK;
  if (!grad || !mask || !out) return fail(LQ_ERR_DEVICE, "lq_mx_fake_quantize_grad: null pointer");
  if (dtype != LQ_F32 && dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_fake_quantize_grad: the gradient must be f32|bf16");
  if (n % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, "lq_mx_fake_quantize_grad: the count must be a multiple of 32");
  if (!aligned16(grad) || !aligned16(out) || reinterpret_cast<uintptr_t>(mask) % 2) return fail(LQ_ERR_ALIGNMENT, "lq_mx_fake_quantize_grad: the gradients must be 16-byte, the mask 2-byte aligned");
  const size_t grid = (n / 16 + kThreads - 1) / kThreads;
  if (int rc = check_grid("lq_mx_fake_quantize_grad", grid)) return rc;
  const int wide = (reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(out)) % 32 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == LQ_F32) mx_fake_quantize_grad_kernel<float><<<(unsigned)grid, kThreads, 0, st>>>((const float*)grad, mask, n, wide, (float*)out);
  else mx_fake_quantize_grad_kernel<bf16><<<(unsigned)grid, kThreads, 0, st>>>((const bf16*)grad, mask, n, wide, (bf16*)out);
  return check_cuda(cudaGetLastError(), "lq_mx_fake_quantize_grad launch");
}
