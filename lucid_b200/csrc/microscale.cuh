// MXFP4 element and scale conversions shared by the microscaled kernels.
//
// A block of 32 values holds 4-bit floats (E2M1: 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one
// power-of-two scale, kept as its biased exponent (E8M0, 255 = NaN).  The scale of a block is
// 2^(floor(log2 amax) - 2), so the largest magnitude lands in [4, 8) of the element grid: 2 is the
// exponent of the grid's largest value.  Scaling by a power of two is exact, so an element is rounded
// once (ties to the even mantissa, clamped at 6).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace lq {
namespace mx {

constexpr int kBlock = 32;        // values per scale
constexpr int kTileRows = 128;    // a scale tile: 128 rows x 8 blocks, 1024 bytes
constexpr int kTileCols = 256;    // ... which cover 256 values of K
constexpr int kTileBytes = 1024;

// Byte of (row, block) inside its tile: two halves of four blocks, each 32 rows x 4 row groups x 4 blocks
// (the order in which the tensor core's scale operand wants its lanes).
__host__ __device__ __forceinline__ int tile_offset(int row, int block) {
  return (block >> 2) * 512 + (row & 31) * 16 + (row >> 5) * 4 + (block & 3);
}

// Scale byte of a block from the float32 bit pattern of its largest magnitude.  The exponent field is
// floor(log2) + 127 for normal values; zero and subnormal blocks, and exponents below the format's
// range, take byte 0 (2^-127); an infinity or NaN anywhere in the block takes byte 255.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : (e < 2u ? 0u : e - 2u);
}
// 1 / scale, exact (byte <= 252 whenever it came from finite float32 values)
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// The scale itself: byte 0 is the subnormal 2^-127, byte 255 NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 0x7fffffffu : byte << 23));
}

// Eight scaled values -> eight 4-bit codes, value i in bits [4i, 4i + 4).
__device__ __forceinline__ uint32_t encode8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight codes -> their values (exact in float16, and so in float32).
__device__ __forceinline__ void decode8(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}

// Loads of data that a kernel before this one wrote, used once.  Plain loads, not the read-only (.nc) form: under
// programmatic launch this kernel's life overlaps the writer's, and the read-only path promises nothing then.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// Sixteen consecutive values of a thread, kept as they were loaded; two threads hold a block.  `amax` is the
// largest magnitude in a form that `merge` combines and `amax_bits` turns into a float32 bit pattern ordered
// like the magnitudes, a NaN above infinity.
template <typename T>
struct Chunk;
template <>
struct Chunk<float> {
  uint32_t w[16];
  __device__ __forceinline__ void load(const float* p, int wide) {
    if (wide) {  // 32-byte aligned
#pragma unroll
      for (int i = 0; i < 16; i += 8)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                     : "l"(p + i)
                     : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const uint4 v = load_once(p + i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 0;
  }
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = w[0] & 0x7fffffffu;
#pragma unroll
    for (int i = 1; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
  static __device__ __forceinline__ uint32_t merge(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t amax_bits(uint32_t m) { return m; }
  __device__ __forceinline__ void values(int half, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[8 * half + i]);
  }
};
template <>
struct Chunk<__nv_bfloat16> {
  uint32_t w[8];
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int wide) {
    if (wide) {
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p)
                   : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const uint4 v = load_once(p + 2 * i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
  }
  // pairwise: two halves a word until the very end
  static __device__ __forceinline__ uint32_t merge(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = merge(m, w[i] & 0x7fff7fffu);
    return m;
  }
  static __device__ __forceinline__ uint32_t amax_bits(uint32_t m) { return max(m << 16, m & 0xffff0000u); }
  __device__ __forceinline__ void values(int half, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[2 * i] = __uint_as_float(w[4 * half + i] << 16), v[2 * i + 1] = __uint_as_float(w[4 * half + i] & 0xffff0000u);
  }
};
// The block's scale byte, known to both threads that hold it.  The whole warp calls this.
template <typename T>
__device__ __forceinline__ uint32_t block_byte(const Chunk<T>& c) {
  const uint32_t m = c.amax();
  return scale_byte(Chunk<T>::amax_bits(Chunk<T>::merge(m, __shfl_xor_sync(0xffffffffu, m, 1))));
}
// Codes of the sixteen values, value i in bits [4i, 4i + 4); zero for a block without a scale.
template <typename T>
__device__ __forceinline__ uint2 encode16(const Chunk<T>& c, uint32_t byte) {
  const float inv = inverse_scale(byte);
  uint32_t q[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[8];
    c.values(h, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], inv);
    q[h] = encode8(v);
  }
  return byte == 255u ? make_uint2(0, 0) : make_uint2(q[0], q[1]);
}

// Eight values -> memory (16-byte aligned), rounded once when T is narrower.
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ uint32_t bf16x2_bits(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]), bf16x2_bits(v[4], v[5]), bf16x2_bits(v[6], v[7]));
}

// ... in one store per 32 bytes where the address allows it (`wide`)
__device__ __forceinline__ void store8(float* p, const float (&v)[8], int wide) {
  if (wide) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
    store_32(p, w);
  } else {
    store8(p, v);
  }
}
// Sixteen values.
__device__ __forceinline__ void store16(float* p, const float (&lo)[8], const float (&hi)[8], int wide) {
  store8(p, lo, wide);
  store8(p + 8, hi, wide);
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, const float (&lo)[8], const float (&hi)[8], int wide) {
  if (wide) {
    const uint32_t w[8] = {bf16x2_bits(lo[0], lo[1]), bf16x2_bits(lo[2], lo[3]), bf16x2_bits(lo[4], lo[5]), bf16x2_bits(lo[6], lo[7]),
                           bf16x2_bits(hi[0], hi[1]), bf16x2_bits(hi[2], hi[3]), bf16x2_bits(hi[4], hi[5]), bf16x2_bits(hi[6], hi[7])};
    store_32(p, w);
  } else {
    store8(p, lo);
    store8(p + 8, hi);
  }
}

}  // namespace mx
}  // namespace lq
