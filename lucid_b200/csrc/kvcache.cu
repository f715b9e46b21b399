// The quantized key / value cache: rows encoded as they are written, and read back by page table.
//
// A cache row is one token's (heads, dim) values, kept contiguous (page, offset, head, dim), so a write is one
// pass over the new tokens and a read one pass over the tokens asked for; both are bound by HBM.  Two formats:
// int8 codes with one float32 scale per (token, head) -- the arithmetic of the per-token encode -- and
// MXFP4 along the head dimension.
#include <cuda_fp16.h>

#include "microscale.cuh"

namespace lq {
namespace {

using mx::Chunk;
using bf16 = __nv_bfloat16;

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;

struct Side {           // keys or values
  uint8_t* codes;
  uint8_t* scales;      // float32 (int8 format) or scale bytes
  void* rows;           // new rows (write), output rows (read)
  long long token, head;  // their strides
};
__device__ __forceinline__ long long index_at(const void* p, int bits, size_t i) {
  return bits == 64 ? __ldg(reinterpret_cast<const long long*>(p) + i) : (long long)__ldg(reinterpret_cast<const int*>(p) + i);
}

// n / d for n * d < 2^40, by a multiplication
struct FastDiv {
  uint32_t d;
  unsigned long long m;  // ceil(2^40 / d)
  __host__ explicit FastDiv(uint32_t div) : d(div), m((((unsigned long long)1 << 40) + div - 1) / div) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)((n * m) >> 40); }
};

// ---- write ---------------------------------------------------------------------------------------------

// When a slot occurs more than once in a call, the last of its tokens is the one that is kept: each CTA
// enters its tokens' slots into a hash table in shared memory (the latest token of a slot wins there) and
// looks the slots of all later tokens up in it.  The rule needs no state between launches and its result
// does not depend on their timing.  The table is thirty-two times too large, so that a slot which is not in it
// is nearly always told by one look.
template <int TOKENS>
struct SlotTable {
  static constexpr uint32_t kSize = 32 * TOKENS;
  long long slot[TOKENS];       // slots of the CTA's tokens; -1: nothing is written
  unsigned short head[kSize];   // 0: empty, else 1 + local token whose slot this entry holds (the latest one)
  uint8_t dead[TOKENS];         // a later token writes the same slot
};

__device__ __forceinline__ uint32_t slot_hash(long long s) {
  uint32_t h = (uint32_t)s ^ (uint32_t)(s >> 32) * 0x9E3779B1u;
  h *= 0x85EBCA6Bu;
  return h ^ (h >> 15);
}

// A row of one head as its group of `group` lanes (a power of two) holds it: lane `sub` has the chunks sub,
// sub + group, .. of sixteen values.
template <typename T, int CHUNKS>
struct Row {
  Chunk<T> c[CHUNKS];
  __device__ __forceinline__ void load(const T* x, int chunks, int group, int sub, bool ok, int wide) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      if (ok && sub + i * group < chunks) c[i].load(x + (sub + i * group) * 16, wide);
      else c[i].clear();
    }
  }
};

// Encode a row and store it at `row` of the cache.  Every lane of the warp takes part (shuffles, whose mask is
// the constant full one: a mask that names the group costs a synchronisation unit's round trip each);
// `ok` says whether the row is written.
template <typename T, bool MXF, int CHUNKS>
__device__ __forceinline__ void encode_row(const Side& sd, const Row<T, CHUNKS>& x, size_t row, int dim, int group, int sub,
                                           bool ok) {
  const int chunks = dim / 16;
  if (MXF) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = sub + i * group;
      const uint32_t byte = mx::block_byte<T>(x.c[i]);
      if (ok && c < chunks) {
        reinterpret_cast<uint2*>(sd.codes + row * (dim / 2))[c] = mx::encode16<T>(x.c[i], byte);
        if ((c & 1) == 0) sd.scales[row * (dim / 32) + c / 2] = (uint8_t)byte;
      }
    }
  } else {
    uint32_t m = x.c[0].amax();
#pragma unroll
    for (int i = 1; i < CHUNKS; ++i) m = Chunk<T>::merge(m, x.c[i].amax());
    for (int o = group >> 1; o > 0; o >>= 1) m = Chunk<T>::merge(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!ok) return;
    const uint32_t amax = Chunk<T>::amax_bits(m);
    // the arithmetic of the per-token encode on the grid [-128, 127]; a row that holds a NaN or an
    // infinity has no scale and reads back as NaN
    const float scale = amax >= 0x7f800000u ? __uint_as_float(0x7fffffffu)
                                            : fmaxf(__fdiv_rn(__uint_as_float(amax), 127.5f), 1e-8f);
    const Divisor d = make_divisor(scale);
    const IntGrid grid = make_int_grid(0.0f, -128.0f, 127.0f, -128, 127);
    const ShortDiv by_scale = make_short_div(d);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = sub + i * group;
      if (c >= chunks) continue;
      uint32_t w[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[8];
        x.c[i].values(h, f);
        const float a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
        if (d.fast) {  // every quotient is at most 127.5 in magnitude
          int q[4];
          code4_short(a, by_scale, grid, q);
          w[2 * h] = pack4i_s8(q);
          code4_short(b, by_scale, grid, q);
          w[2 * h + 1] = pack4i_s8(q);
        } else {
          float q[4];
          code4_f32(a, d, 0.0f, -128.0f, 127.0f, q);
          w[2 * h] = pack4_s8(q);
          code4_f32(b, d, 0.0f, -128.0f, 127.0f, q);
          w[2 * h + 1] = pack4_s8(q);
        }
      }
      reinterpret_cast<uint4*>(sd.codes + row * dim)[c] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (sub == 0) reinterpret_cast<float*>(sd.scales)[row] = scale;
  }
}

// A CTA takes TOKENS tokens (and with gridDim.y > 1 a share of the heads).  The loads of its first rows are on
// their way while the table of slots is built; a group of lanes keeps four rows of bf16 (128 bytes a lane) in
// flight.
template <typename T, bool MXF, int TOKENS, int CHUNKS>
__global__ void __launch_bounds__(kThreads)
kv_write_kernel(const Side k, const Side v, const void* __restrict__ slots, int slot_bits, size_t tokens, long long n_slots,
                int heads, int dim, int group, const FastDiv per_token, int wide, int32_t* status) {
  constexpr int kInFlight = 8 / (int)sizeof(T) / CHUNKS;
  __shared__ SlotTable<TOKENS> tab;
  const size_t t0 = (size_t)blockIdx.x * TOKENS;
  const int mine = (int)(tokens - t0 < (size_t)TOKENS ? tokens - t0 : (size_t)TOKENS);
  const int per = (int)per_token.d / 2, h0 = blockIdx.y * per, here = min(per, heads - h0);  // heads of this CTA
  const int lane = threadIdx.x & 31, sub = lane & (group - 1);
  const int groups = kThreads / group, rows = mine * (int)per_token.d;  // (token, head, side)
  const int r_first = (int)threadIdx.x / group;
  Row<T, CHUNKS> x[kInFlight];
  auto place = [&](int r, int& token, int& head, int& side) {
    token = (int)per_token((uint32_t)r);
    const int w = r - token * (int)per_token.d;
    side = w & 1, head = w >> 1;
    return r < rows && head < here;
  };
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      int token, head, side;
      const bool ok = place(r0 + u * groups, token, head, side);
      const Side& sd = side ? v : k;
      x[u].load(reinterpret_cast<const T*>(sd.rows) + (long long)(t0 + token) * sd.token + (h0 + head) * sd.head, dim / 16, group, sub, ok, wide);
    }
  };
  load(r_first);

  constexpr uint32_t kSize = SlotTable<TOKENS>::kSize;
  for (uint32_t i = threadIdx.x; i < kSize / 8; i += kThreads) reinterpret_cast<uint4*>(tab.head)[i] = make_uint4(0, 0, 0, 0);
  for (int i = threadIdx.x; i < mine; i += kThreads) {
    long long s = index_at(slots, slot_bits, t0 + i);
    if (s >= n_slots) {
      s = -1;
      if (status) atomicExch(status, (int)LQ_ERR_SHAPE);
    }
    tab.slot[i] = s < 0 ? -1 : s;
    tab.dead[i] = 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < mine; i += kThreads) {
    const long long s = tab.slot[i];
    if (s < 0) continue;
    for (uint32_t h = slot_hash(s) % kSize;; h = (h + 1) % kSize) {
      unsigned short old = atomicCAS(&tab.head[h], (unsigned short)0, (unsigned short)(i + 1));
      if (old == 0) break;
      if (tab.slot[old - 1] != s) continue;
      // the entry stays with this slot: keep its latest token
      while (old < i + 1) {
        const unsigned short now = atomicCAS(&tab.head[h], old, (unsigned short)(i + 1));
        if (now == old) break;
        old = now;
      }
      tab.dead[old < i + 1 ? old - 1 : i] = 1;
      break;
    }
  }
  __syncthreads();
  constexpr int kAhead = 4;
  for (size_t t = t0 + TOKENS + threadIdx.x; t < tokens; t += kAhead * kThreads) {
    long long s[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) s[j] = t + j * kThreads < tokens ? index_at(slots, slot_bits, t + j * kThreads) : -1;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (s[j] < 0) continue;
      for (uint32_t h = slot_hash(s[j]) % kSize;; h = (h + 1) % kSize) {
        const int e = tab.head[h];
        if (e == 0) break;
        if (tab.slot[e - 1] == s[j]) {
          tab.dead[e - 1] = 1;
          break;
        }
      }
    }
  }
  __syncthreads();

  for (int r0 = r_first; r0 - r_first < rows; r0 += kInFlight * groups) {
    if (r0 != r_first) load(r0);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      int token, head, side;
      bool ok = place(r0 + u * groups, token, head, side);
      const long long s = ok ? tab.slot[token] : -1;
      ok = ok && s >= 0 && !tab.dead[token];
      encode_row<T, MXF, CHUNKS>(side ? v : k, x[u], (size_t)(ok ? s : 0) * heads + h0 + head, dim, group, sub, ok);
    }
  }
}

// ---- read ----------------------------------------------------------------------------------------------

struct Table {
  const int* pages;
  long long stride;
  int max_blocks;
  const int* cu;
  const int* starts;
  int seqs;
  long long n_pages;
  int page;
};

// Slot of output row r, -1 where the table has none for it; `covered` says whether a sequence has the row.
__device__ __forceinline__ long long find_slot(const Table& t, long long r, bool& covered) {
  covered = r < (long long)__ldg(t.cu + t.seqs) && r >= (long long)__ldg(t.cu);
  if (!covered) return -1;
  int lo = 0, hi = t.seqs;  // the first index with cu[index] > r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((long long)__ldg(t.cu + mid) > r) hi = mid;
    else lo = mid + 1;
  }
  if (lo == 0) return -1;  // cu does not ascend
  const int b = lo - 1;
  const long long pos = r - __ldg(t.cu + b) + (t.starts ? __ldg(t.starts + b) : 0);
  if (pos < 0 || pos > 0x7fffffffll) return -1;
  const int blk = (int)pos / t.page;
  if (blk >= t.max_blocks) return -1;
  const long long p = __ldg(t.pages + b * t.stride + blk);
  return p < 0 || p >= t.n_pages ? -1 : p * t.page + (int)pos % t.page;
}

// A warp reads TOKENS consecutive output rows.  Its lanes first look up one row each (the search through
// cu_seqlens and the page table is a chain of dependent loads, so it is walked for all rows at once), then
// walk the rows' values together, 16 of a head per lane and step, four steps' loads in flight.  Bound by HBM:
// a byte (half a byte) read and two or four written per value.
template <typename T, bool MXF, int TOKENS>
__global__ void __launch_bounds__(kThreads)
kv_read_kernel(const Side k, const Side v, const Table t, int heads, const FastDiv per_row, const FastDiv per_side,
               const FastDiv per_head, long long total, int clear_tail, int wide, int32_t* status) {
  const long long r0 = (((long long)blockIdx.x * kThreads + threadIdx.x) >> 5) * TOKENS;
  if (r0 >= total) return;
  const int lane = threadIdx.x & 31;
  const int rows = (int)(total - r0 < TOKENS ? total - r0 : TOKENS);
  long long slot = -2;  // -2: left alone, -1: zeros
  if (lane < rows) {
    bool covered;
    slot = find_slot(t, r0 + lane, covered);
    if (slot < 0 && covered && status) atomicExch(status, (int)LQ_ERR_SHAPE);
    if (!covered) slot = clear_tail ? -1 : -2;
  }
  const uint32_t chunks = rows * per_row.d;  // 16 values each: row, keys or values, head, place in the head
  const int dim = (int)per_head.d * 16;
  constexpr int kSteps = 4;
  for (uint32_t c0 = 0; c0 < chunks; c0 += 32 * kSteps) {
    uint4 code[kSteps];
    float scale[kSteps];
    T* dst[kSteps];
    long long at[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const uint32_t c = c0 + u * 32 + lane;
      const uint32_t i = per_row(c);
      at[u] = __shfl_sync(0xffffffffu, slot, i < TOKENS ? i : 0);
      if (c >= chunks) at[u] = -2;
      const uint32_t w = c - i * per_row.d, side = per_side(w), x = w - side * per_side.d;
      const uint32_t head = per_head(x), d0 = (x - head * per_head.d) * 16;
      const Side& sd = side ? v : k;
      dst[u] = reinterpret_cast<T*>(sd.rows) + (r0 + i) * sd.token + head * sd.head + d0;
      if (at[u] >= 0) {
        const size_t row = (size_t)at[u] * heads + head;
        if (MXF) {
          const uint2 q = __ldg(reinterpret_cast<const uint2*>(sd.codes + row * (dim / 2) + d0 / 2));
          code[u] = make_uint4(q.x, q.y, 0, 0);
          scale[u] = mx::scale_value(__ldg(sd.scales + row * (dim / 32) + d0 / 32));
        } else {
          code[u] = ld_stream_u4(sd.codes + row * dim + d0);
          scale[u] = __ldg(reinterpret_cast<const float*>(sd.scales) + row);
        }
      } else {
        code[u] = make_uint4(0, 0, 0, 0), scale[u] = 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      if (at[u] == -2) continue;
      float lo[8], hi[8];
      if (MXF) {
        mx::decode8(code[u].x, lo);
        mx::decode8(code[u].y, hi);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = (float)(int8_t)(code[u].x >> (8 * j)), lo[4 + j] = (float)(int8_t)(code[u].y >> (8 * j));
          hi[j] = (float)(int8_t)(code[u].z >> (8 * j)), hi[4 + j] = (float)(int8_t)(code[u].w >> (8 * j));
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) lo[j] = __fmul_rn(lo[j], scale[u]), hi[j] = __fmul_rn(hi[j], scale[u]);
      mx::store16(dst[u], lo, hi, wide);
    }
  }
}

int check_format(const std::string& w, int format, size_t heads, size_t dim) {
  if (format != LQ_KV_INT8 && format != LQ_KV_MXFP4) return fail(LQ_ERR_UNSUPPORTED, w + ": unknown cache format");
  if (heads == 0 || heads > 4096) return fail(LQ_ERR_SHAPE, w + ": between 1 and 4096 heads");
  const size_t step = format == LQ_KV_INT8 ? 16 : 32;
  if (dim == 0 || dim % step != 0 || dim > (size_t)kMaxDim)
    return fail(LQ_ERR_SHAPE, w + ": head_dim must be a multiple of " + std::to_string(step) + ", at most " + std::to_string(kMaxDim));
  return LQ_OK;
}

template <typename T, bool MXF, int TOKENS, int CHUNKS>
int write_tokens(const Side& k, const Side& v, const void* slots, int slot_bits, size_t tokens, long long n_slots, int heads,
                 int dim, int group, int wide, int32_t* status, cudaStream_t st) {
  const size_t tiles = (tokens + TOKENS - 1) / TOKENS;
  if (tiles > 0x7fffffffu) return fail(LQ_ERR_SHAPE, "lq_kv_write: too many tokens for one launch");
  // heads shared out until every SM has a CTA: a share repeats the table, but reads other rows
  int per = heads;
  while (per > 1 && tiles * (size_t)((heads + per - 1) / per) < 2 * (size_t)sm_count()) per = (per + 1) / 2;
  kv_write_kernel<T, MXF, TOKENS, CHUNKS><<<dim3((unsigned)tiles, (unsigned)((heads + per - 1) / per)), kThreads, 0, st>>>(
      k, v, slots, slot_bits, tokens, n_slots, heads, dim, group, FastDiv(2 * (uint32_t)per), wide, status);
  return check_cuda(cudaGetLastError(), "lq_kv_write launch");
}
template <typename T, bool MXF, int CHUNKS>
int write_chunks(const Side& k, const Side& v, const void* slots, int slot_bits, size_t tokens, long long n_slots, int heads,
                 int dim, int group, int wide, int32_t* status, cudaStream_t st) {
  // Every CTA looks at the slots of all later tokens, so its share of the tokens grows with their number.
  if (tokens <= 8192) return write_tokens<T, MXF, 16, CHUNKS>(k, v, slots, slot_bits, tokens, n_slots, heads, dim, group, wide, status, st);
  if (tokens <= 65536) return write_tokens<T, MXF, 64, CHUNKS>(k, v, slots, slot_bits, tokens, n_slots, heads, dim, group, wide, status, st);
  return write_tokens<T, MXF, 256, CHUNKS>(k, v, slots, slot_bits, tokens, n_slots, heads, dim, group, wide, status, st);
}
template <typename T, bool MXF>
int write_dispatch(const Side& k, const Side& v, const void* slots, int slot_bits, size_t tokens, long long n_slots, int heads,
                   int dim, int wide, int32_t* status, cudaStream_t st) {
  int group = MXF ? 2 : 1;
  while (group < 32 && group * 16 < dim) group *= 2;
  if (dim <= 512) return write_chunks<T, MXF, 1>(k, v, slots, slot_bits, tokens, n_slots, heads, dim, group, wide, status, st);
  return write_chunks<T, MXF, 2>(k, v, slots, slot_bits, tokens, n_slots, heads, dim, group, wide, status, st);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" int lq_kv_write(const void* k, const void* v, int in_dtype, size_t tokens, size_t heads, size_t dim, size_t k_token,
                           size_t k_head, size_t v_token, size_t v_head, const void* slots, int slot_bits, size_t n_slots, int format,
                           void* k_codes, void* k_scales, void* v_codes, void* v_scales, int32_t* status, void* stream) {
  if (tokens == 0) return LQ_OK;
  if (!k || !v || !slots || !k_codes || !k_scales || !v_codes || !v_scales) return fail(LQ_ERR_DEVICE, "lq_kv_write: null pointer");
  if (in_dtype != LQ_F32 && in_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_kv_write: k and v must be f32|bf16");
  if (slot_bits != 32 && slot_bits != 64) return fail(LQ_ERR_DTYPE, "lq_kv_write: slots must be int32 or int64");
  if (int rc = check_format("lq_kv_write", format, heads, dim)) return rc;
  const size_t esz = in_dtype == LQ_F32 ? 4 : 2;
  if (!aligned16(k) || !aligned16(v) || (k_token * esz) % 16 || (k_head * esz) % 16 || (v_token * esz) % 16 || (v_head * esz) % 16)
    return fail(LQ_ERR_ALIGNMENT, "lq_kv_write: rows of k and v must be 16-byte aligned");
  if (!aligned16(k_codes) || !aligned16(v_codes) || !aligned16(k_scales) || !aligned16(v_scales))
    return fail(LQ_ERR_ALIGNMENT, "lq_kv_write: the cache must be 16-byte aligned");
  const Side ks = {(uint8_t*)k_codes, (uint8_t*)k_scales, const_cast<void*>(k), (long long)k_token, (long long)k_head};
  const Side vs = {(uint8_t*)v_codes, (uint8_t*)v_scales, const_cast<void*>(v), (long long)v_token, (long long)v_head};
  cudaStream_t st = (cudaStream_t)stream;
  const int h = (int)heads, d = (int)dim;
  const int wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 32 == 0) &&
                   ((k_token | k_head | v_token | v_head) * esz) % 32 == 0;
  if (in_dtype == LQ_F32)
    return format == LQ_KV_MXFP4 ? write_dispatch<float, true>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, wide, status, st)
                                 : write_dispatch<float, false>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, wide, status, st);
  return format == LQ_KV_MXFP4 ? write_dispatch<bf16, true>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, wide, status, st)
                               : write_dispatch<bf16, false>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, wide, status, st);
}

extern "C" int lq_kv_read(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, int format,
                          size_t n_pages, size_t page, size_t heads, size_t dim, const int32_t* table, size_t table_stride,
                          size_t max_blocks, const int32_t* cu_seqlens, const int32_t* starts, size_t seqs, size_t total,
                          void* out_k, void* out_v, int out_dtype, size_t k_token, size_t k_head, size_t v_token, size_t v_head,
                          int clear_tail, int32_t* status, void* stream) {
  if (total == 0) return LQ_OK;
  if (!k_codes || !k_scales || !v_codes || !v_scales || !out_k || !out_v || !cu_seqlens || (!table && max_blocks > 0))
    return fail(LQ_ERR_DEVICE, "lq_kv_read: null pointer");
  if (out_dtype != LQ_F32 && out_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_kv_read: out must be f32|bf16");
  if (int rc = check_format("lq_kv_read", format, heads, dim)) return rc;
  if (page == 0 || page >= ((size_t)1 << 31) || seqs >= ((size_t)1 << 31) || max_blocks >= ((size_t)1 << 31))
    return fail(LQ_ERR_SHAPE, "lq_kv_read: page size, sequences and table width must fit 32 bits, the page not empty");
  if (total >= ((size_t)1 << 31)) return fail(LQ_ERR_SHAPE, "lq_kv_read: at most 2^31 - 1 rows");
  const size_t esz = out_dtype == LQ_F32 ? 4 : 2;
  if (!aligned16(out_k) || !aligned16(out_v) || (k_token * esz) % 16 || (k_head * esz) % 16 || (v_token * esz) % 16 || (v_head * esz) % 16)
    return fail(LQ_ERR_ALIGNMENT, "lq_kv_read: output rows must be 16-byte aligned");
  if (!aligned16(k_codes) || !aligned16(v_codes) || !aligned16(k_scales) || !aligned16(v_scales))
    return fail(LQ_ERR_ALIGNMENT, "lq_kv_read: the cache must be 16-byte aligned");
  const Side ks = {(uint8_t*)const_cast<void*>(k_codes), (uint8_t*)const_cast<void*>(k_scales), out_k, (long long)k_token, (long long)k_head};
  const Side vs = {(uint8_t*)const_cast<void*>(v_codes), (uint8_t*)const_cast<void*>(v_scales), out_v, (long long)v_token, (long long)v_head};
  const Table t = {table, (long long)table_stride, (int)max_blocks, cu_seqlens, starts, (int)seqs, (long long)n_pages, (int)page};
  const uint32_t head_chunks = (uint32_t)(dim / 16), side_chunks = head_chunks * (uint32_t)heads;
  const int wide = ((reinterpret_cast<uintptr_t>(out_k) | reinterpret_cast<uintptr_t>(out_v)) % 32 == 0) &&
                   ((k_token | k_head | v_token | v_head) * esz) % 32 == 0;
  // four rows a warp once that still gives every SM a few dozen warps; one row below
  const bool few = total < 4 * 32 * (size_t)sm_count();
  const size_t warps = few ? total : (total + 3) / 4;
  const unsigned grid = (unsigned)((warps * 32 + kThreads - 1) / kThreads);
  cudaStream_t st = (cudaStream_t)stream;
#define LQ_KV_READ(T, F, N)                                                                                              \
  kv_read_kernel<T, F, N><<<grid, kThreads, 0, st>>>(ks, vs, t, (int)heads, FastDiv(2 * side_chunks), FastDiv(side_chunks), \
                                                     FastDiv(head_chunks), (long long)total, clear_tail, wide, status)
#define LQ_KV_READ_T(T)                                     \
  if (format == LQ_KV_MXFP4) {                              \
    if (few) LQ_KV_READ(T, true, 1);                        \
    else LQ_KV_READ(T, true, 4);                            \
  } else {                                                  \
    if (few) LQ_KV_READ(T, false, 1);                       \
    else LQ_KV_READ(T, false, 4);                           \
  }
  if (out_dtype == LQ_F32) {
    LQ_KV_READ_T(float)
  } else {
    LQ_KV_READ_T(bf16)
  }
#undef LQ_KV_READ_T
#undef LQ_KV_READ
  return check_cuda(cudaGetLastError(), "lq_kv_read launch");
}
