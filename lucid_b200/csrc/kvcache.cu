// The quantized key / value cache: rows encoded as they are written, and read back by page table.
//
// A cache row is one token's (heads, dim) values, kept contiguous (page, offset, head, dim), so a write is one
// pass over the new tokens and a read one pass over the tokens asked for.  Two formats:
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
// Plain loads (through L1, not the read-only path: see load_once) of what a few lanes or warps share.
__device__ __forceinline__ int load_common(const int* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ long long load_common(const long long* p) {
  long long v;
  asm volatile("ld.global.s64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float load_common(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_common(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 load_common(const uint2* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ long long index_at(const void* p, int bits, size_t i) {
  return bits == 64 ? load_common(reinterpret_cast<const long long*>(p) + i) : (long long)load_common(reinterpret_cast<const int*>(p) + i);
}

// n / d for n * d < 2^43 (the rounding of m adds less than d * n / 2^43 < 1 / d to the quotient), n < 2^31, by the
// upper half of a 64-bit product
struct FastDiv {
  uint32_t d;
  unsigned long long m;  // 2^20 * ceil(2^43 / d)
  __host__ explicit FastDiv(uint32_t div) : d(div), m(((((unsigned long long)1 << 43) + div - 1) / div) << 20) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)__umul64hi((unsigned long long)n << 1, m); }
};

// ---- write ---------------------------------------------------------------------------------------------

// When a slot occurs more than once in a call, the last of its tokens is the one that is kept, whatever the
// timing and without state between launches.  Up to kInline tokens, the warp that holds a token's rows compares
// its slot with those of all later tokens itself; for more, a kernel of its own marks the tokens that are
// overwritten: a CTA enters its tokens' slots into a hash table in shared memory (the latest token of a slot
// wins there) and looks the slots of all later tokens up in it.  The table is many times too large, so that a
// slot which is not in it is nearly always told by one look.  The looks grow with the square of the tokens, and with
// narrow rows they are most of the time: 1 x 64 in MXFP4, 8192 tokens 7.8 us, 131072 62 us (6.5 us of rows at the
// measured copy's rate).  (Inside the write itself the looks and their barriers cost 5 of 22 us at 8192 tokens, and
// more than the rows at 32.  256 tokens of 8 x 128, the whole write: 5.0 us in int8 and 4.1 in MXFP4 with the comparison
// in the warp, 5.3 and 4.4 with two kernels, which cost the host a launch and an allocation more.)
constexpr int kInline = 256;
constexpr int kMarkThreads = 1024;
template <int TOKENS>
struct SlotTable {
  static constexpr uint32_t kSize = (TOKENS <= 256 ? 32 : 8) * TOKENS;
  long long slot[TOKENS];                   // slots of the CTA's tokens; negative: nothing is written
  alignas(16) unsigned short head[kSize];   // 0: empty, else 1 + local token whose slot this entry holds (the latest one)
  uint8_t dead[TOKENS];                     // a later token writes the same slot
};

__device__ __forceinline__ uint32_t slot_hash(long long s) {
  uint32_t h = (uint32_t)s ^ (uint32_t)(s >> 32) * 0x9E3779B1u;
  h *= 0x85EBCA6Bu;
  return h ^ (h >> 15);
}

template <int TOKENS>
__global__ void __launch_bounds__(kMarkThreads)
kv_mark_kernel(const void* __restrict__ slots, int slot_bits, size_t tokens, uint8_t* __restrict__ dead) {
  constexpr uint32_t kSize = SlotTable<TOKENS>::kSize;
  __shared__ SlotTable<TOKENS> tab;
  pdl_wait();
  pdl_launch_dependents();
  const size_t t0 = (size_t)blockIdx.x * TOKENS;
  const int mine = (int)(tokens - t0 < (size_t)TOKENS ? tokens - t0 : (size_t)TOKENS);
  for (uint32_t i = threadIdx.x; i < kSize / 8; i += kMarkThreads) reinterpret_cast<uint4*>(tab.head)[i] = make_uint4(0, 0, 0, 0);
  for (int i = threadIdx.x; i < mine; i += kMarkThreads) tab.slot[i] = index_at(slots, slot_bits, t0 + i), tab.dead[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < mine; i += kMarkThreads) {
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
  for (size_t t = t0 + TOKENS + threadIdx.x; t < tokens; t += kAhead * kMarkThreads) {
    long long s[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) s[j] = t + j * kMarkThreads < tokens ? index_at(slots, slot_bits, t + j * kMarkThreads) : -1;
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
  for (int i = threadIdx.x; i < mine; i += kMarkThreads) dead[t0 + i] = tab.dead[i];
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
__device__ __forceinline__ void encode_row(const Side& sd, const Row<T, CHUNKS>& x, size_t row, int dim, int group, int sub, bool ok) {
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
    // The arithmetic of the per-token encode on the grid [-128, 127]: correctly rounded quotients by twice
    // corrected reciprocals.  Every intermediate keeps its bits where a code depends on them: the scale is
    // between 1e-8 and 2^121, a quotient at most 127.5, and an abs-max small enough to lose bits in the first
    // division is below the 1e-8.  A row that holds a NaN or an infinity takes a NaN scale and reads back as NaN.
    const float a = __uint_as_float(amax);
    float q0 = __fmul_rn(a, 1.0f / 127.5f);
    q0 = __fmaf_rn(__fmaf_rn(-q0, 127.5f, a), 1.0f / 127.5f, q0);
    q0 = __fmaf_rn(__fmaf_rn(-q0, 127.5f, a), 1.0f / 127.5f, q0);
    const float scale = amax >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fmaxf(q0, 1e-8f);
    const float y = __frcp_rn(scale);
    ShortDiv by_scale;
    by_scale.y2 = f2_pack(y, y), by_scale.ns2 = f2_pack(-scale, -scale);
    const IntGrid grid = make_int_grid(0.0f, -128.0f, 127.0f, -128, 127);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = sub + i * group;
      if (c >= chunks) continue;
      uint32_t w[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[8];
        x.c[i].values(h, f);
        const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
        int q[4];
        code4_short(lo, by_scale, grid, q);
        w[2 * h] = pack4i_s8(q);
        code4_short(hi, by_scale, grid, q);
        w[2 * h + 1] = pack4i_s8(q);
      }
      reinterpret_cast<uint4*>(sd.codes + row * dim)[c] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (sub == 0) reinterpret_cast<float*>(sd.scales)[row] = scale;
  }
}

// blockIdx.y: keys or values.  A warp takes ROWS times as many consecutive (token, head) rows as fit side by side
// (32 / group), all loads first; no warp waits for another.  8192 tokens of 8 x 128 bf16, with the marking: 18.7 us in
// int8, 15.6 in MXFP4 (2.7 TB/s): the marking before it, then instruction issue (62 and 58 % of the cycles).  MARKED: the
// kernel before this one marks the overwritten tokens.  The rows, which an earlier kernel wrote, are not fetched while
// that one runs (16.6 and 13.6 us): only griddepcontrol.wait promises this grid the writes of the kernels before it.
template <typename T, bool MXF, int CHUNKS, int ROWS, bool MARKED>
__global__ void __launch_bounds__(kThreads)
kv_write_kernel(const Side k, const Side v, const void* __restrict__ slots, int slot_bits, uint32_t tokens, long long n_slots,
                const FastDiv by_heads, long long rows, int dim, int group_bits, const uint8_t* dead, int wide,
                int32_t* status) {
  const int lane = threadIdx.x & 31, group = 1 << group_bits, sub = lane & (group - 1);
  const Side& sd = blockIdx.y ? v : k;
  const int heads = (int)by_heads.d, across = 32 >> group_bits;
  const long long r0 = ((long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * (ROWS * across) + (lane >> group_bits);
  pdl_wait();
  pdl_launch_dependents();
  Row<T, CHUNKS> x[ROWS];
  long long slot[ROWS];
  uint32_t token[ROWS];
  int head[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const long long r = r0 + u * across;
    const bool ok = r < rows;
    token[u] = ok ? by_heads((uint32_t)r) : 0;
    head[u] = ok ? (int)((uint32_t)r - token[u] * heads) : 0;
    x[u].load(reinterpret_cast<const T*>(sd.rows) + token[u] * sd.token + head[u] * sd.head, dim / 16, group, sub, ok, wide);
    slot[u] = ok ? index_at(slots, slot_bits, token[u]) : -1;
  }
  if constexpr (MARKED) {
#pragma unroll
    for (int u = 0; u < ROWS; ++u)
      if (slot[u] >= 0 && dead[token[u]]) slot[u] = -1;
  } else {
    // each lane keeps a share of all slots; every token among the warp's rows is compared with all of them
    long long all[kInline / 32];
#pragma unroll
    for (int j = 0; j < kInline / 32; ++j) all[j] = lane + 32 * j < tokens ? index_at(slots, slot_bits, lane + 32 * j) : -1;
    uint32_t last = 0xffffffffu;
    bool again = false;
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
#pragma unroll 1
      for (int i = 0; i < 32; i += group) {
        const uint32_t t = __shfl_sync(0xffffffffu, token[u], i);
        const long long s = __shfl_sync(0xffffffffu, slot[u], i);
        if (t != last) {  // the same for the whole warp
          again = false;
#pragma unroll
          for (int j = 0; j < kInline / 32; ++j) again |= all[j] == s && lane + 32 * j > t;
          again = __any_sync(0xffffffffu, again);
          last = t;
        }
        if (again && lane >= i && lane < i + group) slot[u] = -1;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    if (slot[u] >= n_slots) {
      if (status) atomicExch(status, (int)LQ_ERR_SHAPE);
      slot[u] = -1;
    }
    const bool ok = slot[u] >= 0;
    encode_row<T, MXF, CHUNKS>(sd, x[u], (size_t)(ok ? slot[u] : 0) * heads + head[u], dim, group, sub, ok);
  }
}

// ---- read ----------------------------------------------------------------------------------------------

// n / d for n * d < 2^31, in two instructions
struct SmallDiv {
  uint32_t d, m;  // ceil(2^31 / d)
  __host__ explicit SmallDiv(uint32_t div) : d(div), m((uint32_t)((((unsigned long long)1 << 31) + div - 1) / div)) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return __umulhi(n << 1, m); }
};

// How the 16-value chunks of an output row are numbered: keys before values, head by head.
struct RowShape {
  uint32_t chunks, side;       // of a row, of its keys
  SmallDiv head;               // chunks of a head
  uint32_t step_rows, step;    // 32 chunks on: this many rows and this many chunks
};

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
  covered = r < (long long)load_common(t.cu + t.seqs) && r >= (long long)load_common(t.cu);
  if (!covered) return -1;
  int lo = 0, hi = t.seqs;  // the first index with cu[index] > r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((long long)load_common(t.cu + mid) > r) hi = mid;
    else lo = mid + 1;
  }
  if (lo == 0) return -1;  // cu does not ascend
  const int b = lo - 1;
  const long long pos = r - load_common(t.cu + b) + (t.starts ? load_common(t.starts + b) : 0);
  if (pos < 0 || pos > 0x7fffffffll) return -1;
  const int blk = (int)pos / t.page;
  if (blk >= t.max_blocks) return -1;
  const long long p = load_common(t.pages + b * t.stride + blk);
  return p < 0 || p >= t.n_pages ? -1 : p * t.page + (int)pos % t.page;
}

// A warp reads TOKENS consecutive output rows.  Its lanes first look up one row each (the search through
// cu_seqlens and the page table is a chain of dependent loads, so it is walked for all rows at once), then
// walk the rows' values together, 16 of a head per lane and step, four steps' loads in flight.  Bound by HBM:
// a byte (half a byte) read and two or four written per value; 67615 rows of 8 x 128 to bf16: 72 us in int8 (5.8
// TB/s), 70 in MXFP4.
template <typename T, bool MXF, int TOKENS>
__global__ void __launch_bounds__(kThreads)
kv_read_kernel(const Side k, const Side v, const Table t, int heads, const RowShape shape, long long total, int clear_tail,
               int wide, int32_t* status) {
  const long long r0 = (((long long)blockIdx.x * kThreads + threadIdx.x) >> 5) * TOKENS;
  pdl_wait();
  pdl_launch_dependents();
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
  const int dim = (int)shape.head.d * 16;
  constexpr int kSteps = 4;
  uint32_t i = (uint32_t)lane / shape.chunks, w = (uint32_t)lane - i * shape.chunks;  // row and chunk of this lane's next step
  const uint32_t steps = (rows * shape.chunks + 31) / 32;
  for (uint32_t s0 = 0; s0 < steps; s0 += kSteps) {
    uint4 code[kSteps];
    float scale[kSteps];
    T* dst[kSteps];
    long long at[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      at[u] = __shfl_sync(0xffffffffu, slot, i < TOKENS ? i : 0);
      if (i >= (uint32_t)rows) at[u] = -2;
      const bool is_v = w >= shape.side;
      const uint32_t x = is_v ? w - shape.side : w, head = shape.head(x), d0 = (x - head * shape.head.d) * 16;
      const Side& sd = is_v ? v : k;
      dst[u] = reinterpret_cast<T*>(sd.rows) + (r0 + i) * sd.token + head * sd.head + d0;
      i += shape.step_rows, w += shape.step;
      if (w >= shape.chunks) w -= shape.chunks, ++i;
      if (at[u] >= 0) {
        const size_t row = (size_t)at[u] * heads + head;
        if (MXF) {
          const uint2 q = load_common(reinterpret_cast<const uint2*>(sd.codes + row * (dim / 2) + d0 / 2));
          code[u] = make_uint4(q.x, q.y, 0, 0);
          scale[u] = mx::scale_value(load_common(sd.scales + row * (dim / 32) + d0 / 32));
        } else {
          code[u] = mx::load_once(sd.codes + row * dim + d0);
          scale[u] = load_common(reinterpret_cast<const float*>(sd.scales) + row);
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

template <int TOKENS>
int mark(const void* slots, int slot_bits, size_t tokens, uint8_t* dead, cudaStream_t st) {
  return check_cuda(launch_pdl(kv_mark_kernel<TOKENS>, dim3((unsigned)((tokens + TOKENS - 1) / TOKENS)), dim3(kMarkThreads), 0, st, slots,
                               slot_bits, tokens, dead),
                    "lq_kv_write (mark) launch");
}
template <typename T, bool MXF, int CHUNKS>
int write_rows(const Side& k, const Side& v, const void* slots, int slot_bits, size_t tokens, long long n_slots, int heads, int dim,
               int group_bits, const uint8_t* dead, int wide, int32_t* status, cudaStream_t st) {
  constexpr int ROWS = 8 / (int)sizeof(T) / CHUNKS;  // 128 bytes a lane in flight
  const long long rows = (long long)tokens * heads, per_cta = (long long)(kThreads / 32) * ROWS * (32 >> group_bits);
  auto kernel = dead ? kv_write_kernel<T, MXF, CHUNKS, ROWS, true> : kv_write_kernel<T, MXF, CHUNKS, ROWS, false>;
  return check_cuda(launch_pdl(kernel, dim3((unsigned)((rows + per_cta - 1) / per_cta), 2), dim3(kThreads), 0, st, k, v, slots,
                               slot_bits, (uint32_t)tokens, n_slots, FastDiv((uint32_t)heads), rows, dim, group_bits, dead,
                               wide, status),
                    "lq_kv_write launch");
}
template <typename T, bool MXF>
int write_dispatch(const Side& k, const Side& v, const void* slots, int slot_bits, size_t tokens, long long n_slots, int heads,
                   int dim, uint8_t* dead, int wide, int32_t* status, cudaStream_t st) {
  int group_bits = MXF ? 1 : 0;
  while (group_bits < 5 && (16 << group_bits) < dim) ++group_bits;
  if (tokens > kInline) {
    // every CTA looks at the slots of all later tokens: few tokens a CTA until the looks outweigh the shorter
    // table (us of the whole write in MXFP4, 128 / 1024 tokens a CTA: 32768 tokens 45.8 / 49.3, 131072 213 / 175)
    if (int rc = tokens <= 65536 ? mark<128>(slots, slot_bits, tokens, dead, st) : mark<1024>(slots, slot_bits, tokens, dead, st)) return rc;
  } else {
    dead = nullptr;
  }
  if (dim <= 512) return write_rows<T, MXF, 1>(k, v, slots, slot_bits, tokens, n_slots, heads, dim, group_bits, dead, wide, status, st);
  return write_rows<T, MXF, 2>(k, v, slots, slot_bits, tokens, n_slots, heads, dim, group_bits, dead, wide, status, st);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_kv_write_workspace_bytes(size_t tokens) { return tokens > (size_t)kInline ? tokens : 0; }

extern "C" int lq_kv_write(const void* k, const void* v, int in_dtype, size_t tokens, size_t heads, size_t dim, size_t k_token,
                           size_t k_head, size_t v_token, size_t v_head, const void* slots, int slot_bits, size_t n_slots, int format,
                           void* k_codes, void* k_scales, void* v_codes, void* v_scales, void* workspace, size_t workspace_bytes,
                           int32_t* status, void* stream) {
  if (tokens == 0) return LQ_OK;
  // a cache without pages has no memory: every slot is past it
  if (!k || !v || !slots || (n_slots > 0 && (!k_codes || !k_scales || !v_codes || !v_scales)))
    return fail(LQ_ERR_DEVICE, "lq_kv_write: null pointer");
  if (in_dtype != LQ_F32 && in_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_kv_write: k and v must be f32|bf16");
  if (slot_bits != 32 && slot_bits != 64) return fail(LQ_ERR_DTYPE, "lq_kv_write: slots must be int32 or int64");
  if (int rc = check_format("lq_kv_write", format, heads, dim)) return rc;
  // row numbers are 32-bit (2^31 rows of 16 values are 137 GB of float32)
  if (tokens > 0x7fffffffu / heads) return fail(LQ_ERR_SHAPE, "lq_kv_write: tokens x heads must be below 2^31");
  if (workspace_bytes < lq_kv_write_workspace_bytes(tokens) || (!workspace && tokens > (size_t)kInline))
    return fail(LQ_ERR_WORKSPACE, "lq_kv_write: workspace too small");
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
    return format == LQ_KV_MXFP4 ? write_dispatch<float, true>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, (uint8_t*)workspace, wide, status, st)
                                 : write_dispatch<float, false>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, (uint8_t*)workspace, wide, status, st);
  return format == LQ_KV_MXFP4 ? write_dispatch<bf16, true>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, (uint8_t*)workspace, wide, status, st)
                               : write_dispatch<bf16, false>(ks, vs, slots, slot_bits, tokens, (long long)n_slots, h, d, (uint8_t*)workspace, wide, status, st);
}

extern "C" int lq_kv_read(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, int format,
                          size_t n_pages, size_t page, size_t heads, size_t dim, const int32_t* table, size_t table_stride,
                          size_t max_blocks, const int32_t* cu_seqlens, const int32_t* starts, size_t seqs, size_t total,
                          void* out_k, void* out_v, int out_dtype, size_t k_token, size_t k_head, size_t v_token, size_t v_head,
                          int clear_tail, int32_t* status, void* stream) {
  if (total == 0) return LQ_OK;
  if (!out_k || !out_v || !cu_seqlens || (!table && seqs > 0 && max_blocks > 0) ||
      (n_pages > 0 && (!k_codes || !k_scales || !v_codes || !v_scales)))
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
  const RowShape shape = {2 * side_chunks, side_chunks, SmallDiv(head_chunks), 32 / (2 * side_chunks), 32 % (2 * side_chunks)};
  const int wide = ((reinterpret_cast<uintptr_t>(out_k) | reinterpret_cast<uintptr_t>(out_v)) % 32 == 0) &&
                   ((k_token | k_head | v_token | v_head) * esz) % 32 == 0;
  // Rows a warp: one, or four or sixteen of short rows once that still leaves enough warps (their look-ups then
  // overlap).  Measured, 1 / 4 / 16 rows, us, in one sequence (in 32): int8 8 x 128, 16384 rows 19.8 / 22.2 / 32.8 (20.9 /
  // 22.9 / 33.3), 32768 35.9 / 37.1 / 42.9 (37.7 / 37.6 / 43.4), 49152 51.7 / 52.7 / 60.7 (54.0 / 53.7 / 60.3), 65536 67.9 /
  // 68.1 / 80.0 (70.6 / 69.2 / 81.7); int8 8 x 64, 4096 4.7 / 5.1 / 13.6, 16384 13.5 / 10.4 / 17.1; int8 1 x 64, 4096 4.1 /
  // 2.9 / 3.6, 16384 10.6 / 4.1 / 3.7, 65536 37.7 / 11.4 / 6.3; MXFP4 8 x 128, 16384 21.2 / 20.0 / 40.7, 65536 71.6 / 66.5 /
  // 66.4; MXFP4 4 x 64, 4096 4.0 / 3.8 / 7.8, 36903 23.5 / 12.2 / 12.7, 65536 40.8 / 21.1 / 18.7.
  auto fits = [&](size_t n) {
    const size_t work = n * shape.chunks;  // chunks of sixteen values a warp
    const size_t enough = work <= 128 ? 1024 : (work <= 256 || format == LQ_KV_MXFP4 ? 4096 : 16384);
    return work <= 512 && total >= n * enough;
  };
  const size_t per_warp = fits(16) ? 16 : (fits(4) ? 4 : 1);
  const size_t warps = (total + per_warp - 1) / per_warp;
  const unsigned grid = (unsigned)((warps * 32 + kThreads - 1) / kThreads);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
#define LQ_KV_READ(T, F, N)                                                                                         \
  e = launch_pdl(kv_read_kernel<T, F, N>, dim3(grid), dim3(kThreads), 0, st, ks, vs, t, (int)heads, shape, (long long)total, \
                 clear_tail, wide, status)
#define LQ_KV_READ_T(T, F)                     \
  if (per_warp == 1) LQ_KV_READ(T, F, 1);      \
  else if (per_warp == 4) LQ_KV_READ(T, F, 4); \
  else LQ_KV_READ(T, F, 16);
  if (out_dtype == LQ_F32) {
    if (format == LQ_KV_MXFP4) { LQ_KV_READ_T(float, true) } else { LQ_KV_READ_T(float, false) }
  } else {
    if (format == LQ_KV_MXFP4) { LQ_KV_READ_T(bf16, true) } else { LQ_KV_READ_T(bf16, false) }
  }
#undef LQ_KV_READ_T
#undef LQ_KV_READ
  return check_cuda(e, "lq_kv_read launch");
}
