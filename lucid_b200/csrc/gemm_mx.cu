// Product of two MXFP4 matrices on the 4-bit tensor cores (sm_100a):
//   out[m, n] = sum_k a[m, k] * w[n, k] (+ bias[n]) (ReLU), float32 accumulation in TMEM.
//
// tcgen05.mma kind::mxf4 multiplies the packed codes and applies both operands' block scales itself, so the
// kernel moves bytes: codes by TMA (128 bytes = 256 values of K a row and stage, 128-byte swizzle), scale
// tiles by TMA as they lie (1024 bytes = 128 rows x 256 values, which is why the encode writes them that
// way), from shared memory into TMEM by tcgen05.cp.  The weight is the operand whose rows become TMEM
// lanes (128 output features a CTA) and the activations the one whose rows become columns: a decode step
// of a few tokens then pays for 16 columns instead of 128 rows, every lane owns one output feature and
// its bias, and neighbouring lanes store neighbouring outputs.
#include <string.h>

#include <mutex>
#include <type_traits>

#include "microscale.cuh"
#include "tcgen05.cuh"

namespace lq {
namespace {

constexpr int kRows = 128;            // output features of a CTA
constexpr int kStageK = 256;          // values of K per stage: one 128-byte swizzle row
constexpr int kWBytes = kRows * 128;  // weight codes of a stage

struct Args {
  int M, N, num_kb;      // tokens, output features, stages of K
  int tiles_t, tiles_f;
  int split;             // CTAs (a cluster) that share the K axis of a tile
  const void* x;         // activations to encode on the way (fused form): row stride, 32-byte loads, columns
  long long ldx;
  int x_wide, K;
  const float* bias;
  int relu;
  void* out;
  long long ldo;
  int pairs_ok;          // two neighbouring bf16 outputs of a row share an aligned word
  int quads_ok;          // four neighbouring outputs are one aligned store
  int32_t* status;
  long long budget;
};

// ---- PTX ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(tm), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(tm), "r"(x), "r"(y), "r"(z), "r"(cluster_bar)
      : "memory");
}
__device__ __forceinline__ void tc_mma_mxf4_pair(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                 uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// in both CTAs of the pair, each from its own shared memory
__device__ __forceinline__ void tc_cp_scales_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
__device__ __forceinline__ void tc_mma_mxf4(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows x 16 bytes of shared memory -> four TMEM columns, the same in each of the four lane quadrants
__device__ __forceinline__ void tc_cp_scales(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
// 512 contiguous bytes as rows of 16 without swizzle: eight rows (128 bytes) a core matrix
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)1 << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// Instruction descriptor: both operands E2M1 and K-major, scales UE8M0; `id` selects which two of the
// four scale bytes of a column a multiply of 64 values uses (0 or 2).
__device__ __forceinline__ constexpr uint32_t mx_idesc(int m, int n, int id) {
  return ((uint32_t)id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) |
         ((uint32_t)id << 29);
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// ---- epilogue ------------------------------------------------------------------------------------------
__device__ __forceinline__ float finish(float v, float bias, bool has_bias, int relu) {
  if (has_bias) v = __fadd_rn(v, bias);
  return relu && v < 0.0f ? 0.0f : v;  // a NaN stays
}

// Four neighbouring features of a token, of which `valid` exist.
__device__ __forceinline__ void store4(float* p, const float (&v)[4], int valid, int whole) {
  if (whole && valid >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < valid) p[j] = v[j];
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4], int valid, int whole) {
  if (whole && valid >= 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(mx::bf16x2_bits(v[0], v[1]), mx::bf16x2_bits(v[2], v[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < valid) p[j] = __float2bfloat16_rn(v[j]);
  }
}

// COUNT tokens [t, t + COUNT) of this lane's feature.  A warp writes 32 neighbouring features of a token per
// store.  In bf16 two lanes trade halves, so that each writes one word of two features (of the first or
// second token of a pair): half as many store instructions.
template <int COUNT>
__device__ __forceinline__ void store_block(const Args& g, const float (&y)[COUNT], int t, int f, int lane, float*) {
  float* out = reinterpret_cast<float*>(g.out) + (long long)t * g.ldo + f;
#pragma unroll
  for (int j = 0; j < COUNT; ++j)
    if (f < g.N && t + j < g.M) out[j * g.ldo] = y[j];
}
template <int COUNT>
__device__ __forceinline__ void store_block(const Args& g, const float (&y)[COUNT], int t, int f, int lane, __nv_bfloat16*) {
  if (g.pairs_ok) {
    const int odd = lane & 1;
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(g.out) + (long long)(t + odd) * g.ldo + (f - odd);
#pragma unroll
    for (int j = 0; j < COUNT; j += 2) {
      const float theirs = __shfl_xor_sync(0xffffffffu, odd ? y[j] : y[j + 1], 1);
      const uint32_t w = odd ? mx::bf16x2_bits(theirs, y[j + 1]) : mx::bf16x2_bits(y[j], theirs);
      if (f < g.N && t + j + odd < g.M) *reinterpret_cast<uint32_t*>(out + j * g.ldo) = w;
    }
  } else {
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(g.out) + (long long)t * g.ldo + f;
#pragma unroll
    for (int j = 0; j < COUNT; ++j)
      if (f < g.N && t + j < g.M) out[j * g.ldo] = __float2bfloat16_rn(y[j]);
  }
}

// ---- one tile per CTA, K shared by a cluster --------------------------------------------------------------
//
// TN tokens x 128 features a CTA.  For few tokens the weight's stream from HBM is the bound: `split` CTAs of
// a cluster each take a contiguous run of K, so that a narrow layer still occupies the GPU, and two CTAs
// fit an SM, so that the copies of one run during the epilogue of the other.  The partial sums meet in
// shared memory: every CTA reads the others' through the cluster and adds them in rank order (the same
// result whatever the timing), each for its share of the outputs.  1 x 8192 x 28672: 21.3 us, 5.9 TB/s of weight;
// below that, launch, fill and exchange add about 4 us to the stream.  1000 x 4096 x 4096 to float32 (128 tokens a tile,
// one wave of 256 CTAs): 14.3 us with the tensor cores 29 % and L2 25 % busy; neither bounds it, the time is the fill of
// the ring, 16 stages, and an epilogue that little overlaps.
constexpr int kMaxSplit = 8;
constexpr int kThreads = 192;  // producer, multiply, four epilogue warps

template <int TN>
struct Cfg {
  static constexpr int kXBytes = TN * 128;
  static constexpr int kStageBytes = kWBytes + kXBytes + 2 * mx::kTileBytes;
  static constexpr int kStages = TN <= 64 ? 4 : 3;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 128;
  // TMEM: the accumulator, then a buffer of 8 + 8 scale columns per stage (a power of two is allocated)
  static constexpr int kTmemCols = TN + 16 * kStages <= 128 ? 128 : 256;
  static_assert(2 * kSmemBytes <= 226 * 1024, "two CTAs share an SM");
  static_assert(TN * kRows * 4 <= kStages * kStageBytes, "partial sums reuse the ring");
};

// With X other than void the activations are still float32 or bf16: the epilogue warps, idle until the product
// is done, encode them stage by stage into the places where TMA would have put codes and scales (every CTA of
// a layer repeats that for its part of K: a few KB of a few tokens).  One launch instead of two.
template <int TN, typename T, typename X = void>
__global__ void __launch_bounds__(kThreads, 2)
mx_tile_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
               const __grid_constant__ CUtensorMap tm_sw, const __grid_constant__ CUtensorMap tm_sx, const __grid_constant__ Args g) {
  using C = Cfg<TN>;
  extern __shared__ uint8_t smem_raw[];
  // the same offset in every CTA of a cluster (the partial sums are read across it)
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* tail = smem + C::kStages * C::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail);  // full[S], empty[S], done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 96);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 100);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * C::kStages, bar_done = bar_empty + 8 * C::kStages;

  const int tile = (int)blockIdx.x / g.split, rank = (int)blockIdx.x % g.split;
  const int t0 = tile % g.tiles_t * TN, f0 = tile / g.tiles_t * kRows;
  const int kb0 = (int)((long long)g.num_kb * rank / g.split), kb1 = (int)((long long)g.num_kb * (rank + 1) / g.split);
  const int n = kb1 - kb0;
  const uint32_t smem0 = smem_u32(smem);
  constexpr bool kFused = !std::is_same<X, void>::value;
  constexpr int kEncodeWarps = 4;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * C::kStages + 1; ++s) mbar_init(bar_full + 8 * s, kFused && s < C::kStages ? 1 + kEncodeWarps : 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_x) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Every warp waits here, the multiplying one too: a bounded wait on the first stage that began while the kernel
  // before this one still ran would run out on that kernel's time.  The weight too is fetched only now: an earlier
  // kernel may have encoded it, and the wait is what makes its writes visible here.  (48 x 8192 x 10240 15.3 us; 14.6
  // with its first stages in flight during the encode of the activations.)
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    int s = 0;
    uint32_t phase = 1;
    for (int i = 0; i < n; ++i) {
      if (!mbar_wait_warp(bar_empty + 8 * s, phase, abort_flag, g.budget)) break;
      if (elect_one()) {
        const uint32_t dst = smem0 + s * C::kStageBytes, bar = bar_full + 8 * s;
        mbar_expect_tx(bar, kFused ? kWBytes + mx::kTileBytes : C::kStageBytes);
        tma_load_2d(dst, &tm_w, (kb0 + i) * 128, f0, bar);
        tma_load_3d(dst + kWBytes + C::kXBytes, &tm_sw, 0, kb0 + i, f0 / mx::kTileRows, bar);
        if (!kFused) {
          tma_load_2d(dst + kWBytes, &tm_x, (kb0 + i) * 128, t0, bar);
          tma_load_3d(dst + kWBytes + C::kXBytes + mx::kTileBytes, &tm_sx, 0, kb0 + i, t0 / mx::kTileRows, bar);
        }
      }
      if (++s == C::kStages) s = 0, phase ^= 1;
    }
    __syncwarp();
  } else if (warp == 1) {
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      // a full stage also says that the multiplies which read its scale columns before are complete: its
      // copies were issued after them
      if (!mbar_wait_warp(bar_full + 8 * s, phase, abort_flag, g.budget)) { ok = false; break; }
      tc_fence_after();
      const uint32_t src = smem0 + s * C::kStageBytes;
      const uint64_t wdesc = make_smem_desc(src), xdesc = make_smem_desc(src + kWBytes);
      const uint64_t sdesc = scale_desc(src + kWBytes + C::kXBytes);
      // a column holds the scales of 32 rows: a tile of 64 tokens may begin in the middle of a scale tile
      const uint32_t sfw = tmem + TN + s * 16, sfx = sfw + 8, sft = sfx + (TN < mx::kTileRows ? t0 % mx::kTileRows / 32 : 0);
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tc_cp_scales(sfw + 4 * h, sdesc + h * 32);
          tc_cp_scales(sfx + 4 * h, sdesc + 64 + h * 32);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma_mxf4(tmem, wdesc + 2 * k, xdesc + 2 * k, mx_idesc(kRows, TN, 2 * (k & 1)), sfw + 4 * (k >> 1), sft + 4 * (k >> 1),
                      i | k ? 1u : 0u);
        tc_commit(bar_empty + 8 * s);
      }
      __syncwarp();
      if (++s == C::kStages) s = 0, phase ^= 1;
    }
    if (ok && elect_one()) tc_commit(bar_done);
    __syncwarp();
  }
  const bool epilogue = warp >= 2;
  const int quad = warp & 3;
  bool ok = true;
  if constexpr (kFused) {
    static_assert(TN == 16, "one scale tile, two swizzle atoms of tokens");
    if (epilogue) {
      const int tid = (int)threadIdx.x - 64;
      // a thread encodes chunk c of sixteen values of row r and of row r + 8
      const int c = tid & 15, r = tid >> 4;
      const bool high = g.M > 8;
      const X* x = reinterpret_cast<const X*>(g.x) + r * g.ldx + c * 16;
      // stages fetched ahead (one ahead left a load's latency in every stage: 16 x 8192 x 28672 40.2 us against 24.7)
      constexpr int kAhead = 8 / (int)sizeof(X);
      mx::Chunk<X> v[kAhead][2];
      auto fetch = [&](int i, mx::Chunk<X> (&w)[2]) {
        const int k = (kb0 + i) * kStageK;
        const bool in_k = i < n && k + c * 16 < g.K;
        if (in_k && r < g.M) w[0].load(x + k, g.x_wide);
        else w[0].clear();
        if (in_k && r + 8 < g.M) w[1].load(x + 8 * g.ldx + k, g.x_wide);
        else w[1].clear();
      };
      // row r of the swizzled tile: 16-byte piece p lies at piece p ^ (r % 8); rows 8.. are the next 1024 bytes
      const int code_at = kWBytes + r * 128 + (((c >> 1) ^ r) << 4) + (c & 1) * 8;
      const int scale_at = kWBytes + C::kXBytes + mx::kTileBytes + mx::tile_offset(r, c >> 1);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) fetch(j, v[j]);
      // rows past the last token stay zero
      constexpr int kPieces = (C::kXBytes + mx::kTileBytes) / 16;
      for (int i = tid; i < C::kStages * kPieces; i += 32 * kEncodeWarps) {
        const int s = i / kPieces, o = (i - s * kPieces) * 16;
        const int at = o < C::kXBytes ? kWBytes + o : kWBytes + mx::kTileBytes + o;  // codes, then (past the weight's) scales
        *reinterpret_cast<uint4*>(smem + s * C::kStageBytes + at) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      int s = 0;
      uint32_t phase = 1;
      for (int i0 = 0; i0 < n; i0 += kAhead) {
        bool more = true;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          more = more && i0 + j < n && mbar_wait_warp(bar_empty + 8 * s, phase, abort_flag, g.budget);
          if (!more) break;
          uint8_t* stage = smem + s * C::kStageBytes;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !high) break;
            const uint32_t byte = mx::block_byte<X>(v[j][h]);
            if (r + 8 * h < g.M) {
              *reinterpret_cast<uint2*>(stage + code_at + h * 1024) = mx::encode16<X>(v[j][h], byte);
              if (!(c & 1)) stage[scale_at + h * 8 * 16] = (uint8_t)byte;
            }
          }
          fetch(i0 + j + kAhead, v[j]);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads what these stores wrote
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_full + 8 * s);
          if (++s == C::kStages) s = 0, phase ^= 1;
        }
        if (!more) break;
      }
    }
  }
  if (epilogue) {
    ok = mbar_wait_warp(bar_done, 0, abort_flag, g.budget);
    tc_fence_after();
  }
  const int valid = min(TN, g.M - t0);
  const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
  if (g.split == 1) {
    if (epilogue && ok) {
      const int f = f0 + quad * 32 + lane;
      const float b = g.bias && f < g.N ? __ldcg(g.bias + f) : 0.0f;
#pragma unroll 1
      for (int c = 0; c < valid; c += 16) {
        uint32_t r[16];
        tc_ld16_sync(taddr + c, r);
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = finish(__uint_as_float(r[j]), b, g.bias != nullptr, g.relu);
        store_block<16>(g, y, t0 + c, f, lane, (T*)nullptr);
      }
    }
  } else {
    float* part = reinterpret_cast<float*>(smem);  // [token][feature]
    if (epilogue && ok) {
#pragma unroll 1
      for (int c = 0; c < valid; c += 16) {
        uint32_t r[16];
        tc_ld16_sync(taddr + c, r);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * kRows + quad * 32 + lane] = __uint_as_float(r[j]);
      }
    }
    cluster_sync_all();
    // four features a step; the loads from all CTAs are issued before the first addition
    const int total = valid * (kRows / 4);
    const int lo = (int)((long long)total * rank / g.split), hi = (int)((long long)total * (rank + 1) / g.split);
    const uint32_t base = smem_u32(part);
    for (int i = lo + (int)threadIdx.x; i < hi; i += kThreads) {
      float4 p[kMaxSplit];
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < g.split) p[r] = ld_cluster_f32x4(map_to_cta(base + 16 * i, r));
      const int f = f0 + i % (kRows / 4) * 4, t = t0 + i / (kRows / 4);
      float v[4] = {p[0].x, p[0].y, p[0].z, p[0].w};
#pragma unroll
      for (int r = 1; r < kMaxSplit; ++r)
        if (r < g.split) v[0] = __fadd_rn(v[0], p[r].x), v[1] = __fadd_rn(v[1], p[r].y), v[2] = __fadd_rn(v[2], p[r].z), v[3] = __fadd_rn(v[3], p[r].w);
      if (*abort_flag != 0) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = finish(v[j], g.bias && f + j < g.N ? __ldcg(g.bias + f + j) : 0.0f, g.bias != nullptr, g.relu);
      store4(reinterpret_cast<T*>(g.out) + (long long)t * g.ldo + f, v, g.N - f, g.quads_ok);
    }
    cluster_sync_all();  // nobody's partial sums go away while they are read
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    for (int i = 0; i < 50; ++i) __nanosleep(20000);  // copies and multiplies in flight land first
    if (threadIdx.x == 0 && g.status) atomicExch(g.status, (int)LQ_ERR_TIMEOUT);
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
  }
}

// ---- CTA pairs, persistent ---------------------------------------------------------------------------------
//
// 256 features x 256 tokens per pair of CTAs (cta_group::2): each CTA stages its 128 weight rows and half of
// the tokens, so a stage of 256 values of K moves 32 KB of codes into each SM for 512 cycles of multiplies --
// half of what a lone 128 x 128 tile needs, whose operand traffic from L2 is its bound.  TMEM holds two
// accumulators of 256 columns and four buffers of 24 scale columns only because the accumulators overlap:
// columns 0..255 and 160..415, scales from 416.  The epilogue reads the 96 shared columns into registers
// first and says so on a barrier of their own; the next tile's multiplies then run while it works on the
// rest.  (Two scale buffers leave 48 shared columns but make every stage wait for the multiplies two stages
// back to be reported: 350 us against 339.)  4096 x 8192 x 28672 in bf16: 339 us, 5.67 PFLOP/s; repeated for
// seconds 392 us at 1.5 GHz, where the power cap is the bound.
constexpr int kPairTokens = 256;
constexpr int kPairStages = 6;
constexpr int kPairXBytes = kPairTokens / 2 * 128;
constexpr int kPairStageBytes = kWBytes + kPairXBytes + 3 * mx::kTileBytes;
constexpr int kPairSmemBytes = kPairStages * kPairStageBytes + 1024 + 256;
constexpr int kPairEpilogueWarps = 8;
constexpr int kPairThreads = 64 + 32 * kPairEpilogueWarps;
constexpr int kPairScaleBufs = 4;
constexpr int kScaleCols = 512 - 24 * kPairScaleBufs;
constexpr int kAccStep = kScaleCols - kPairTokens, kAccShared = kPairTokens - kAccStep;  // columns between the accumulators, and shared
static_assert(kAccStep % 32 == 0 && kAccShared == 96, "the epilogue's two halves take whole blocks of 16 columns");
static_assert(kPairSmemBytes <= 227 * 1024, "shared memory");

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
mx_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
               const __grid_constant__ CUtensorMap tm_sw, const __grid_constant__ CUtensorMap tm_sx, const __grid_constant__ Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* tail = smem + kPairStages * kPairStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail);  // full[S], empty[S], tfull[2], tempty[2], shared columns
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 192);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 196);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * kPairStages;
  const uint32_t bar_tfull = bar_empty + 8 * kPairStages, bar_tempty = bar_tfull + 16, bar_shared = bar_tempty + 16;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int worker = (int)(blockIdx.x >> 1), workers = (int)(gridDim.x >> 1);
  const int total = g.tiles_t * g.tiles_f;
  const uint32_t smem0 = smem_u32(smem);

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * kPairStages + 2; ++s) mbar_init(bar_full + 8 * s, 1);
    for (int s = 0; s < 3; ++s) mbar_init(bar_tempty + 8 * s, 2 * kPairEpilogueWarps);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_x) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before anyone signals them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  // The issuing warps run their loops with all lanes and elect one for each instruction, with stage and
  // phase kept as counters: descriptors and loop state then live in uniform registers.  (One lane in a
  // branch of its own, with the stage taken modulo the ring, cost 820 cycles of issue per stage of 512
  // cycles of multiplies.)
  if (warp == 0) {
    int s = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int tile = worker; ok && tile < total; tile += workers) {
      const int t0 = tile % g.tiles_t * kPairTokens, f0 = tile / g.tiles_t * 2 * kRows + (int)rank * kRows;
      const int x0 = t0 + (int)rank * (kPairTokens / 2), fr = f0 / mx::kTileRows, tr = t0 / mx::kTileRows;
      for (int kb = 0; kb < g.num_kb; ++kb) {
        if (!mbar_wait_warp(bar_empty + 8 * s, phase, abort_flag, g.budget)) { ok = false; break; }
        const uint32_t dst = smem0 + s * kPairStageBytes;
        if (elect_one()) {
          const uint32_t full = map_to_cta(bar_full + 8 * s, 0);  // both CTAs' bytes count on the leader's barrier
          if (leader) mbar_expect_tx(bar_full + 8 * s, 2 * kPairStageBytes);
          tma_load_2d_pair(dst, &tm_w, kb * 128, f0, full);
          tma_load_2d_pair(dst + kWBytes, &tm_x, kb * 128, x0, full);
          tma_load_3d_pair(dst + kWBytes + kPairXBytes, &tm_sw, 0, kb, fr, full);
          tma_load_3d_pair(dst + kWBytes + kPairXBytes + mx::kTileBytes, &tm_sx, 0, kb, tr, full);
        }
        if (++s == kPairStages) s = 0, phase ^= 1;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader) {
      int s = 0, q = 0, buf = 0, done = 0;           // stage; tiles; scale buffer; stages issued (up to their number)
      int sb = kPairStages - kPairScaleBufs;         // the stage that used this scale buffer before
      uint32_t phase = 0, phase_b = 1;
      bool ok = true;
      for (int tile = worker; ok && tile < total; tile += workers, ++q) {
        const int acc = q & 1;
        // this accumulator is empty, and so are the columns it shares with the one before
        if (q >= 2 && !mbar_wait_warp(bar_tempty + 8 * acc, ((q >> 1) - 1) & 1, abort_flag, g.budget)) break;
        if (q >= 1 && !mbar_wait_warp(bar_shared, (q - 1) & 1, abort_flag, g.budget)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * kAccStep;
        for (int kb = 0; kb < g.num_kb; ++kb) {
          // the multiplies that read this buffer of scale columns before are complete
          if (done == kPairScaleBufs ? !mbar_wait_warp(bar_empty + 8 * sb, phase_b, abort_flag, g.budget) : (++done, false)) { ok = false; break; }
          if (!mbar_wait_warp(bar_full + 8 * s, phase, abort_flag, g.budget)) { ok = false; break; }
          tc_fence_after();
          const uint32_t src = smem0 + s * kPairStageBytes;
          const uint64_t wdesc = make_smem_desc(src), xdesc = make_smem_desc(src + kWBytes);
          const uint64_t sdesc = scale_desc(src + kWBytes + kPairXBytes);
          const uint32_t sfw = tmem + kScaleCols + buf * 24, sfx = sfw + 8;
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              tc_cp_scales_pair(sfw + 4 * h, sdesc + h * 32);
              tc_cp_scales_pair(sfx + 8 * h, sdesc + 64 + h * 32);
              tc_cp_scales_pair(sfx + 8 * h + 4, sdesc + 128 + h * 32);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma_mxf4_pair(d, wdesc + 2 * k, xdesc + 2 * k, mx_idesc(2 * kRows, kPairTokens, 2 * (k & 1)), sfw + 4 * (k >> 1),
                               sfx + 8 * (k >> 1), kb | k ? 1u : 0u);
            tc_commit_pair(bar_empty + 8 * s);
          }
          __syncwarp();
          if (++buf == kPairScaleBufs) buf = 0;
          if (++s == kPairStages) s = 0, phase ^= 1;
          if (++sb == kPairStages) sb = 0, phase_b ^= 1;
        }
        if (!ok) break;
        if (elect_one()) tc_commit_pair(bar_tfull + 8 * acc);
        __syncwarp();
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const uint32_t tempty = map_to_cta(bar_tempty, 0), shared_cols = map_to_cta(bar_shared, 0);
    int q = 0;
    for (int tile = worker; tile < total; tile += workers, ++q) {
      const int t0 = tile % g.tiles_t * kPairTokens;
      const int f = tile / g.tiles_t * 2 * kRows + (int)rank * kRows + quad * 32 + lane;
      const int acc = q & 1;
      const float b = g.bias && f < g.N ? __ldcg(g.bias + f) : 0.0f;
      if (!mbar_wait_warp(bar_tfull + 8 * acc, (q >> 1) & 1, abort_flag, g.budget)) break;
      tc_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + acc * kAccStep;
      auto put = [&](const uint32_t (&r)[16], int c) {
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = finish(__uint_as_float(r[j]), b, g.bias != nullptr, g.relu);
        if (t0 + c < g.M) store_block<16>(g, y, t0 + c, f, lane, (T*)nullptr);
      };
      // the shared columns of TMEM: the last tokens of the first accumulator, the first of the second
      const int c_shared = (acc ? 0 : kAccStep) + half * (kAccShared / 2), c_rest = (acc ? kAccShared : 0) + half * (kAccStep / 2);
      uint32_t r[3][16];
#pragma unroll
      for (int i = 0; i < 3; ++i) tc_ld16(taddr + c_shared + 16 * i, r[i]);
#pragma unroll
      for (int i = 0; i < 3; ++i) tc_wait_ld_dep16(r[i]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(shared_cols);
#pragma unroll
      for (int i = 0; i < 3; ++i) put(r[i], c_shared + 16 * i);
      // the rest, one block of 16 columns read ahead
      tc_ld16(taddr + c_rest, r[0]);
#pragma unroll
      for (int i = 0; i < kAccStep / 32; ++i) {
        tc_wait_ld_dep16(r[i & 1]);
        if (i + 1 < kAccStep / 32) tc_ld16(taddr + c_rest + 16 * (i + 1), r[(i + 1) & 1]);
        put(r[i & 1], c_rest + 16 * i);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty + 8 * acc);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    for (int i = 0; i < 50; ++i) __nanosleep(20000);  // copies and multiplies in flight land first
    if (threadIdx.x == 0 && g.status) atomicExch(g.status, (int)LQ_ERR_TIMEOUT);
  }
  cluster_sync_all();  // the peer may still signal this CTA's barriers or read its stages
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---- host --------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn get_encode() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = (EncodeFn)p;
  });
  return fn;
}
// codes: (rows, K / 2) bytes, boxes of 128 bytes x box_rows, rows and bytes past the end read as zeros
int code_map(CUtensorMap* tm, const void* base, size_t rows, size_t K, int box_rows) {
  if (!get_encode()) return fail(LQ_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[2] = {K / 2, rows}, strides[1] = {K / 2};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUresult r = get_encode()(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, ones,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? LQ_OK : fail(LQ_ERR_CUDA, "lq_mx_matmul: tensor map of the codes failed: " + std::to_string((int)r));
}
// scale tiles: (row tiles, column tiles, 256 words), boxes of one column tile x box_tiles row tiles
int scale_map(CUtensorMap* tm, const void* base, size_t rows, size_t K, int box_tiles) {
  if (!get_encode()) return fail(LQ_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t ct = (K + kStageK - 1) / kStageK, rt = (rows + mx::kTileRows - 1) / mx::kTileRows;
  const cuuint64_t dims[3] = {256, ct, rt}, strides[2] = {mx::kTileBytes, ct * mx::kTileBytes};
  const cuuint32_t box[3] = {256, 1, (cuuint32_t)box_tiles}, ones[3] = {1, 1, 1};
  const CUresult r = get_encode()(tm, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box, ones,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? LQ_OK : fail(LQ_ERR_CUDA, "lq_mx_matmul: tensor map of the scales failed: " + std::to_string((int)r));
}

struct Operands {
  const uint8_t *x, *sx, *w, *sw;
  size_t M, N, K;
};
// Up to this many rows lq_mx_linear encodes them inside the product.  More take longer to encode in every CTA than
// in a kernel of their own: 32 x 8192 x 8192 15.2 us against 12.7, 48 x 8192 x 10240 23.5 against 14.6; at 16 x 8192 x
// 28672 24.2 against 24.3, 8 x 8192 x 8192 9.2 against 11.4, and one launch of the host's time less.
constexpr size_t kFusedTokens = 16;

template <int TN, typename T, typename X = void>
int launch_tile(const Operands& o, Args g, cudaStream_t st) {
  static PerDeviceOnce once;
  using C = Cfg<TN>;
  auto kernel = mx_tile_kernel<TN, T, X>;
  const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes); });
  if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(max dynamic smem)");
  g.tiles_t = (g.M + TN - 1) / TN, g.tiles_f = (g.N + kRows - 1) / kRows;
  const long long tiles = (long long)g.tiles_t * g.tiles_f;
  const long long room = 2ll * sm_count();
  g.split = 1;
  // Share K while all CTAs fit and each keeps enough stages to pay for the exchange of partial sums (which
  // grows with the tokens).  Measured, split 1 / 2 / 4, us: 256 x 4096 x 4096 (16 stages, 64 tokens a tile)
  // 8.2 / 9.3 / 9.3; 48 x 8192 x 10240 (32 stages) 14.4 / 13.7 / 12.0; 1 x 8192 x 8192 12.0 / 9.8 / 9.0;
  // 1 x 1024 x 8192 (4 stages) 2.9 / 3.3 / 4.2.
  const int least = TN <= 32 ? 4 : 10;
  while (g.split < kMaxSplit && g.num_kb >= least * (g.split + 1) && tiles * (g.split + 1) <= room) ++g.split;
  if (tiles * g.split > 0x7fffffffll) return fail(LQ_ERR_SHAPE, "lq_mx_matmul: too many tiles for one launch");
  CUtensorMap tw, tx, tsw, tsx;
  if (int rc = code_map(&tw, o.w, o.N, o.K, kRows)) return rc;
  if (int rc = scale_map(&tsw, o.sw, o.N, o.K, 1)) return rc;
  if (std::is_same<X, void>::value) {
    if (int rc = code_map(&tx, o.x, o.M, o.K, TN)) return rc;
    if (int rc = scale_map(&tsx, o.sx, o.M, o.K, 1)) return rc;
  } else {
    tx = tw, tsx = tsw;  // not used
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * g.split)), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = C::kSmemBytes, cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)g.split, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, tw, tx, tsw, tsx, g), "lq_mx_matmul launch");
}

template <typename T>
int launch_pair(const Operands& o, Args g, cudaStream_t st) {
  static PerDeviceOnce once;
  static int max_clusters[kMaxDevices] = {};
  auto kernel = mx_pair_kernel<T>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * sm_count()), cfg.blockDim = dim3(kPairThreads), cfg.dynamicSmemBytes = kPairSmemBytes, cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  const int dev = current_device();
  const cudaError_t e = once.run([&]() -> cudaError_t {
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmemBytes);
    int mc = 0;
    if (err == cudaSuccess) err = cudaOccupancyMaxActiveClusters(&mc, kernel, &cfg);
    max_clusters[dev] = mc > 0 ? mc : 1;
    return err;
  });
  if (e != cudaSuccess) return check_cuda(e, "mx_pair_kernel setup");
  g.split = 1;
  g.tiles_t = (g.M + kPairTokens - 1) / kPairTokens, g.tiles_f = (g.N + 2 * kRows - 1) / (2 * kRows);
  const long long tiles = (long long)g.tiles_t * g.tiles_f;
  if (tiles > 0x3fffffffll) return fail(LQ_ERR_SHAPE, "lq_mx_matmul: too many tiles for one launch");
  CUtensorMap tw, tx, tsw, tsx;
  if (int rc = code_map(&tw, o.w, o.N, o.K, kRows)) return rc;
  if (int rc = code_map(&tx, o.x, o.M, o.K, kPairTokens / 2)) return rc;
  if (int rc = scale_map(&tsw, o.sw, o.N, o.K, 1)) return rc;
  if (int rc = scale_map(&tsx, o.sx, o.M, o.K, 2)) return rc;
  cfg.gridDim = dim3(2 * (unsigned)(tiles < max_clusters[dev] ? tiles : max_clusters[dev]));
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, tw, tx, tsw, tsx, g), "lq_mx_matmul (pair) launch");
}

template <typename T>
int launch(const Operands& o, const Args& g, cudaStream_t st) {
  // Up to 64 tokens: the narrowest tile that holds them all (the weight's stream is the bound, the rest of
  // a wider tile would be multiplied for nothing).  More: the narrowest tile whose count fits the GPU at
  // once, two CTAs an SM, and pairs beyond that.  Measured, tile of 64 / 128 tokens / pair, us: 256 x 4096 x
  // 4096 8.2 / 10.1 / 13.7; 1000 x 4096 x 4096 17.9 / 12.2 / 14.4; 2048 x 4096 x 4096 34.0 / 24.4 / 22.5.
  if (o.M <= 16) return launch_tile<16, T>(o, g, st);
  if (o.M <= 32) return launch_tile<32, T>(o, g, st);
  const long long rows = (long long)((o.N + kRows - 1) / kRows), room = 2ll * sm_count();
  if (o.M <= 64 || (long long)((o.M + 63) / 64) * rows <= room) return launch_tile<64, T>(o, g, st);
  if ((long long)((o.M + 127) / 128) * rows <= room) return launch_tile<128, T>(o, g, st);
  return launch_pair<T>(o, g, st);
}

// What every form of the product asks of its weight, result and extents; fills the common arguments.
int prepare(const char* who, Args* g, size_t M, const uint8_t* w_codes, const uint8_t* w_scales, size_t N, size_t K, const float* bias,
            int relu, void* out, int out_dtype, size_t ldo, int32_t* status) {
  const std::string w(who);
  if (!w_codes || !w_scales || !out) return fail(LQ_ERR_DEVICE, w + ": null pointer");
  if (out_dtype != LQ_F32 && out_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, w + ": out must be f32|bf16");
  if (K == 0 || K % mx::kBlock != 0) return fail(LQ_ERR_SHAPE, w + ": K must be a multiple of 32");
  if (M >= ((size_t)1 << 30) || N >= ((size_t)1 << 30) || K >= ((size_t)1 << 30)) return fail(LQ_ERR_SHAPE, w + ": extents must be below 2^30");
  if (ldo < N) return fail(LQ_ERR_SHAPE, w + ": output row stride shorter than a row");
  const size_t esz = out_dtype == LQ_F32 ? 4 : 2;
  if (!aligned16(w_codes) || !aligned16(w_scales) || reinterpret_cast<uintptr_t>(out) % esz != 0)
    return fail(LQ_ERR_ALIGNMENT, w + ": codes and scales must be 16-byte aligned, out to its type");
  memset(g, 0, sizeof(*g));
  g->M = (int)M, g->N = (int)N, g->K = (int)K, g->num_kb = (int)((K + kStageK - 1) / kStageK);
  g->bias = bias, g->relu = relu, g->out = out, g->ldo = (long long)ldo, g->status = status, g->budget = kWaitBudgetCycles;
  g->pairs_ok = out_dtype == LQ_BF16 && reinterpret_cast<uintptr_t>(out) % 4 == 0 && ldo % 2 == 0 && N % 2 == 0;
  g->quads_ok = reinterpret_cast<uintptr_t>(out) % (4 * esz) == 0 && ldo % 4 == 0;
  return LQ_OK;
}

template <typename T>
int launch_fused(const Operands& o, const Args& g, int in_dtype, cudaStream_t st) {
  return in_dtype == LQ_F32 ? launch_tile<16, T, float>(o, g, st) : launch_tile<16, T, __nv_bfloat16>(o, g, st);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_mx_linear_workspace_bytes(size_t M, size_t K) {
  return M <= kFusedTokens ? 0 : (M * (K / 2) + 1023) / 1024 * 1024 + lq_mx_scale_bytes(M, K);
}

extern "C" int lq_mx_matmul(const uint8_t* a_codes, const uint8_t* a_scales, size_t M, const uint8_t* w_codes,
                            const uint8_t* w_scales, size_t N, size_t K, const float* bias, int relu, void* out,
                            int out_dtype, size_t ldo, int32_t* status, void* stream) {
  if (M == 0 || N == 0) return LQ_OK;
  if (!a_codes || !a_scales) return fail(LQ_ERR_DEVICE, "lq_mx_matmul: null pointer");
  Args g;
  if (int rc = prepare("lq_mx_matmul", &g, M, w_codes, w_scales, N, K, bias, relu, out, out_dtype, ldo, status)) return rc;
  if (!aligned16(a_codes) || !aligned16(a_scales)) return fail(LQ_ERR_ALIGNMENT, "lq_mx_matmul: codes and scales must be 16-byte aligned");
  const Operands o = {a_codes, a_scales, w_codes, w_scales, M, N, K};
  cudaStream_t st = (cudaStream_t)stream;
  return out_dtype == LQ_F32 ? launch<float>(o, g, st) : launch<__nv_bfloat16>(o, g, st);
}

extern "C" int lq_mx_linear(const void* x, int in_dtype, size_t M, size_t ldx, const uint8_t* w_codes, const uint8_t* w_scales,
                            size_t N, size_t K, const float* bias, int relu, void* out, int out_dtype, size_t ldo,
                            uint8_t* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  if (M == 0 || N == 0) return LQ_OK;
  Args g;
  if (int rc = prepare("lq_mx_linear", &g, M, w_codes, w_scales, N, K, bias, relu, out, out_dtype, ldo, status)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  Operands o = {nullptr, nullptr, w_codes, w_scales, M, N, K};
  if (M <= kFusedTokens) {
    if (!x) return fail(LQ_ERR_DEVICE, "lq_mx_linear: null pointer");
    if (in_dtype != LQ_F32 && in_dtype != LQ_BF16) return fail(LQ_ERR_DTYPE, "lq_mx_linear: x must be f32|bf16");
    const size_t esz = in_dtype == LQ_F32 ? 4 : 2;
    if (ldx < K) return fail(LQ_ERR_SHAPE, "lq_mx_linear: row stride shorter than a row");
    if (!aligned16(x) || (ldx * esz) % 16 != 0) return fail(LQ_ERR_ALIGNMENT, "lq_mx_linear: rows of x must be 16-byte aligned");
    g.x = x, g.ldx = (long long)ldx, g.x_wide = reinterpret_cast<uintptr_t>(x) % 32 == 0 && (ldx * esz) % 32 == 0;
    return out_dtype == LQ_F32 ? launch_fused<float>(o, g, in_dtype, st) : launch_fused<__nv_bfloat16>(o, g, in_dtype, st);
  }
  if (!workspace) return fail(LQ_ERR_DEVICE, "lq_mx_linear: null workspace");
  if (!aligned16(workspace)) return fail(LQ_ERR_ALIGNMENT, "lq_mx_linear: the workspace must be 16-byte aligned");
  if (workspace_bytes < lq_mx_linear_workspace_bytes(M, K)) return fail(LQ_ERR_WORKSPACE, "lq_mx_linear: workspace too small");
  uint8_t* a_scales = workspace + (M * (K / 2) + 1023) / 1024 * 1024;
  if (int rc = lq_mx_quantize(x, in_dtype, M, K, ldx, workspace, a_scales, stream)) return rc;
  o.x = workspace, o.sx = a_scales;
  return out_dtype == LQ_F32 ? launch<float>(o, g, st) : launch<__nv_bfloat16>(o, g, st);
}
