// Attention over the 8-bit cache (kvcache.cuh):
//
//   out[b, i, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(q[b, i, h] . k_j / sqrt(128)),   j < seen(b, i)
//   seen = lengths[b], or lengths[b] - nq + i + 1 (causal: the queries are the cache's last nq rows);
//   a row that sees nothing is zeros.  heads / kv_heads query heads share a key head.
//
// Numbers.  k = K 2^ek and v = V 2^ev with K, V in e4m3 and one ek, ev a block
// of 64 keys and head.  e4m3 values are exact in f16, so both products run on
// f16 operands with fp32 sums:
//   q is divided by a power of two of its row (largest magnitude in [1, 2)) and
//   taken to f16: exact down to 2^-14 of the row's largest value, off by at most
//   2^-25 of it below;
//   x_j = (Q . K_j) 2^eq 2^ek log2(e) / sqrt(128) + ev, and the running maximum m is
//   taken over x, so P_j = 2^(x_j - m + 5) carries V's scale; m follows the maximum
//   only when that has grown by more than 2^8, so P_j <= 2^13 never overflows f16
//   (full precision down to 2^-19 of the largest, steps of 2^-29 of it below);
//   P V adds up to the numerator, sum_j P_j 2^-ev (fp32, before P is rounded) to the
//   denominator, and 2^(5 - m) cancels.
//   The denominator counts every key, whatever its values' scale: of 64 zeros (ev -60) beside values of 1e23 too,
//   whose x differ by more than fp32's exponents reach.  So where a row's x lie 2^100 and more below m throughout a
//   unit or step, P is taken against their own maximum, only for the sum (f16 has zeros for them anyway), which then
//   gets the difference; and a change of m takes the denominator along as two factors (folded).  The sum itself stays
//   between 2^(5 - ev) of the largest x's ev and 2^(13 - ev) of the smallest, so within 2^-121 .. 2^73 a key.
//
// Masked keys have x = -inf.  Rows past a sequence's length are whatever the
// block held before; they, and NaN in a value that only some rows of a tile see,
// must not reach the product (0 x NaN): in units where a row sees less than the
// whole, V is cleaned, and the lowest key with a NaN in each dim is kept so that
// the rows that do see it get it back.
#pragma once

#include <cfloat>

#include "kvcache.cuh"
#include "ptx.cuh"

namespace wamffn {

struct KvAttnParams {
  CacheView c;
  const __nv_bfloat16* q;
  long long q_row, q_batch;  // strides, elements
  __nv_bfloat16* out;        // [batch, nq, heads 128]
  int nq, heads, group, causal, split;
  int tile_rows;             // many rows: packed rows of a CTA, 256 or 128
  int parts;                 // of the keys, each with a cluster of its own
  float* part_o;             // parts > 1: unnormalised rows [parts, batch, nq, heads, 128]
  float2* part_ml;           // and their (maximum, normaliser) [parts, batch, nq, heads]
  float scale_log2;          // log2(e) / sqrt(128)
};

// Four dims of a row: the result, or with parts this part's share of it.
__device__ __forceinline__ void kv_emit(const KvAttnParams& p, int part, int b, int token, int head, int d,
                                        const float4& v, float top, float sum) {
  const size_t row = (size_t(b) * p.nq + token) * p.heads + head;
  if (p.parts == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // nothing seen: zeros
    *reinterpret_cast<uint2*>(p.out + row * kCacheDim + d) =
        make_uint2(bf2_pack(v.x * inv, v.y * inv), bf2_pack(v.z * inv, v.w * inv));
  } else {
    const size_t at = size_t(part) * p.c.batch * p.nq * p.heads + row;
    *reinterpret_cast<float4*>(p.part_o + at * kCacheDim + d) = v;
    if (d == 0) p.part_ml[at] = make_float2(top, sum);
  }
}

// x times h^2, where h^2 may be too small for a float and x too large.
__device__ __forceinline__ float folded(float x, float h) { return x * h * h; }

// The parts' shares of a row in their order; a warp a row.
constexpr int kMergeThreads = 256;
__global__ void __launch_bounds__(kMergeThreads) kv_merge_kernel(const KvAttnParams p, long long rows) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const long long row = (long long)blockIdx.x * (kMergeThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int d = (threadIdx.x & 31) * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float top = -INFINITY, sum = 0.f;
  for (int k = 0; k < p.parts; ++k) {
    const float2 ml = p.part_ml[k * rows + row];
    const float4 u = *reinterpret_cast<const float4*>(p.part_o + (k * rows + row) * kCacheDim + d);
    const float next = fmaxf(top, ml.x), safe = next == -INFINITY ? 0.f : next;
    const float ho = ex2_approx(0.5f * (top - safe)), hn = ex2_approx(0.5f * (ml.x - safe));
    const float fo = ho * ho, fn = hn * hn;
    v.x = v.x * fo + u.x * fn, v.y = v.y * fo + u.y * fn;
    v.z = v.z * fo + u.z * fn, v.w = v.w * fo + u.w * fn;
    sum = folded(sum, ho) + folded(ml.y, hn);
    top = next;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(p.out + row * kCacheDim + d) =
      make_uint2(bf2_pack(v.x * inv, v.y * inv), bf2_pack(v.z * inv, v.w * inv));
}

constexpr float kPBias = 5.f, kLag = 8.f;  // P <= 2^(5 + 8)
constexpr float kDeep = 100.f;             // x below m by this: P - 31 binades of it are still normal numbers

__device__ __forceinline__ uint32_t f16x2_pack(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transposes an 8 x 8 matrix of f16 held two a lane (row lane / 4, columns 2 (lane % 4) ..).
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// Power of two of a query row from its largest magnitude (fp32 bits): the row is
// multiplied by 2^-eq; infinities and NaN pass through.  At least -60, so that
// 2^eq 2^ek / sqrt(128) stays a normal number (-inf times it is -inf).
__device__ __forceinline__ int query_exp(float top) {
  return max(-60, min(126, ((__float_as_int(top) >> 23) & 255) - 127));
}

__device__ __forceinline__ int cache_length(const CacheView& c, int b) {
  return int(max(0ll, min((long long)c.lengths[b], (long long)c.width * kCacheBlock)));
}
// Keys that query token i sees.
__device__ __forceinline__ int keys_seen(int length, int nq, int i, int causal) {
  return causal ? max(0, length - nq + i + 1) : length;
}

// Whether one of 16 e4m3 values is NaN (a byte is 0x7f but for its sign).
__device__ __forceinline__ bool any_nan(const uint4& u) {
  const uint32_t x = (u.x & 0x7f7f7f7fu) + 0x01010101u, y = (u.y & 0x7f7f7f7fu) + 0x01010101u,
                 z = (u.z & 0x7f7f7f7fu) + 0x01010101u, w = (u.w & 0x7f7f7f7fu) + 0x01010101u;
  return ((x | y | z | w) & 0x80808080u) != 0;
}
// 16 e4m3 values, dims [dim, dim + 16) of key `key`, without their NaN, whose key is noted (rare).
__device__ __noinline__ uint4 drop_nan(uint4 u, int key, int dim, int* nan_key, int* nan_any) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const uint32_t at = 8 * (i & 3), word = i < 8 ? (i < 4 ? w[0] : w[1]) : (i < 12 ? w[2] : w[3]);
    if (((word >> at) & 0x7fu) == 0x7fu) {
      atomicMin(&nan_key[dim + i], key);
      *nan_any = 1;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] &= ~__vcmpeq4(w[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// What the product may see of 16 values: nothing past the sequence; no NaN in a
// unit that some rows see less of than others (`scan`).
__device__ __forceinline__ uint4 clean_chunk(uint4 u, int key, int length, bool scan, int dim, int* nan_key,
                                             int* nan_any) {
  if (key >= length) return make_uint4(0, 0, 0, 0);
  if (scan && any_nan(u)) u = drop_nan(u, key, dim, nan_key, nan_any);
  return u;
}

// ---------------------------------------------------------------------------
// Few rows (a decode step: at most 16 packed rows, query token x head of the
// group): matrix products by mma.sync from registers.
//
// Bound: HBM (the cache is read once, 256 bytes a key and head).  A unit is 32
// keys of one head, 4 KB of K and of V, loaded by TMA with the 128-byte swizzle
// into a ring; the fragments are converted in registers (a lane takes 16
// neighbouring dims of K, which the product's order of k allows, and the same
// 16 dims of four rows of V), so nothing is written back to shared memory.
// Up to 8 rows stand as the products' columns (S^T = K Q^T, O^T = V^T P^T: half the
// instructions of rows as rows, 32 instead of 64 accumulators), up to 16 as their rows.
// On a B200, 16 x 1 token of 32 heads over up to 16381 rows of 8 key heads: 67 us, 80 %
// of the measured copy bandwidth (80 us with rows as rows; 94 us with two CTAs an
// SM; 88 % where all sequences are equally long, two thirds with 12 packed rows, as rows); one
// token over 577 rows of 24 heads 6 us, latency: length and block ids, then the rows, then
// two reductions.
// Four warps with rings and units of their own, three CTAs an SM (a unit is one
// long chain of dependent steps, and warps hide each other's);
// a cluster of `split` CTAs shares the keys of a part, and the partial results meet
// through distributed shared memory.
// ---------------------------------------------------------------------------
constexpr int kFewRows = 16;  // packed rows of a key head at most; beyond, kvattend_many.cuh
constexpr int kUnitKeys = 32;
constexpr int kUnitBytes = kUnitKeys * kCacheDim;  // of K, and of V
constexpr int kFewWarps = 4;
constexpr int kFewStages = 2;                      // of a warp's ring
constexpr int kFewPitch = kCacheDim + 4;           // floats between rows of a partial result
constexpr int kFewRing = kFewStages * 2 * kUnitBytes;  // of a warp
constexpr int kFewSmem = kFewWarps * kFewRing + 1024;
static_assert(kFewRows * kFewPitch * 4 <= kFewRing, "a partial result fits its warp's ring");

template <bool kNarrow>
__global__ void __launch_bounds__(kFewWarps * 32, 3)
    kv_attend_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                         const KvAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[kFewWarps][kFewStages];
  __shared__ __align__(16) float2 part_ml[kFewWarps][kFewRows];  // (maximum, normaliser) of a warp's rows
  __shared__ __align__(16) float2 cta_ml[kFewRows];
  __shared__ int nan_key[kCacheDim];
  __shared__ int nan_any;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = p.split, part = int(blockIdx.x) / split, rank = int(blockIdx.x) - part * split;
  const int kh = blockIdx.y, b = blockIdx.z;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kFewWarps * kFewStages; ++s) mbar_init(smem_addr(&full[0][s]), 1);
    nan_any = 0;
    abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  nan_key[threadIdx.x] = 0x7fffffff;  // kFewWarps * 32 == kCacheDim
  __syncthreads();
  pdl_wait_prior();
  pdl_launch_dependents();

  const CacheView& c = p.c;
  const int worker = int(blockIdx.x) * kFewWarps + warp, workers = int(gridDim.x) * kFewWarps;
  uint8_t* my_ring = ring + warp * kFewRing;
  uint64_t* my_full = full[warp];
  // Block ids and scales of 32 of this warp's units (worker + i * workers) at a time, one a lane.  The scales are
  // taken apart where they are used: no load waits for them.
  struct Info {
    int id;         // tile row of the unit in the pool's tensor map; -1: bad block id
    float ks, vs;
  };
  auto table_at = [&](int i) {  // any entry of the table, whatever the length
    const int at = (worker + i * workers) >> 1;
    return at < c.width ? c.table[b * c.table_stride + at] : -1;
  };
  auto info_of = [&](int i, int id) {
    Info f{-1, 1.f, 1.f};
    if (id >= 0 && id < c.blocks) {
      const size_t at = size_t(id) * c.kv_heads + kh;
      f.id = int(at * kCacheBlock) + ((worker + i * workers) & 1) * kUnitKeys;
      f.ks = c.key_scales[at];
      f.vs = c.value_scales[at];
    }
    return f;
  };
  const int first_id = table_at(lane);  // on its way together with the length
  const int length = cache_length(c, b);
  const int rows = p.nq * p.group;
  const int least = keys_seen(length, p.nq, 0, p.causal), most = keys_seen(length, p.nq, p.nq - 1, p.causal);
  const int units = (most + kUnitKeys - 1) / kUnitKeys;
  const int mine = units > worker ? (units - worker + workers - 1) / workers : 0;

  const uint64_t policy = l2_policy_evict_first();
  Info ahead = info_of(lane, first_id);  // of the units being loaded
  int ahead_chunk = 0, issued = 0;
  auto issue = [&](int i) {  // unit i into stage i % kFewStages
    if ((i >> 5) != ahead_chunk) {
      ahead_chunk = i >> 5;
      ahead = info_of(ahead_chunk * 32 + lane, table_at(ahead_chunk * 32 + lane));
    }
    const int id = __shfl_sync(0xffffffffu, ahead.id, i & 31);
    if (lane == 0) {
      const int s = i % kFewStages;
      const uint32_t bar = smem_addr(&my_full[s]), dst = smem_addr(my_ring + s * 2 * kUnitBytes);
      if (id >= 0) {
        mbar_arrive_expect_tx(bar, 2 * kUnitBytes);
        tma_load_2d(dst, &kmap, bar, 0, id, policy);
        tma_load_2d(dst + kUnitBytes, &vmap, bar, 0, id, policy);
      } else {
        mbar_arrive_local(bar);
        if (c.status) atomicOr(c.status, WAMFFN_DEV_BAD_INDEX);
      }
    }
    issued = i + 1;
  };
  for (int i = 0; i < min(mine, kFewStages); ++i) issue(i);

  // Query fragments, dims [32 t, 32 t + 32) of row g (and of row g + 8 unless narrow): step ks = 4 c + w takes dims
  // 32 t + 16 c + 4 w + {0, 1} and {2, 3} as its k columns 2 t, 2 t + 1 and 2 t + 8, 2 t + 9.
  constexpr int kHalves = kNarrow ? 1 : 2;
  uint32_t qa[8][2 * kHalves];
  float qf[2];      // 2^eq log2(e) / sqrt(128) of the lane's rows: 2 t, 2 t + 1 if narrow, else g, g + 8
  int seen[2];      // keys that these see
#pragma unroll
  for (int half = 0; half < kHalves; ++half) {
    const int r = g + 8 * half;
    const bool live = r < rows;
    const int token = live ? r / p.group : 0;
    const int head = kh * p.group + (live ? r - token * p.group : 0);
    const __nv_bfloat16* src = p.q + b * p.q_batch + token * p.q_row + size_t(head) * kCacheDim + 32 * t;
    uint4 u[4];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = live ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(bf2_lo(w[e])), fabsf(bf2_hi(w[e]))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int eq = query_exp(top);
    const float inv = exp2_int(-eq);
    qf[half] = exp2_int(eq) * p.scale_log2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)  // words 4 i + e: dims 32 t + 8 i + 2 e; step 2 i + e / 2, column pair e % 2
        qa[2 * i + (e >> 1)][half + kHalves * (e & 1)] = f16x2_pack(bf2_lo(w[e]) * inv, bf2_hi(w[e]) * inv);
    }
  }
  if constexpr (kNarrow) {
    const float mine_qf = qf[0];
    qf[0] = __shfl_sync(0xffffffffu, mine_qf, 8 * t);
    qf[1] = __shfl_sync(0xffffffffu, mine_qf, 8 * t + 4);
  }
  auto row_of = [&](int i) { return kNarrow ? 2 * t + i : g + 8 * i; };  // the lane's two rows
#pragma unroll
  for (int i = 0; i < 2; ++i)
    seen[i] = row_of(i) < rows ? keys_seen(length, p.nq, row_of(i) / p.group, p.causal) : 0;

  // Narrow: o[i] = dims 16 g + 2 i (+ 1 in the upper two) of rows 2 t, 2 t + 1; else o[n] = dims 32 t + n (+ 16) of
  // rows g, g + 8.
  float o[kNarrow ? 8 : 16][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  Info now = ahead;
  int now_chunk = 0;
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const int s = i % kFewStages;
    if ((i >> 5) != now_chunk) {
      now_chunk = i >> 5;
      now = info_of(now_chunk * 32 + lane, table_at(now_chunk * 32 + lane));
    }
    const int id = __shfl_sync(0xffffffffu, now.id, i & 31);
    const float kf = exp2_int(scale_exp(__shfl_sync(0xffffffffu, now.ks, i & 31)));
    const int ev = scale_exp(__shfl_sync(0xffffffffu, now.vs, i & 31));
    ok = wait_bounded(smem_addr(&my_full[s]), uint32_t(i / kFewStages) & 1u, &abort_flag, c.status, WAMFFN_DEV_TIMEOUT);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    if (id >= 0) {
      const int key0 = (worker + i * workers) * kUnitKeys;
      const uint32_t kb = smem_addr(my_ring + s * 2 * kUnitBytes), vb = kb + kUnitBytes;
      // S: x[j][e] is row row_of(e & 1) (narrow) or row_of(e >> 1), key 16 j + g + 8 (e >> 1) (narrow) or
      // 8 j + 2 t + (e & 1).  The tiles' sums advance together.
      constexpr int kTiles = kNarrow ? 2 : 4;
      float x[kTiles][4] = {};
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        uint32_t w[4][4];  // keys 8 j + g, 16 dims
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 u = lds128(kb + (j * 8 + g) * kCacheDim + (((2 * t + cc) ^ g) << 4));
          w[j][0] = u.x, w[j][1] = u.y, w[j][2] = u.z, w[j][3] = u.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            const uint32_t* q = qa[cc * 4 + e];
            if constexpr (kNarrow) {
              const uint32_t ka[4] = {e4m3x2_to_f16x2(w[2 * j][e]), e4m3x2_to_f16x2(w[2 * j + 1][e]),
                                      e4m3x2_hi_to_f16x2(w[2 * j][e]), e4m3x2_hi_to_f16x2(w[2 * j + 1][e])};
              mma_f16(x[j], ka, q[0], q[1]);
            } else {
              const uint32_t a[4] = {q[0], q[1], q[2], q[3]};
              mma_f16(x[j], a, e4m3x2_to_f16x2(w[j][e]), e4m3x2_hi_to_f16x2(w[j][e]));
            }
          }
      }
      auto slot = [](int e) { return kNarrow ? e & 1 : e >> 1; };  // which of the lane's rows x[.][e] belongs to
      const bool whole = key0 + kUnitKeys <= least;  // every row sees every key of the unit
      if (!whole) {
        // Keys that every row sees need no look.
#pragma unroll 1
        for (int e = max(0, (least < most ? least : length) - key0) * 8 + lane; e < kUnitKeys * 8; e += 32) {
          const int row = e >> 3, chunk = e & 7;
          const uint32_t at = vb + row * kCacheDim + (chunk << 4);
          sts128(at, clean_chunk(lds128(at), key0 + row, length, least < most, 16 * (chunk ^ (row & 7)), nan_key,
                                 &nan_any));
        }
        fence_proxy_async();  // the place is refilled by a bulk copy
        __syncwarp();
      }
      // Finite, so that a product of zero stays zero: two huge powers of two may stand for vectors that do not meet.
      const float f[2] = {fminf(qf[0] * kf, FLT_MAX), fminf(qf[1] * kf, FLT_MAX)}, evf = float(ev);
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = fmaf(x[j][e], f[slot(e)], evf);
          const int key = key0 + (kNarrow ? 16 * j + g + 8 * (e >> 1) : 8 * j + 2 * t + (e & 1));
          if (!whole && key >= seen[slot(e)]) v = -INFINITY;
          x[j][e] = v;
          top[slot(e)] = fmaxf(top[slot(e)], v);
        }
      // The first maximum needs no correction; one that grows by at most 2^kLag is left as it is: P stays below f16's
      // range.
      bool apart[2];
      float base[2], sum[2] = {0.f, 0.f}, back[2] = {exp2_int(-ev), exp2_int(-ev)};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int w = kNarrow ? 4 : 1; w < (kNarrow ? 32 : 4); w <<= 1)
          top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], w));
        if (m[half] == -INFINITY) m[half] = top[half];
        apart[half] = top[half] > m[half] + kLag || (top[half] < m[half] - kDeep && top[half] > -INFINITY);
        const float ref = apart[half] ? top[half] : m[half];
        base[half] = kPBias - (ref == -INFINITY ? 0.f : ref);
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = ex2_approx(x[j][e] + base[slot(e)]);
          sum[slot(e)] += x[j][e];
        }
      if (__any_sync(0xffffffffu, apart[0] || apart[1])) {
        float corr[2], keep[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          corr[half] = keep[half] = 1.f;
          if (apart[half]) {
            const bool grown = top[half] > m[half];
            const float fold = ex2_approx(0.5f * (grown ? m[half] - top[half] : top[half] - m[half] - evf));
            if (grown) {
              corr[half] = fold * fold;
              l[half] = folded(l[half], fold);
              m[half] = top[half];
            } else {  // deep: the sum alone gets these
              keep[half] = 0.f;
              back[half] = fold;
              sum[half] *= fold;
            }
          }
        }
#pragma unroll
        for (int n = 0; n < (kNarrow ? 8 : 16); ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] *= corr[slot(e)];
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[j][e] *= keep[slot(e)];
      }
      l[0] = fmaf(sum[0], back[0], l[0]);
      l[1] = fmaf(sum[1], back[1], l[1]);
      // O += P V, 16 keys a step.
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t pa[4];
        if constexpr (kNarrow) {  // keys x rows to rows x keys
          pa[0] = transpose8(f16x2_pack(x[ks][0], x[ks][1]));
          pa[1] = transpose8(f16x2_pack(x[ks][2], x[ks][3]));
        } else {
          pa[0] = f16x2_pack(x[2 * ks][0], x[2 * ks][1]), pa[1] = f16x2_pack(x[2 * ks][2], x[2 * ks][3]);
          pa[2] = f16x2_pack(x[2 * ks + 1][0], x[2 * ks + 1][1]), pa[3] = f16x2_pack(x[2 * ks + 1][2], x[2 * ks + 1][3]);
        }
        uint32_t w[4][4];  // rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the step, dims [16 g, 16 g + 16)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = ks * 16 + 2 * t + (r & 1) + 8 * (r >> 1);
          const uint4 u = lds128(vb + row * kCacheDim + ((g ^ (2 * t + (r & 1))) << 4));
          w[r][0] = u.x, w[r][1] = u.y, w[r][2] = u.z, w[r][3] = u.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = __byte_perm(w[0][e], w[1][e], 0x5140), z = __byte_perm(w[2][e], w[3][e], 0x5140);
          const uint32_t a2 = __byte_perm(w[0][e], w[1][e], 0x7362), z2 = __byte_perm(w[2][e], w[3][e], 0x7362);
          if constexpr (kNarrow) {
            const uint32_t v0[4] = {e4m3x2_to_f16x2(a), e4m3x2_hi_to_f16x2(a), e4m3x2_to_f16x2(z), e4m3x2_hi_to_f16x2(z)};
            const uint32_t v1[4] = {e4m3x2_to_f16x2(a2), e4m3x2_hi_to_f16x2(a2), e4m3x2_to_f16x2(z2),
                                    e4m3x2_hi_to_f16x2(z2)};
            mma_f16(o[2 * e], v0, pa[0], pa[1]);
            mma_f16(o[2 * e + 1], v1, pa[0], pa[1]);
          } else {
            mma_f16(o[4 * e], pa, e4m3x2_to_f16x2(a), e4m3x2_to_f16x2(z));
            mma_f16(o[4 * e + 1], pa, e4m3x2_hi_to_f16x2(a), e4m3x2_hi_to_f16x2(z));
            mma_f16(o[4 * e + 2], pa, e4m3x2_to_f16x2(a2), e4m3x2_to_f16x2(z2));
            mma_f16(o[4 * e + 3], pa, e4m3x2_hi_to_f16x2(a2), e4m3x2_hi_to_f16x2(z2));
          }
        }
      }
    }
    __syncwarp();  // the stage has been read
    if (i + kFewStages < mine) issue(i + kFewStages);
  }
  if (!ok && lane == 0)  // copies in flight land before the shared memory is given up
    for (int i = max(0, issued - kFewStages); i < issued; ++i)
      wait_drain(smem_addr(&my_full[i % kFewStages]), uint32_t(i / kFewStages) & 1u);
  __syncthreads();  // every ring is idle: partial results go over them
  float* held = reinterpret_cast<float*>(my_ring);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int w = kNarrow ? 4 : 1; w < (kNarrow ? 32 : 4); w <<= 1) l[half] += __shfl_xor_sync(0xffffffffu, l[half], w);
    const int r = row_of(half);
    if ((kNarrow ? g : t) == 0) part_ml[warp][r] = make_float2(m[half], l[half]);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int col = 0; col < (kNarrow ? 1 : 2); ++col) {  // four neighbouring dims
        const int dim = kNarrow ? 16 * g + 4 * n : 32 * t + 16 * col + 4 * n;
        float4 v;
        if constexpr (kNarrow)
          v = make_float4(o[2 * n][half], o[2 * n][2 + half], o[2 * n + 1][half], o[2 * n + 1][2 + half]);
        else
          v = make_float4(o[4 * n][2 * half + col], o[4 * n + 1][2 * half + col], o[4 * n + 2][2 * half + col],
                          o[4 * n + 3][2 * half + col]);
        if (nan_any) {
          const float bad = __int_as_float(0x7fffffff);
          if (nan_key[dim] < seen[half]) v.x = bad;
          if (nan_key[dim + 1] < seen[half]) v.y = bad;
          if (nan_key[dim + 2] < seen[half]) v.z = bad;
          if (nan_key[dim + 3] < seen[half]) v.w = bad;
        }
        *reinterpret_cast<float4*>(held + r * kFewPitch + dim) = v;
      }
  }
  __syncthreads();
  // The warps' partial results into warp 0's place.
  for (int i = threadIdx.x; i < rows * (kCacheDim / 4); i += kFewWarps * 32) {
    const int r = i >> 5, d = (i & 31) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kFewWarps; ++k) top = fmaxf(top, part_ml[k][r].x);
    const float safe = top == -INFINITY ? 0.f : top;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kFewWarps; ++k) {
      const float fold = ex2_approx(0.5f * (part_ml[k][r].x - safe)), f = fold * fold;
      const float4 u = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(ring + k * kFewRing) + r * kFewPitch + d);
      v.x += u.x * f, v.y += u.y * f, v.z += u.z * f, v.w += u.w * f;
      sum += folded(part_ml[k][r].y, fold);
    }
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(ring) + r * kFewPitch + d) = v;
    if (d == 0) cta_ml[r] = make_float2(top, sum);
  }
  if (split > 1)
    cluster_sync();
  else
    __syncthreads();
  // The cluster's partial results, in rank order; rank r takes every split-th 4-dim piece.
  for (int i = rank + split * int(threadIdx.x); i < rows * (kCacheDim / 4); i += split * kFewWarps * 32) {
    const int r = i >> 5, d = (i & 31) * 4;
    const uint32_t ml_at = smem_addr(&cta_ml[r]), o_at = smem_addr(reinterpret_cast<float*>(ring) + r * kFewPitch + d);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f), u[8];
    float2 ml[8];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {  // all peers' loads before the first use
      ml[k] = make_float2(-INFINITY, 0.f);
      u[k] = v;
      if (split == 1 && k == 0) {
        ml[k] = cta_ml[r];
        u[k] = *reinterpret_cast<float4*>(reinterpret_cast<float*>(ring) + r * kFewPitch + d);
      } else if (k < split) {
        ml[k] = ld_cluster2(map_to_cta(ml_at, k));
        u[k] = ld_cluster4(map_to_cta(o_at, k));
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
    const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float fold = ex2_approx(0.5f * (ml[k].x - safe)), f = fold * fold;
      v.x += u[k].x * f, v.y += u[k].y * f, v.z += u[k].z * f, v.w += u[k].w * f;
      sum += folded(ml[k].y, fold);
    }
    const int token = r / p.group, head = kh * p.group + r - token * p.group;
    if (!abort_flag) kv_emit(p, part, b, token, head, d, v, top, sum);
  }
  if (split > 1) cluster_sync();  // no CTA leaves while a peer reads its shared memory
}

}  // namespace wamffn
