// Attention over the 8-bit cache for many query rows (kvattend.cuh has the
// formulas and the numbers): tcgen05, 256 packed rows (query token x head of
// the group) a CTA as two tiles of 128.
//
// Bound: the tensor cores and the exponentials, about even (512 flops and one
// exp2 a (row, key); 4096 f16 multiply-adds and 16 exp2 a clock and SM make 128
// rows x 128 keys 1024 clocks of either).  So the two tiles alternate: while one's
// S is turned into P by its warps, the tensor cores work for the other, and a
// converted key block serves both.
//
//   warps 0-3, 4-7  softmax of tile 0 and 1, a query row a thread: Q to f16 in
//                   shared memory once; per step the row maximum, P = 2^(x - m) in f16
//                   over S's own TMEM columns, O rescaled only when the maximum has
//                   grown by more than 2^8 (P then stays below f16's range)
//   warps 8-11      e4m3 -> f16: rows straight from global memory to registers (one
//                   step ahead), converted, stored as 128-byte-swizzled operand tiles
//                   (K: K-major operand of Q K^T; V as it lies: MN-major operand of P V)
//   warp 12         issues S = Q K^T and O += P V (P from TMEM); 13-15 are idle
//
// A step is 128 keys, two blocks with scales of their own.  `split` CTAs of a
// cluster share a row tile's steps and meet through distributed shared memory.
// Every wait is bounded in time and raises WAMFFN_DEV_TIMEOUT.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "kvattend.cuh"

namespace wamffn {

constexpr int kManyRows = 256;
constexpr int kManyStep = 128;
constexpr int kManySoftmaxWarps = 8;
constexpr int kManyConvWarps = 4;
constexpr int kManyThreads = (kManySoftmaxWarps + kManyConvWarps + 4) * 32;  // four warpgroups; three warps of the last idle
// Registers a thread, by warpgroup: the launch gives every thread 128 (65536 / 512), the softmax warpgroups take
// what the others give back (2 * 176 + 112 + 48 = 4 * 128).
constexpr int kManyLaunchRegs = 128, kManySoftmaxRegs = 176, kManyConvRegs = 112, kManyMmaRegs = 48;
static_assert(2 * kManySoftmaxRegs + kManyConvRegs + kManyMmaRegs <= 4 * kManyLaunchRegs, "register split");
constexpr int kManyTile = 128 * 64 * 2;         // 128 rows x 64 f16: half of a [128, 128] operand
constexpr int kManyOperand = 2 * kManyTile;     // 32 KB
constexpr int kManyData = (2 + 2 * 2) * kManyOperand;  // Q of two tiles, two stages of K and V
constexpr int kManySmem = kManyData + 1024;
constexpr int kManyPitch = kCacheDim + 4;       // floats between rows of a partial result
constexpr float kManyBias = 5.f, kManyLag = 8.f;  // P <= 2^(5 + 8)

// f16 operands (K-major A; B K-major or, with bit 16, MN-major), fp32 accumulator.
__host__ __device__ constexpr uint32_t umma_idesc_f16(int m, int n) {
  return (1u << 4) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// D[tmem] (+)= A[tmem] * B[smem]^T.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int kRegs>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// (a.x * f + c, a.y * f + c) in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float f, float c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rf, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rf, {%4, %4};\n\tmov.b64 rc, {%5, %5};\n\t"
      "fma.rn.f32x2 rd, ra, rf, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(f), "f"(c));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Scales of one block for the softmax: x = S (qf kf) + ev, normaliser += sum P * back.
struct ManyScale {
  float kf, ev, back, pad;
};

__global__ void __launch_bounds__(kManyThreads, 1) kv_attend_many_kernel(const KvAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                       // tile x at + x * 32 KB
  uint8_t* k_s = smem + 2 * kManyOperand;    // stage s at + s * 32 KB
  uint8_t* v_s = smem + 4 * kManyOperand;
  __shared__ __align__(8) uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2],
      o_done[2];
  __shared__ __align__(16) ManyScale scale_s[4][2];  // of the steps in flight
  __shared__ __align__(16) float2 cta_ml[kManyRows];
  __shared__ int nan_key[kCacheDim];
  __shared__ int nan_any;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  volatile int* abort = &abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split, kh = blockIdx.y, b = blockIdx.z;
  // The last row tile first: with a causal mask it has the most keys.
  const int tile = int(gridDim.x / split) - 1 - int(blockIdx.x) / split, rank = int(blockIdx.x) % split;
  constexpr int kMmaWarp = kManySoftmaxWarps + kManyConvWarps;

  if (threadIdx.x == 0) {
    mbar_init(smem_addr(&q_full), kManySoftmaxWarps);
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_addr(&k_full[s]), kManyConvWarps);
      mbar_init(smem_addr(&v_full[s]), kManyConvWarps);
      mbar_init(smem_addr(&k_empty[s]), 1);
      mbar_init(smem_addr(&v_empty[s]), 1);
      mbar_init(smem_addr(&s_full[s]), 1);
      mbar_init(smem_addr(&p_full[s]), 4);
      mbar_init(smem_addr(&o_done[s]), 1);
    }
    abort_flag = 0;
    nan_any = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < kCacheDim) nan_key[threadIdx.x] = 0x7fffffff;
  if (warp == kMmaWarp) {
    tmem_alloc(smem_addr(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait_prior();
  pdl_launch_dependents();
  const uint32_t tmem = tmem_slot;  // S0 [0, 128), S1 [128, 256), O0 [256, 384), O1 [384, 512)

  const CacheView& c = p.c;
  const int length = cache_length(c, b);
  const int total_rows = p.nq * p.group, row0 = tile * kManyRows;
  const int rows = min(kManyRows, total_rows - row0);
  const int tiles = rows > 128 ? 2 : 1;
  const int least = keys_seen(length, p.nq, row0 / p.group, p.causal);
  const int most = keys_seen(length, p.nq, (row0 + rows - 1) / p.group, p.causal);
  const int all_steps = (most + kManyStep - 1) / kManyStep;
  const int first = int((long long)rank * all_steps / split);
  const int steps = int((long long)(rank + 1) * all_steps / split) - first;

  float m = -INFINITY, l = 0.f;  // of this softmax thread's row
  int seen = 0;
  bool ok = true;

  if (warp >= kMmaWarp) {
    // ------------------------------------------------------------ products
    give_registers<kManyMmaRegs>();
    constexpr uint32_t idesc_s = umma_idesc_f16(128, kManyStep);
    constexpr uint32_t idesc_o = umma_idesc_f16(128, kCacheDim) | (1u << 16);  // V MN-major
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      int good = 1;
      if (lane == 0) good = wait_bounded(smem_addr(bar), parity, abort, c.status, WAMFFN_DEV_TIMEOUT);
      good = __shfl_sync(0xffffffffu, good, 0);
      tc_fence_after();
      return good != 0;
    };
    auto issue_s = [&](int x, int j) {
      if (elect_one()) {
        const uint32_t qa = smem_addr(q_s + x * kManyOperand), ka = smem_addr(k_s + (j & 1) * kManyOperand);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_bf16(tmem + x * 128, umma_desc_sw128(qa + (k >> 2) * kManyTile) + 2 * (k & 3),
                    umma_desc_sw128(ka + (k >> 2) * kManyTile) + 2 * (k & 3), idesc_s, k ? 1u : 0u);
        umma_commit(smem_addr(&s_full[x]));
        if (x == tiles - 1) umma_commit(smem_addr(&k_empty[j & 1]));
      }
      __syncwarp();
    };
    if (warp == kMmaWarp && steps > 0) {
      ok = wait(&q_full, 0u) && wait(&k_full[0], 0u);
      if (ok)
        for (int x = 0; x < tiles; ++x) issue_s(x, 0);
      for (int j = 0; j < steps && ok; ++j) {
        for (int x = 0; x < tiles && ok; ++x) {
          ok = wait(&v_full[j & 1], uint32_t(j >> 1) & 1u) && wait(&p_full[x], uint32_t(j) & 1u);
          if (!ok) break;
          if (elect_one()) {
            const uint32_t va = smem_addr(v_s + (j & 1) * kManyOperand);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_f16_ts(tmem + 256 + x * 128, tmem + x * 128 + k * 8,
                          umma_desc_sw128_mn(va + uint32_t(k) * 2 * kVGroupBytes, kVHalfBytes, kVGroupBytes), idesc_o,
                          (j | k) ? 1u : 0u);
            if (x == tiles - 1) umma_commit(smem_addr(&v_empty[j & 1]));
            if (j == steps - 1) umma_commit(smem_addr(&o_done[x]));
          }
          __syncwarp();
          if (j + 1 < steps) {
            ok = wait(&k_full[(j + 1) & 1], uint32_t((j + 1) >> 1) & 1u);
            if (ok) issue_s(x, j + 1);
          }
        }
      }
    }
    __syncwarp();
    if (split > 1) {  // the softmax warps' two cluster barriers
      cluster_sync();
      cluster_sync();
    }
  } else if (warp >= kManySoftmaxWarps) {
    // ------------------------------------------------------------ e4m3 -> f16
    // Thread: raw 16-byte chunk 4 half + c4 (dims 64 half + 16 c4) of rows
    // r0 + 16 i.  Eight neighbouring lanes store 4 chunks of an even and of an odd
    // row: distinct banks under the swizzle.
    give_registers<kManyConvRegs>();
    const int tid = threadIdx.x - kManySoftmaxWarps * 32;
    const int c4 = tid & 3, half = (tid >> 3) & 1, r0 = ((tid >> 2) & 1) + 2 * (tid >> 4);
    const int* table = c.table + b * c.table_stride;
    const size_t in_tile = size_t(r0) * kCacheDim + half * 64 + c4 * 16;
    auto block_of = [&](int j, int i) -> long long {  // pool tile of block i of step j; -1: none or a bad id
      const int at = 2 * (first + j) + i;
      if (j >= steps || at >= c.width) return -1;  // a length that ends in the step's first block
      const int id = table[at];
      if (id >= 0 && id < c.blocks) return (long long)id * c.kv_heads + kh;
      if (at * kCacheBlock < most && c.status && tid == 0) atomicOr(c.status, WAMFFN_DEV_BAD_INDEX);
      return -1;
    };
    auto load = [&](const uint8_t* base, const long long (&at)[2], uint4 (&raw)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        raw[i] = at[i >> 2] >= 0 ? *reinterpret_cast<const uint4*>(base + at[i >> 2] * kCacheTile + in_tile +
                                                                   (i & 3) * 16 * kCacheDim)
                                 : make_uint4(0, 0, 0, 0);
    };
    auto store = [&](uint8_t* operand, const uint4 (&raw)[8]) {
      uint8_t* dst = operand + half * kManyTile;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + 16 * i;
        *reinterpret_cast<uint4*>(dst + sw128_offset(r, 2 * c4)) =
            make_uint4(e4m3x2_to_f16x2(raw[i].x), e4m3x2_hi_to_f16x2(raw[i].x), e4m3x2_to_f16x2(raw[i].y),
                       e4m3x2_hi_to_f16x2(raw[i].y));
        *reinterpret_cast<uint4*>(dst + sw128_offset(r, 2 * c4 + 1)) =
            make_uint4(e4m3x2_to_f16x2(raw[i].z), e4m3x2_hi_to_f16x2(raw[i].z), e4m3x2_to_f16x2(raw[i].w),
                       e4m3x2_hi_to_f16x2(raw[i].w));
      }
    };
    auto wait = [&](uint64_t* bar, int j) {  // the stage's operand of step j - 2 has been read
      int good = 1;
      if (lane == 0)
        good = wait_bounded(smem_addr(bar), uint32_t((j >> 1) - 1) & 1u, abort, c.status, WAMFFN_DEV_TIMEOUT);
      return __shfl_sync(0xffffffffu, good, 0) != 0;
    };
    auto signal = [&](uint64_t* bar) {
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(smem_addr(bar));
    };
    long long at[2], next[2];
    uint4 kraw[8], vraw[8];
    float ks = 0.f, vs = 0.f;  // scales of block tid, of the step in kraw
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      at[i] = block_of(0, i);
      next[i] = block_of(1, i);
    }
    auto load_scales = [&]() {
      const long long t = tid == 0 ? at[0] : at[1];
      if (tid < 2 && t >= 0) {
        ks = c.key_scales[t];
        vs = c.value_scales[t];
      }
      if (t < 0) ks = vs = 0.f;
    };
    if (steps > 0) {
      load(c.keys, at, kraw);
      load(c.values, at, vraw);
      load_scales();
    }
    for (int j = 0; j < steps; ++j) {
      const int key0 = (first + j) * kManyStep;
      if (j >= 2 && !wait(&k_empty[j & 1], j)) break;
      if (tid < 2) {
        ManyScale s{1.f, -INFINITY, 0.f, 0.f};  // a block that is not there: nothing seen
        if (ks > 0.f) {
          const int ev = scale_exp(vs);
          s = ManyScale{exp2_int(scale_exp(ks)), float(ev), exp2_int(-ev), 0.f};
        }
        scale_s[j & 3][tid] = s;
      }
      store(k_s + (j & 1) * kManyOperand, kraw);
      signal(&k_full[j & 1]);
      if (j >= 2 && !wait(&v_empty[j & 1], j)) break;
      if (key0 + kManyStep > least) {  // some row sees less than the whole step
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = key0 + r0 + 16 * i, dim = half * 64 + c4 * 16;
          vraw[i].x = clean_word(vraw[i].x, key, length, dim, nan_key, &nan_any);
          vraw[i].y = clean_word(vraw[i].y, key, length, dim + 4, nan_key, &nan_any);
          vraw[i].z = clean_word(vraw[i].z, key, length, dim + 8, nan_key, &nan_any);
          vraw[i].w = clean_word(vraw[i].w, key, length, dim + 12, nan_key, &nan_any);
        }
      }
      store(v_s + (j & 1) * kManyOperand, vraw);
      signal(&v_full[j & 1]);
      at[0] = next[0];
      at[1] = next[1];
      if (j + 1 < steps) {
        load(c.keys, at, kraw);
        load(c.values, at, vraw);
        load_scales();
        next[0] = block_of(j + 2, 0);
        next[1] = block_of(j + 2, 1);
      }
    }
    __syncwarp();
    if (split > 1) {
      cluster_sync();
      cluster_sync();
    }
  } else {
    // ------------------------------------------------------------ softmax
    take_registers<kManySoftmaxRegs>();
    const int x = warp >> 2, r = threadIdx.x;  // tile; row of the CTA's 256
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + x * 128 + lanes, to = tmem + 256 + x * 128 + lanes;
    const bool live = r < rows;
    const int row = row0 + (live ? r : 0), token = row / p.group, head = kh * p.group + row - token * p.group;
    float qf;
    {  // this row of Q: largest magnitude, power of two, f16, operand tile
      const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.q_batch + token * p.q_row + size_t(head) * kCacheDim);
      uint4 u[16];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) u[i] = live ? src[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(bf2_lo(w[e])), fabsf(bf2_hi(w[e]))));
      }
      const int eq = query_exp(top);
      const float inv = exp2_int(-eq);
      qf = exp2_int(eq) * p.scale_log2;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = f16x2_pack(bf2_lo(w[e]) * inv, bf2_hi(w[e]) * inv);
        *reinterpret_cast<uint4*>(q_s + x * kManyOperand + (i >> 3) * kManyTile + sw128_offset(r & 127, i & 7)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(smem_addr(&q_full));
    }
    seen = live ? keys_seen(length, p.nq, token, p.causal) : 0;
    // One step: S of the row's 128 keys to P.
    auto step = [&](int j, auto whole_c) {
      constexpr bool kWhole = decltype(whole_c)::value;
      const int limit = seen - (first + j) * kManyStep;  // keys of the step that the row sees
      const ManyScale sc[2] = {scale_s[j & 3][0], scale_s[j & 3][1]};
      uint32_t v[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_ld32(ts + q * 32, v[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_wait_ld(v[q]);
      if constexpr (!kWhole) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= limit) v[i >> 5][i & 31] = 0xff800000u;  // -inf
      }
      // The row's maximum: of S in each block (its factor is positive), then of x.
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            t[e] = fmaxf(fmaxf(t[e], __uint_as_float(v[2 * h + (i >> 5)][(i & 31) + 2 * e])),
                         __uint_as_float(v[2 * h + (i >> 5)][(i & 31) + 2 * e + 1]));
        const float u = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        // A block that is not there has ev -inf; nothing seen leaves u at -inf.
        top = fmaxf(top, u == -INFINITY ? -INFINITY : fmaf(u, qf * sc[h].kf, sc[h].ev));
      }
      // A maximum that grows by at most 2^kManyLag is left as it is.
      float corr = 1.f;
      const bool grown = top > m + kManyLag || (m == -INFINITY && top > m);
      if (grown) {
        corr = ex2_approx(m - top);
        m = top;
        l *= corr;
      }
      const float safe = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = qf * sc[h].kf, base = sc[h].ev - safe + kManyBias;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t out[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const uint32_t a = v[2 * h + (i >> 4)][2 * (i & 15)], z = v[2 * h + (i >> 4)][2 * (i & 15) + 1];
          float2 e = fma2(make_float2(__uint_as_float(a), __uint_as_float(z)), f, base);
          e.x = ex2_approx(e.x);
          e.y = ex2_approx(e.y);
          sum[i & 1] = add2(sum[i & 1], e);
          out[i] = f16x2_pack(e.x, e.y);
        }
        l = fmaf((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), sc[h].back, l);
        tmem_st32(ts + h * 32, out);
      }
      if (__any_sync(0xffffffffu, grown) && j > 0) {
        // S of this step is complete, so every product into O before it is.
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[32];
          tmem_ld32(to + q * 32, w);
          tmem_wait_ld(w);
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * corr);
          tmem_st32(to + q * 32, w);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(smem_addr(&p_full[x]));
    };
    if (x < tiles) {
      for (int j = 0; j < steps; ++j) {
        if (lane == 0) ok = wait_bounded(smem_addr(&s_full[x]), uint32_t(j) & 1u, abort, c.status, WAMFFN_DEV_TIMEOUT);
        ok = __shfl_sync(0xffffffffu, int(ok), 0);
        if (!ok) break;
        tc_fence_after();
        if ((first + j + 1) * kManyStep <= least)
          step(j, std::true_type{});
        else
          step(j, std::false_type{});
      }
    }
    if (steps > 0 && ok) {  // both tiles: the rings are reused below
      if (lane == 0)
        for (int y = 0; y < tiles; ++y)
          ok = ok && wait_bounded(smem_addr(&o_done[y]), 0u, abort, c.status, WAMFFN_DEV_TIMEOUT);
      ok = __shfl_sync(0xffffffffu, int(ok), 0);
      tc_fence_after();
    }
    if (split == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
      __nv_bfloat16* dst = p.out + ((size_t(b) * p.nq + token) * p.heads + head) * kCacheDim;
      if (x < tiles && ok) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t v[32];
          if (steps > 0) {
            tmem_ld32(to + q * 32, v);
            tmem_wait_ld(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
          }
          if (nan_any)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (nan_key[q * 32 + i] < seen) v[i] = 0x7fffffffu;
          if (live)
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              float o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(v[i + e]) * inv;
              *reinterpret_cast<uint4*>(dst + q * 32 + i) =
                  make_uint4(bf2_pack(o[0], o[1]), bf2_pack(o[2], o[3]), bf2_pack(o[4], o[5]), bf2_pack(o[6], o[7]));
            }
        }
      }
    } else {
      // This CTA's partial rows (unnormalised O, maximum, normaliser) to shared memory.
      float* part = reinterpret_cast<float*>(smem);
      named_sync(1, kManySoftmaxWarps * 32);  // every softmax warp has seen both tiles' products complete
      if (x < tiles) {
        cta_ml[r] = make_float2(m, l);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t v[32];
          if (steps > 0) {
            tmem_ld32(to + q * 32, v);
            tmem_wait_ld(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
          }
          if (nan_any)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (nan_key[q * 32 + i] < seen) v[i] = 0x7fffffffu;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(part + r * kManyPitch + q * 32 + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
      __syncwarp();
      cluster_sync();
      // Rank order; rank k takes rows k, k + split, ...
      const int pieces = ((rows - rank + split - 1) / split) * (kCacheDim / 4);
      for (int i = threadIdx.x; i < pieces; i += kManySoftmaxWarps * 32) {
        const int pr = rank + (i >> 5) * split, d = (i & 31) * 4;
        const uint32_t ml_at = smem_addr(&cta_ml[pr]), o_at = smem_addr(part + pr * kManyPitch + d);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, sum = 0.f;
        for (int k = 0; k < split; ++k) {
          const float2 ml = ld_cluster2(map_to_cta(ml_at, k));
          const float4 u = ld_cluster4(map_to_cta(o_at, k));
          const float next = fmaxf(top, ml.x), safe = next == -INFINITY ? 0.f : next;
          const float fo = ex2_approx(top - safe), fn = ex2_approx(ml.x - safe);
          v.x = v.x * fo + u.x * fn, v.y = v.y * fo + u.y * fn;
          v.z = v.z * fo + u.z * fn, v.w = v.w * fo + u.w * fn;
          sum = sum * fo + ml.y * fn;
          top = next;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int prow = row0 + pr, ptoken = prow / p.group, phead = kh * p.group + prow - ptoken * p.group;
        if (!*abort)
          *reinterpret_cast<uint2*>(p.out + ((size_t(b) * p.nq + ptoken) * p.heads + phead) * kCacheDim + d) =
              make_uint2(bf2_pack(v.x * inv, v.y * inv), bf2_pack(v.z * inv, v.w * inv));
      }
      __syncwarp();
      cluster_sync();  // no CTA leaves while a peer reads its shared memory
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace wamffn
