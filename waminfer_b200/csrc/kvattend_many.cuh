// Attention over the 8-bit cache for many query rows (kvattend.cuh has the
// formulas and the numbers): tcgen05, 256 packed rows (query token x head of
// the group) a CTA as two tiles of 128, a step of 64 keys (one block).
//
// Bound: shared memory, then the tensor cores and the exponentials (512 flops and one
// exp2 a (row, key); 4096 f16 multiply-adds and 16 exp2 a clock and SM make two tiles
// of 128 rows x 64 keys 1024 clocks of either).  A step of two tiles moves 192 KB through
// shared memory: the products 128 (S: Q 64 and K 32; P V: V 32), the block's copy 16, its
// conversion 16 in and 32 out; at 128 bytes a clock 1536 clocks.  So
//   - a converted block serves both tiles; a CTA with at most 128 rows has them in both,
//     the even steps in one and the odd steps in the other;
//   - each tile has two S buffers: S of step j + 1 is there before P of step j is,
//     so neither the warps nor the tensor cores wait for a step's whole chain;
//   - blocks arrive by bulk copies, as they are held, two steps ahead of their
//     conversion.  (Loads to registers instead are slower the further ahead they are:
//     the fence between a conversion's stores and the products waits for them.)
//
// On a B200, 512 queries of 37 heads over 16384 rows (every SM busy) take 161 us, 989
// TFLOP/s, 60 % of the measured bf16 GEMM burst; 392 queries of 24 heads over 32768 rows
// 215 us (232 once the card is at its power limit).  Of the 2310 clocks of a step the
// counters show shared memory's data pipe busy for 1620 (70 %: 1024 wavefronts of the
// products, 600 of the warps) beside the bulk copies, the tensor pipe for 44 %, the
// exponentials' for 45 %.  What stretches a step beyond them is the chain of a tile's
// products, row maximum and exponentials (P of step j must be read before S of step j + 2
// takes its columns; TMEM has no room for a third buffer).
//
//   warps 8-11, 12-15  softmax of tile 0 and 1, a query row a thread: Q to f16 in shared
//                   memory once; per step the row maximum, P = 2^(x - m) in f16 over
//                   S's own TMEM columns, O rescaled only when the maximum has grown by
//                   more than 2^8 (P then stays below f16's range)
//   warps 4-7       e4m3 -> f16 through registers, stored as 128-byte-swizzled operand tiles (K: K-major
//                   operand of Q K^T; V as it lies: MN-major operand of P V)
//   warps 0, 1      one thread a tile issues S = Q K^T and O += P V; warp 3 is idle
//   warp 2          bulk copies of the blocks, 8 KB of K and of V, and their scales
//
// TMEM: S of tile x, step j at 128 x + 64 (j & 1), O of tile x at 256 + 128 x.
// `split` CTAs of a cluster share a row tile's steps (of a part) and meet through
// distributed shared memory.  Every wait is bounded in time and raises WAMFFN_DEV_TIMEOUT.
// The loops are kept small (one copy of each, rare paths not unrolled): all roles
// share the instruction cache.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "kvattend.cuh"

namespace wamffn {

constexpr int kManyRows = 256;
constexpr int kManyStep = kCacheBlock;
constexpr int kManySoftmaxWarps = 8, kManyConvWarps = 4;
// Warps in the order of their urgency: the scheduler prefers older ones.
constexpr int kManyConvWarp0 = 4, kManySoftmaxWarp0 = 8;
constexpr int kManyThreads = 16 * 32;
// Registers a thread, by warpgroup: the launch gives every thread 128 (65536 / 512); the warpgroup of the issuing
// threads hands over what the others take (80 + 112 + 2 * 160 = 4 * 128).
constexpr int kManyLaunchRegs = 128, kManyMmaRegs = 80, kManyConvRegs = 112, kManySoftmaxRegs = 160;
static_assert(kManyMmaRegs + kManyConvRegs + 2 * kManySoftmaxRegs <= 4 * kManyLaunchRegs, "register split");
constexpr int kManyHalf = kManyStep * 64 * 2;   // 64 rows x 64 f16: half of an operand tile
constexpr int kManyOperand = 2 * kManyHalf;     // 16 KB
constexpr int kManyStages = 5;                  // of K, and of V, in f16, with one tile's Q; one less with two
constexpr int kManyRaw = 2;                     // blocks (K and V) as they are held, 16 KB each
constexpr int kManyQuery = 2 * 128 * 64 * 2;    // Q of a tile: two halves of 128 rows x 64 f16
constexpr int kManyOperands = kManyQuery + 2 * kManyStages * kManyOperand;  // Q and the stages
static_assert(kManyQuery == 2 * kManyOperand, "a second Q takes a stage's place");
constexpr int kManyData = kManyOperands + kManyRaw * 2 * kCacheTile;
constexpr int kManyPitch = kCacheDim + 4;       // floats between rows of a partial result
constexpr uint32_t kManyO = 256;  // TMEM column of tile 0's O

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
__device__ __forceinline__ void set_registers() {
  if constexpr (kRegs < kManyLaunchRegs)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
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

// Scales of a block for the softmax: x = S (qf kf) + ev, normaliser += sum P * back.
struct ManyScale {
  float kf, ev, back, there;
};

struct ManyShared {
  uint64_t q_full, s_full[2][2], p_full[2][2];            // S, P: tile, buffer
  uint64_t o_step[2], o_last[2];                         // a step's, the last step's product into O is complete: tile
  uint64_t full[kManyStages], empty[kManyStages];        // K and V of a step in f16
  uint64_t raw_full[kManyRaw], raw_empty[kManyRaw];
  ManyScale scale[8];                                    // of the steps in flight
  int nan_key[kCacheDim];
  int nan_any, abort_flag;
  uint32_t tmem_slot;
};
constexpr int kManySmem = 1024 + kManyData + int(sizeof(ManyShared));
static_assert(kManySmem <= 232448, "227 KB a CTA");
static_assert(kManyRows * (kManyPitch * 4 + 8) <= kManyData, "partial rows fit the operands' place");
static_assert(kManyStages + kManyRaw < 8, "a step's scales are kept until it is done");

__global__ void __launch_bounds__(kManyThreads, 1) kv_attend_many_kernel(const KvAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  ManyShared& sh = *reinterpret_cast<ManyShared*>(smem + kManyData);
  volatile int* abort = &sh.abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int shares = split * p.parts, share = int(blockIdx.x) % shares;  // of the keys: rank of the cluster in its part
  const int rank = share % split, part = share / split;
  // In the order of launch: with a causal mask the last row tile, which has the most keys, of every head, then the one
  // before, so that the short ones even out the end (16384 rows over 4096: 174 us; head by head 16 % more); without one
  // head by head, whose CTAs then read the same blocks (392 queries over 32768 rows: 215 us; 216 us tile by tile).
  const int tiles = int(gridDim.x) / shares, unit = int(blockIdx.y) * tiles + int(blockIdx.x) / shares;
  const int b = blockIdx.z, kh = p.causal ? unit % int(gridDim.y) : int(blockIdx.y);
  const int tile = tiles - 1 - (p.causal ? unit / int(gridDim.y) : int(blockIdx.x) / shares);
  const int total_rows = p.nq * p.group, row0 = tile * p.tile_rows;
  const int rows = min(p.tile_rows, total_rows - row0);
  const bool dual = rows <= 128;  // both tiles hold the same rows and take every second step
  const int stride = dual ? 2 : 1;
  const int stages = dual ? kManyStages : kManyStages - 1;
  // Q of tile x (dual: the same for both), operand tile of K (w = 0) or V (w = 1) in stage s, raw block r.
  auto query = [&](int x) { return smem + (dual ? 0 : x) * kManyQuery; };
  auto operand = [&](int w, int s) {
    return smem + (dual ? 1 : 2) * kManyQuery + (w * stages + s) * kManyOperand;
  };
  auto raw_block = [&](int r) { return smem + kManyOperands + r * 2 * kCacheTile; };

  if (threadIdx.x == 0) {
    mbar_init(smem_addr(&sh.q_full), kManySoftmaxWarps);
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_addr(&sh.o_step[x]), 1);
      mbar_init(smem_addr(&sh.o_last[x]), 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_addr(&sh.s_full[x][i]), 1);
        mbar_init(smem_addr(&sh.p_full[x][i]), 4);
      }
    }
    for (int s = 0; s < kManyStages; ++s) {
      mbar_init(smem_addr(&sh.full[s]), kManyConvWarps);
      mbar_init(smem_addr(&sh.empty[s]), dual ? 1 : 2);  // tiles that read a step
    }
    for (int r = 0; r < kManyRaw; ++r) {
      mbar_init(smem_addr(&sh.raw_full[r]), 1);
      mbar_init(smem_addr(&sh.raw_empty[r]), kManyConvWarps);
    }
    sh.abort_flag = 0;
    sh.nan_any = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < kCacheDim) sh.nan_key[threadIdx.x] = 0x7fffffff;
  if (warp == 0) {
    tmem_alloc(smem_addr(&sh.tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait_prior();
  pdl_launch_dependents();
  const uint32_t tmem = sh.tmem_slot;

  const CacheView& c = p.c;
  const int length = cache_length(c, b);
  const int least = keys_seen(length, p.nq, row0 / p.group, p.causal);
  const int most = keys_seen(length, p.nq, (row0 + rows - 1) / p.group, p.causal);
  const int all_steps = (most + kManyStep - 1) / kManyStep;
  const int first = int((long long)share * all_steps / shares);
  const int steps = int((long long)(share + 1) * all_steps / shares) - first;

  if (warp < kManyConvWarp0) {
    // ------------------------------------------------------------ products
    set_registers<kManyMmaRegs>();
    // The elected lane runs the whole loop: its operands then stay in uniform registers (11 cycles to issue a
    // product; 27 with a lane elected for each group of products, 54 from a lane chosen by its index).
    if (warp < 2 && (dual ? warp : 0) < steps && elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_f16(128, kManyStep);
      constexpr uint32_t idesc_o = umma_idesc_f16(128, kCacheDim) | (1u << 16);  // V MN-major
      const int x = warp;
      const uint32_t ts = tmem + x * 128, to = tmem + kManyO + x * 128, qa = smem_addr(query(x));
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return wait_spin(smem_addr(bar), parity, abort, c.status, WAMFFN_DEV_TIMEOUT);
      };
      // S of the tile into buffer i from K stage s.
      auto issue_s = [&](int i, int s) {
        const uint32_t ka = smem_addr(operand(0, s));
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_bf16(ts + i * 64, umma_desc_sw128(qa + (k >> 2) * (kManyQuery / 2)) + 2 * (k & 3),
                    umma_desc_sw128(ka + (k >> 2) * kManyHalf) + 2 * (k & 3), idesc_s, k ? 1u : 0u);
        umma_commit(smem_addr(&sh.s_full[x][i]));
      };
      const int first_step = dual ? x : 0;
      bool ok = wait(&sh.q_full, 0u) && wait(&sh.full[first_step], 0u);
      tc_fence_after();
      if (ok) issue_s(0, first_step);
      int s = first_step, n = first_step + stride;  // stages of this tile's steps i and i + 1
      uint32_t phn = 0;                             // phase of n
      for (int i = 0, j = first_step; j < steps && ok; ++i, j += stride) {
        // S of the next step goes over P of the one before: that step's product must be complete (products of
        // different shapes are not ordered among themselves).
        if (j + stride < steps) {
          ok = wait(&sh.full[n], phn) && (i == 0 || wait(&sh.o_step[x], uint32_t(i - 1) & 1u));
          if (!ok) break;
          tc_fence_after();
          issue_s((i + 1) & 1, n);
        }
        ok = wait(&sh.p_full[x][i & 1], uint32_t(i >> 1) & 1u);
        if (!ok) break;
        tc_fence_after();
        const uint32_t va = smem_addr(operand(1, s));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16_ts(to, ts + (i & 1) * 64 + k * 8,
                      umma_desc_sw128_mn(va + uint32_t(k) * 2 * kVGroupBytes, kManyHalf, kVGroupBytes), idesc_o,
                      (i | k) ? 1u : 0u);
        umma_commit(smem_addr(&sh.o_step[x]));
        umma_commit(smem_addr(&sh.empty[s]));
        s = n;
        n += stride;
        if (n >= stages) n -= stages, phn ^= 1u;
      }
      umma_commit(smem_addr(&sh.o_last[x]));
      if (!ok) wait_drain(smem_addr(&sh.o_last[x]), 0u);  // no product reads memory that is given up
    }
    if (warp == 2) {
      // ---------------------------------------------------------- blocks and their scales
      const int* table = c.table + b * c.table_stride;
      auto id_of = [&](int i) { return i < steps ? table[first + i] : -1; };
      int chunk = 0, id = id_of(lane), next_id = id_of(32 + lane);  // of steps 32 chunk + lane, and of the 32 after
      float ks = 0.f, vs = 0.f;
      auto load_scales = [&]() {
        if (id < 0 || id >= c.blocks) {
          id = -1;
        } else {
          const size_t at = size_t(id) * c.kv_heads + kh;
          ks = c.key_scales[at];
          vs = c.value_scales[at];
        }
      };
      load_scales();
      int r = 0, sent = 0, ok = 1;
      uint32_t ph = 1u;
      for (int j = 0; j < steps; ++j) {
        if ((j >> 5) != chunk) {
          chunk = j >> 5;
          id = next_id;
          load_scales();
          next_id = id_of(32 * chunk + 32 + lane);
        }
        const int at = __shfl_sync(0xffffffffu, id, j & 31);
        const float kj = __shfl_sync(0xffffffffu, ks, j & 31), vj = __shfl_sync(0xffffffffu, vs, j & 31);
        if (lane == 0) {
          const uint32_t bar = smem_addr(&sh.raw_full[r]), dst = smem_addr(raw_block(r));
          if (j >= kManyRaw) ok = wait_spin(smem_addr(&sh.raw_empty[r]), ph, abort, c.status, WAMFFN_DEV_TIMEOUT);
          if (ok) {
            if (at >= 0) {
              const int ev = scale_exp(vj);
              sh.scale[j & 7] = ManyScale{exp2_int(scale_exp(kj)), float(ev), exp2_int(-ev), 1.f};
              mbar_arrive_expect_tx(bar, 2 * kCacheTile);
              const size_t from = (size_t(at) * c.kv_heads + kh) * kCacheTile;
              bulk_load(dst, c.keys + from, kCacheTile, bar);
              bulk_load(dst + kCacheTile, c.values + from, kCacheTile, bar);
            } else {
              sh.scale[j & 7] = ManyScale{1.f, -INFINITY, 0.f, 0.f};  // a block that is not there: nothing seen
              if (c.status) atomicOr(c.status, WAMFFN_DEV_BAD_INDEX);
              mbar_arrive_local(bar);
            }
            sent = j + 1;
          }
        }
        ok = warp_verdict(ok);
        if (!ok) break;
        if (++r == kManyRaw) r = 0, ph ^= 1u;
      }
      if (lane == 0 && *abort)  // copies in flight land before the shared memory is given up
        for (int j = max(0, sent - kManyRaw); j < sent; ++j)
          wait_drain(smem_addr(&sh.raw_full[j % kManyRaw]), uint32_t(j / kManyRaw) & 1u);
    }
    __syncwarp();
    if (split > 1) {  // the softmax warps' two cluster barriers
      cluster_sync();
      cluster_sync();
    }
  } else if (warp < kManySoftmaxWarp0) {
    // ------------------------------------------------------------ e4m3 -> f16
    set_registers<kManyConvRegs>();
    // Thread: 16 bytes `chunk` (dims 16 chunk ..) of rows r0 + 16 i, 32 bytes of operand half chunk / 4.  Lanes of
    // the upper dims store their second half first: eight neighbouring lanes then meet eight different 16-byte
    // columns of the swizzle.
    const int tid = threadIdx.x - kManyConvWarp0 * 32;
    const int chunk = tid & 7, r0 = tid >> 3, upper = chunk >> 2, column = 2 * (chunk & 3);
    int s = 0, r = 0;                    // operand stage, raw block
    uint32_t parity = 1u, raw_ph = 0u;   // of the stage's last use; of the block
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      const int key0 = (first + j) * kManyStep;
      if (lane == 0) {
        ok = wait_spin(smem_addr(&sh.raw_full[r]), raw_ph, abort, c.status, WAMFFN_DEV_TIMEOUT);
        if (ok && j >= stages)  // the products of step j - stages have read the stage
          ok = wait_spin(smem_addr(&sh.empty[s]), parity, abort, c.status, WAMFFN_DEV_TIMEOUT);
      }
      ok = warp_verdict(ok);
      if (!ok) break;
      const bool there = sh.scale[j & 7].there != 0.f;
      const uint32_t src = smem_addr(raw_block(r) + r0 * kCacheDim + chunk * 16);
      uint4 raw[2][4];
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          raw[w][i] = there ? lds128(src + w * kCacheTile + i * 16 * kCacheDim) : make_uint4(0, 0, 0, 0);
      if (key0 + kManyStep > least) {  // some row sees less than the whole step
#pragma unroll
        for (int i = 0; i < 4; ++i)
          raw[1][i] = clean_chunk(raw[1][i], key0 + r0 + 16 * i, length, least < most, 16 * chunk, sh.nan_key, &sh.nan_any);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_local(smem_addr(&sh.raw_empty[r]));
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint8_t* dst = operand(w, s) + upper * kManyHalf;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 u = raw[w][i];
          const int row = r0 + 16 * i;
          const uint32_t a = upper ? u.z : u.x, z = upper ? u.w : u.y, a2 = upper ? u.x : u.z, z2 = upper ? u.y : u.w;
          *reinterpret_cast<uint4*>(dst + sw128_offset(row, column + upper)) =
              make_uint4(e4m3x2_to_f16x2(a), e4m3x2_hi_to_f16x2(a), e4m3x2_to_f16x2(z), e4m3x2_hi_to_f16x2(z));
          *reinterpret_cast<uint4*>(dst + sw128_offset(row, column + 1 - upper)) =
              make_uint4(e4m3x2_to_f16x2(a2), e4m3x2_hi_to_f16x2(a2), e4m3x2_to_f16x2(z2), e4m3x2_hi_to_f16x2(z2));
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(smem_addr(&sh.full[s]));
      if (++s == stages) s = 0, parity ^= 1u;
      if (++r == kManyRaw) r = 0, raw_ph ^= 1u;
    }
    __syncwarp();
    if (split > 1) {
      cluster_sync();
      cluster_sync();
    }
  } else {
    // ------------------------------------------------------------ softmax
    set_registers<kManySoftmaxRegs>();
    const int r = threadIdx.x - kManySoftmaxWarp0 * 32, x = (warp - kManySoftmaxWarp0) >> 2;  // row of 256; tile
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t to = tmem + kManyO + x * 128 + lanes;
    const int rr = dual ? r & 127 : r;
    const bool live = rr < rows;
    const int row = row0 + (live ? rr : 0), token = row / p.group, head = kh * p.group + row - token * p.group;
    const int seen = live ? keys_seen(length, p.nq, token, p.causal) : 0;
    bool ok = true;
    float qf;
    {  // this row of Q: largest magnitude, power of two, f16, operand tile
      const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.q_batch + token * p.q_row + size_t(head) * kCacheDim);
      uint32_t u[64];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint4 w = live ? src[i] : make_uint4(0, 0, 0, 0);
        u[4 * i] = w.x, u[4 * i + 1] = w.y, u[4 * i + 2] = w.z, u[4 * i + 3] = w.w;
      }
#pragma unroll
      for (int i = 0; i < 64; ++i) top = fmaxf(top, fmaxf(fabsf(bf2_lo(u[i])), fabsf(bf2_hi(u[i]))));
      const int eq = query_exp(top);
      const float inv = exp2_int(-eq);
      qf = exp2_int(eq) * p.scale_log2;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = f16x2_pack(bf2_lo(u[4 * i + e]) * inv, bf2_hi(u[4 * i + e]) * inv);
        *reinterpret_cast<uint4*>(query(x) + (i >> 3) * (kManyQuery / 2) + sw128_offset(r & 127, i & 7)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(smem_addr(&sh.q_full));
    }
    float m = -INFINITY, l = 0.f;
    const int mine = dual ? (steps - x + 1) / 2 : steps;  // steps of this tile
    {
      for (int n = 0; n < mine; ++n) {
        const int j = dual ? 2 * n + x : n;
        const uint32_t ts = tmem + x * 128 + (n & 1) * 64 + lanes;
        if (lane == 0)
          ok = wait_spin(smem_addr(&sh.s_full[x][n & 1]), uint32_t(n >> 1) & 1u, abort, c.status, WAMFFN_DEV_TIMEOUT);
        ok = warp_verdict(ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld32(ts, v[0]);
        tmem_ld32(ts + 32, v[1]);
        const ManyScale sc = sh.scale[j & 7];
        const int key0 = (first + j) * kManyStep;
        tmem_wait_ld(v[0]);
        tmem_wait_ld(v[1]);
        // Some row of the CTA sees less than the whole step, or no row sees a block that is not there (its zeros
        // would be NaN to a query of NaN).
        if (key0 + kManyStep > least || sc.there == 0.f) {
          const int limit = sc.there == 0.f ? 0 : seen - key0;
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= limit) v[i >> 5][i & 31] = 0xff800000u;  // -inf
        }
        // The row's maximum, of S (its factor is positive) and so of x.
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            t[e] = fmaxf(fmaxf(t[e], __uint_as_float(v[i >> 5][(i & 31) + 2 * e])),
                         __uint_as_float(v[i >> 5][(i & 31) + 2 * e + 1]));
        const float u = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        const float f = fminf(qf * sc.kf, FLT_MAX);  // finite: a product of zero stays zero
        // A block that is not there has ev -inf; nothing seen leaves u at -inf.
        const float top = u == -INFINITY ? -INFINITY : fmaf(u, f, sc.ev);
        // The first maximum needs no correction; one that grows by at most 2^kLag is left as it is.
        if (m == -INFINITY) m = top;
        const bool apart = top > m + kLag || (top < m - kDeep && top > -INFINITY);
        const bool rare = __any_sync(0xffffffffu, apart);
        const float ref = apart ? top : m;
        const float base = sc.ev - (ref == -INFINITY ? 0.f : ref) + kPBias;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t out[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const uint32_t a = v[i >> 4][2 * (i & 15)], z = v[i >> 4][2 * (i & 15) + 1];
          float2 e = fma2(make_float2(__uint_as_float(a), __uint_as_float(z)), f, base);
          e.x = ex2_approx(e.x);
          e.y = ex2_approx(e.y);
          sum[i & 1] = add2(sum[i & 1], e);
          out[i] = f16x2_pack(e.x, e.y);
        }
        float back = sc.back, corr = 1.f;
        if (rare) {
          if (apart) {
            const bool grown = top > m;
            const float fold = ex2_approx(0.5f * (grown ? m - top : top - m - sc.ev));
            if (grown) {
              corr = fold * fold;
              l = folded(l, fold);
              m = top;
            } else {  // deep: the sum alone gets these (kvattend.cuh)
              back = fold;
              sum[0] = make_float2((sum[0].x + sum[1].x) * fold, (sum[0].y + sum[1].y) * fold);
              sum[1] = make_float2(0.f, 0.f);
#pragma unroll
              for (int i = 0; i < 32; ++i) out[i] = 0u;
            }
          }
          __syncwarp();
        }
        tmem_st32(ts, out);
        l = fmaf((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y), back, l);
        if (rare && __any_sync(0xffffffffu, corr != 1.f)) {  // not in the first step: m was new
          if (lane == 0)
            ok = wait_spin(smem_addr(&sh.o_step[x]), uint32_t(n - 1) & 1u, abort, c.status, WAMFFN_DEV_TIMEOUT);
          ok = warp_verdict(ok);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
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
        if (lane == 0) mbar_arrive_local(smem_addr(&sh.p_full[x][n & 1]));
      }
    }
    if (ok) {
      // Both tiles: the operands' place is reused below, by a CTA without steps too (every warp's Q is written then).
      if (lane == 0) {
        ok = wait_spin(smem_addr(&sh.q_full), 0u, abort, c.status, WAMFFN_DEV_TIMEOUT);
        for (int y = 0; y < 2; ++y)
          if ((dual ? y : 0) < steps)
            ok = ok && wait_spin(smem_addr(&sh.o_last[y]), 0u, abort, c.status, WAMFFN_DEV_TIMEOUT);
      }
      ok = warp_verdict(ok);
      tc_fence_after();
    }
    // 32 dims of this row's O; a NaN that was cleaned out of a value this row sees comes back.
    auto load_o = [&](int q, uint32_t (&v)[32]) {
      if (mine > 0) {
        tmem_ld32(to + q * 32, v);
        tmem_wait_ld(v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0u;
      }
      if (sh.nan_any)
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (sh.nan_key[q * 32 + i] < seen) v[i] = 0x7fffffffu;
    };
    float* held = reinterpret_cast<float*>(smem);  // rows of O; every product has read the operands that lay there
    float2* held_ml = reinterpret_cast<float2*>(held + kManyRows * kManyPitch);
    auto place = [&](int at, int d) { return reinterpret_cast<float4*>(held + at * kManyPitch + d); };
    auto emit = [&](int q, const uint32_t (&v)[32], float inv) {  // 32 dims of a row that is complete in this CTA
      if (p.parts > 1) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          kv_emit(p, part, b, token, head, q * 32 + i,
                  make_float4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]),
                              __uint_as_float(v[i + 3])), m, l);
      } else {
        __nv_bfloat16* dst = p.out + ((size_t(b) * p.nq + token) * p.heads + head) * kCacheDim + q * 32;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(v[i + e]) * inv;
          *reinterpret_cast<uint4*>(dst + i) =
              make_uint4(bf2_pack(o[0], o[1]), bf2_pack(o[2], o[3]), bf2_pack(o[4], o[5]), bf2_pack(o[6], o[7]));
        }
      }
    };
    float f = 1.f;
    if (dual) {
      // The two tiles' shares of a row: each hands half of the dims to the other and adds what it gets to its half.
      held_ml[r] = make_float2(m, l);
      __syncwarp();
      named_sync(1, kManySoftmaxWarps * 32);
      const float2 e0 = held_ml[rr], e1 = held_ml[rr + 128];
      const float top = fmaxf(e0.x, e1.x), safe = top == -INFINITY ? 0.f : top;
      const float h0 = ex2_approx(0.5f * (e0.x - safe)), h1 = ex2_approx(0.5f * (e1.x - safe));
      f = x ? h1 * h1 : h0 * h0;
      m = top;
      l = folded(e0.y, h0) + folded(e1.y, h1);
#pragma unroll 1
      for (int q = x ? 0 : 2, n = 0; n < 2; ++n, ++q) {
        uint32_t v[32];
        load_o(q, v);
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *place(rr, q * 32 + i) = make_float4(__uint_as_float(v[i]) * f, __uint_as_float(v[i + 1]) * f,
                                               __uint_as_float(v[i + 2]) * f, __uint_as_float(v[i + 3]) * f);
      }
      __syncwarp();
      named_sync(1, kManySoftmaxWarps * 32);
    }
    if (dual) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int q = x ? 2 : 0, n = 0; n < 2; ++n, ++q) {
        uint32_t v[32];
        load_o(q, v);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 o = *place(rr, q * 32 + i);
          v[i] = __float_as_uint(fmaf(__uint_as_float(v[i]), f, o.x));
          v[i + 1] = __float_as_uint(fmaf(__uint_as_float(v[i + 1]), f, o.y));
          v[i + 2] = __float_as_uint(fmaf(__uint_as_float(v[i + 2]), f, o.z));
          v[i + 3] = __float_as_uint(fmaf(__uint_as_float(v[i + 3]), f, o.w));
          if (split > 1) *reinterpret_cast<uint4*>(place(rr, q * 32 + i)) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        if (split == 1 && live && ok) emit(q, v, inv);
      }
      if (split > 1 && x == 0) held_ml[rr] = make_float2(m, l);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
      if (split > 1) held_ml[r] = make_float2(m, l);
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
        uint32_t v[32];
        load_o(q, v);
        if (split == 1) {
          if (live && ok) emit(q, v, inv);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(place(r, q * 32 + i)) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
    }
    if (split > 1) {
      // The cluster's shares of the rows, in rank order; rank k takes rows k, k + split, ...
      __syncwarp();
      cluster_sync();
      const int pieces = ((rows - rank + split - 1) / split) * (kCacheDim / 4);
      auto merge = [&](auto batch) {  // pieces of a thread whose eight loads are in flight together
        constexpr int kBatch = decltype(batch)::value, kShares = 8 / kBatch;
        for (int i0 = r; i0 < pieces; i0 += kBatch * kManySoftmaxWarps * 32) {
          float4 u[kBatch][kShares];
          float2 ml[kBatch][kShares];
#pragma unroll
          for (int n = 0; n < kBatch; ++n) {
            const int i = i0 + n * kManySoftmaxWarps * 32, at = rank + (i >> 5) * split;
            const uint32_t ml_at = smem_addr(&held_ml[at]), o_at = smem_addr(place(at, (i & 31) * 4));
#pragma unroll
            for (int k = 0; k < kShares; ++k) {
              ml[n][k] = make_float2(-INFINITY, 0.f);
              u[n][k] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (k < split && i < pieces) {
                ml[n][k] = ld_cluster2(map_to_cta(ml_at, k));
                u[n][k] = ld_cluster4(map_to_cta(o_at, k));
              }
            }
          }
#pragma unroll
          for (int n = 0; n < kBatch; ++n) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < kShares; ++k) top = fmaxf(top, ml[n][k].x);
            const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int k = 0; k < kShares; ++k) {
              const float fold = ex2_approx(0.5f * (ml[n][k].x - safe)), fk = fold * fold;
              v.x += u[n][k].x * fk, v.y += u[n][k].y * fk, v.z += u[n][k].z * fk, v.w += u[n][k].w * fk;
              sum += folded(ml[n][k].y, fold);
            }
            const int i = i0 + n * kManySoftmaxWarps * 32, prow = row0 + rank + (i >> 5) * split;
            const int ptoken = prow / p.group, phead = kh * p.group + prow - ptoken * p.group;
            if (i < pieces && !*abort) kv_emit(p, part, b, ptoken, phead, (i & 31) * 4, v, top, sum);
          }
        }
      };
      if (split == 2)
        merge(std::integral_constant<int, 4>{});
      else if (split <= 4)
        merge(std::integral_constant<int, 2>{});
      else
        merge(std::integral_constant<int, 1>{});
      __syncwarp();
      cluster_sync();  // no CTA leaves while a peer reads its shared memory
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace wamffn
