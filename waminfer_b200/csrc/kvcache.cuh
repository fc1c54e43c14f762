// Keys and values held in 8 bits: blocks of 64 tokens, e4m3 values, one scale
// for each block and head (no counterpart in the reference, whose cached
// prefix is bf16: WAMInfer/_triton_attention.py:337-484).
//
//   keys, values   [blocks, kv_heads, 64, 128] e4m3: a (block, head) tile is one contiguous 8 KB run
//   scales         [blocks, kv_heads] fp32, 2^e;  a row is value * scale
//   block_table    [batch, width]: the block of rows [64 i, 64 i + 64) of a sequence
//   lengths        [batch]: rows held
//
// The scale is a power of two, the least with max|x| <= 448 * 2^e over the
// block's finite values (e >= -60): e4m3 is a floating format, so a finer scale
// would buy no precision, only up to one more binade above its smallest normal
// value; in return x / 2^e and a change of scale are exact shifts, and
// the attention folds the scales into its exponents.
// Bound: HBM, 3 bytes an element to store and to read back.  2 x 8001 rows of 24
// heads stored and read take 101 us on a B200, 90 % of its measured copy
// bandwidth; 16 single tokens 5.2 us, latency (two launches).  Rows start on
// their way before the block ids are checked (with the checks first 139 us), and a
// reading thread has two rows in flight (one: 105 us, four: 105 us).
#pragma once

#include "ptx.cuh"
#include "wamffn.h"

namespace wamffn {

constexpr int kCacheBlock = 64;   // tokens of a block
constexpr int kCacheDim = 128;    // head dim
constexpr int kCacheTile = kCacheBlock * kCacheDim;  // bytes of a (block, head) tile
// A scale's exponent: from -60 (the store's floor; 2^eq 2^ek of a query and a block stays normal) to 126 (its
// reciprocal is a normal number; the store never makes more than 120).
constexpr int kCacheLeastExp = -60, kCacheMostExp = 126;

struct CacheView {
  uint8_t *keys, *values;
  float *key_scales, *value_scales;
  const int* table;
  long long table_stride;
  int* lengths;
  int* tickets;
  unsigned int* status;
  int blocks, kv_heads, batch, width;
};

// Two e4m3 values (low byte first) as f16x2, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(two));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t two) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(d) : "r"(two));
  return d;
}
__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) {
  float2 f;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}"
      : "=f"(f.x), "=f"(f.y)
      : "r"(h));
  return f;
}
// Four fp32 values rounded to e4m3 (to nearest even; beyond 448, infinities too, to 448; NaN stays), low byte first.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// 2^e, -126 <= e <= 127.
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }
// The exponent of a stored scale (a power of two; infinities and NaN count as the largest).
__device__ __forceinline__ int scale_exp(float s) {
  return max(kCacheLeastExp, min(kCacheMostExp, ((__float_as_int(s) >> 23) & 255) - 127));
}
// e(block) from the largest finite |x| as bf16 bits: the least e with |x| <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int cache_exp(uint32_t bits) {
  return max(kCacheLeastExp, int(bits >> 7) - 127 - 8 + int((bits & 127u) > 96u));
}
// Larger of `top` and the magnitudes of two bf16 values; infinities and NaN do not count.
__device__ __forceinline__ uint32_t finite_max(uint32_t top, uint32_t two) {
  const uint32_t lo = two & 0x7fffu, hi = (two >> 16) & 0x7fffu;
  top = max(top, lo < 0x7f80u ? lo : 0u);
  return max(top, hi < 0x7f80u ? hi : 0u);
}

struct AppendParams {
  CacheView c;
  const __nv_bfloat16 *k, *v;
  long long k_row, k_batch, v_row, v_batch;  // strides, elements
  const int *counts, *at;                    // null: rows / lengths
  int rows, places;                          // places: blocks that a sequence's rows may touch
};

constexpr int kAppendThreads = 128;

// One CTA a (touched block, head, batch) of the keys or of the values (neighbouring
// CTAs take neighbouring heads of the same rows, which lie side by side in k and v): largest
// magnitude of its new rows, scale, conversion.  The rows that the block holds
// already are rewritten only where its scale grows.  A sequence whose rows do not
// fit (past its table, behind a gap, through a block id outside the pool) is left
// as it is, and the status word gets WAMFFN_DEV_BAD_INDEX.
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const AppendParams p) {
  __shared__ uint32_t tops[kAppendThreads / 32];
  pdl_wait_prior();
  pdl_launch_dependents();
  const CacheView& c = p.c;
  const int b = blockIdx.y, place = blockIdx.x / (2 * c.kv_heads), side = blockIdx.x % (2 * c.kv_heads);
  const bool value = side >= c.kv_heads;
  const int h = value ? side - c.kv_heads : side;
  const int tid = threadIdx.x;
  const int length = c.lengths[b];
  const long long at = p.at ? p.at[b] : length;
  const long long count = p.counts ? max(0, min(p.counts[b], p.rows)) : p.rows;
  const long long end = at + count;
  const long long first = at / kCacheBlock, low = (first + place) * kCacheBlock;  // the block's first row in the sequence
  bool good = at >= 0 && at <= length && end <= (long long)c.width * kCacheBlock;
  const int* table = c.table + b * c.table_stride;
  const int lo = int(max(at - low, 0ll)), hi = good ? int(max(min(end - low, (long long)kCacheBlock), 0ll)) : 0;  // new rows
  // The rows are on their way while the block ids are looked over.
  const __nv_bfloat16* x = value ? p.v + b * p.v_batch + h * kCacheDim : p.k + b * p.k_batch + h * kCacheDim;
  const long long stride = value ? p.v_row : p.k_row;
  const int lane = tid & 15;       // 8 dims of a row
  constexpr int kStep = kAppendThreads / 16, kPer = kCacheBlock / kStep;
  uint4 u[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = lo + (tid >> 4) + i * kStep;
    u[i] = r < hi ? *reinterpret_cast<const uint4*>(x + (low + r - at) * stride + lane * 8) : make_uint4(0, 0, 0, 0);
  }
  if (good)
    for (long long i = first + tid; i * kCacheBlock < end; i += kAppendThreads) {
      const int id = table[i];
      good = good && id >= 0 && id < c.blocks;
    }
  good = __syncthreads_and(good);
  // The last CTA of a sequence to have read its length writes the new one (in flight while the rows are stored).
  int ticket = -1;
  if (tid == 0) {
    if (!good && c.status) atomicOr(c.status, WAMFFN_DEV_BAD_INDEX);
    ticket = atomicAdd(&c.tickets[b], 1);
  }
  auto leave = [&]() {
    if (ticket == int(gridDim.x) - 1) {
      c.tickets[b] = 0;
      if (good) c.lengths[b] = int(end);
    }
  };
  if (!good || count == 0 || low >= end) return leave();
  const size_t tile = size_t(table[first + place]) * c.kv_heads + h;
  uint8_t* codes = (value ? c.values : c.keys) + tile * kCacheTile;
  float* scale = (value ? c.value_scales : c.key_scales) + tile;
  const int held = lo > 0 ? scale_exp(*scale) : kCacheLeastExp;  // the block's scale, while it holds rows
  // Magnitudes of bf16 order as their bits do: the largest of each half, two instructions a pair; infinities and NaN
  // (bits from 0x7f80 up) send a thread through the pairs once more.
  uint32_t pair = 0, top = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    pair = __vmaxu2(__vmaxu2(__vmaxu2(pair, u[i].x & 0x7fff7fffu), u[i].y & 0x7fff7fffu),
                    __vmaxu2(u[i].z & 0x7fff7fffu, u[i].w & 0x7fff7fffu));
  top = max(pair & 0xffffu, pair >> 16);
  if (top >= 0x7f80u) {
    top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      top = finite_max(finite_max(finite_max(finite_max(top, u[i].x), u[i].y), u[i].z), u[i].w);
  }
  __syncwarp();
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) top = max(top, tops[w]);
  const int e = max(held, cache_exp(top));
  const float inv = exp2_int(-e);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = lo + (tid >> 4) + i * kStep;
    if (r < hi)
      *reinterpret_cast<uint2*>(codes + r * kCacheDim + lane * 8) =
          make_uint2(e4m3x4(bf2_lo(u[i].x) * inv, bf2_hi(u[i].x) * inv, bf2_lo(u[i].y) * inv, bf2_hi(u[i].y) * inv),
                     e4m3x4(bf2_lo(u[i].z) * inv, bf2_hi(u[i].z) * inv, bf2_lo(u[i].w) * inv, bf2_hi(u[i].w) * inv));
  }
  if (lo > 0 && e > held) {  // the held rows take the new scale
    const float f = held - e < -126 ? 0.f : exp2_int(held - e);
    for (int r = tid >> 4; r < lo; r += kStep) {
      uint2* at8 = reinterpret_cast<uint2*>(codes + r * kCacheDim + lane * 8);
      const uint2 o = *at8;
      const float2 a = f16x2_to_float2(e4m3x2_to_f16x2(o.x)), a2 = f16x2_to_float2(e4m3x2_hi_to_f16x2(o.x));
      const float2 z = f16x2_to_float2(e4m3x2_to_f16x2(o.y)), z2 = f16x2_to_float2(e4m3x2_hi_to_f16x2(o.y));
      *at8 = make_uint2(e4m3x4(a.x * f, a.y * f, a2.x * f, a2.y * f), e4m3x4(z.x * f, z.y * f, z2.x * f, z2.y * f));
    }
  }
  if (tid == 0) *scale = exp2_int(e);
  leave();
}

struct CacheReadParams {
  CacheView c;
  const int* start;  // null: start_all
  int start_all, count;
  __nv_bfloat16 *k, *v;  // [batch, count, kv_heads 128]
};

constexpr int kReadThreads = 256;
constexpr int kReadPer = 2;                                  // rows of a thread, all loaded before the first is stored
constexpr int kReadRows = kReadThreads / 8 * kReadPer;       // rows of one head a CTA

// Rows back as bf16 (exact: 4 significant bits times a power of two); zeros past
// a sequence's length.  8 lanes a row: 16 bytes in, 32 out.
__global__ void __launch_bounds__(kReadThreads) cache_read_kernel(const CacheReadParams p) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const CacheView& c = p.c;
  const int b = blockIdx.y, side = blockIdx.x % (2 * c.kv_heads);  // as the store: heads side by side
  const bool value = side >= c.kv_heads;
  const int h = value ? side - c.kv_heads : side;
  const int i0 = int(blockIdx.x / (2 * c.kv_heads)) * kReadRows + (threadIdx.x >> 3), lane = threadIdx.x & 7;
  const long long start = p.start ? p.start[b] : p.start_all;
  const long long end = min((long long)c.lengths[b], (long long)c.width * kCacheBlock);
  uint4 u[kReadPer];
  float s[kReadPer];
#pragma unroll
  for (int k = 0; k < kReadPer; ++k) {
    const int i = i0 + k * (kReadThreads / 8);
    const long long row = start + i;
    u[k] = make_uint4(0, 0, 0, 0);
    s[k] = 0.f;
    if (i < p.count && row >= 0 && row < end) {
      const int id = c.table[b * c.table_stride + row / kCacheBlock];
      if (id >= 0 && id < c.blocks) {
        const size_t tile = size_t(id) * c.kv_heads + h;
        s[k] = (value ? c.value_scales : c.key_scales)[tile];
        u[k] = *reinterpret_cast<const uint4*>((value ? c.values : c.keys) + tile * kCacheTile +
                                               (row % kCacheBlock) * kCacheDim + lane * 16);
      } else if (c.status && lane == 0) {
        atomicOr(c.status, WAMFFN_DEV_BAD_INDEX);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kReadPer; ++k) {
    const int i = i0 + k * (kReadThreads / 8);
    if (i >= p.count) return;
    const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
    const float scale = exp2_int(scale_exp(s[k]));  // a row that is not there: zero times this
    uint32_t out[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = f16x2_to_float2(e4m3x2_to_f16x2(w[j])), z = f16x2_to_float2(e4m3x2_hi_to_f16x2(w[j]));
      out[2 * j] = bf2_pack(a.x * scale, a.y * scale);
      out[2 * j + 1] = bf2_pack(z.x * scale, z.y * scale);
    }
    uint4* dst = reinterpret_cast<uint4*>((value ? p.v : p.k) + (size_t(b) * p.count + i) * c.kv_heads * kCacheDim +
                                          size_t(h) * kCacheDim + lane * 16);
    dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
    dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
  }
}

}  // namespace wamffn
