// Norm of queries and keys with the position rotation in the same pass: what a
// DiT (or any transformer with a query / key norm) runs between its QKV
// projection and its attention (WAMInfer/_triton_inference.py:13-112 is the
// reference's form for whole rows).
//
//   r = rsqrt(mean(x^2) + eps)        over one head (weight of D) or the whole row (weight of H D)
//   y = x r w
//   (y[a], y[b]) <- (y[a] c - y[b] s, y[a] s + y[b] c),   c + i s = rope[position, pair]
//
// with (a, b) = (2i, 2i+1) (interleaved, a complex view of the head) or
// (i, i + R) (halves), i < R <= D / 2; dims past 2 R are not turned.  All of it
// in fp32, rounded to bf16 once (the reference rounds after the norm, after the
// weight and after the rotation; one rounding is nearer to the formula).
//
// Bound: HBM, 4 bytes an element: 2 x 8191 tokens of 32 + 8 heads take 54.0 us on a
// B200, 97 % of its measured copy bandwidth, norm of each head (up to 8 heads a
// group of lanes; 59 us with 4, 74 us with 2: fewer loads in flight, the table's
// entries and addresses made for fewer heads); with the norm over the row 90 us, 59 %
// (a CTA a token, whose loads wait for the one block-wide sum).  One token takes 3 us:
// latency.  A lane holds 8 dims of a head in registers (16 bytes in, 16 out) as two
// runs of 4, laid so that both members of every pair are in the lane: the rotation
// needs no exchange.  A lane keeps its dims for all the heads it visits, so its 4 table
// entries are read once.  A sum of squares past fp32's range (values beyond some 1e18)
// is infinite, and the row or head zeros.
#pragma once

#include "ptx.cuh"

namespace wamffn {

struct RopeSide {  // queries or keys
  const __nv_bfloat16* x;
  long long row_stride, batch_stride;  // elements
  const __nv_bfloat16* weight;
  __nv_bfloat16* y;                    // [batch, rows, heads D], contiguous
  int heads;
};

struct RopeParams {
  RopeSide q, k;
  const float2* rope;          // [table_rows, table_stride], null: no rotation
  long long table_stride;      // complex elements between table rows
  const void* positions;       // int32 / int64, null: the row's index
  long long position_stride;   // elements between batches
  int position_bytes;
  int table_rows, pairs, rows, batch;
  float eps;
};

// A lane's 8 dims: runs of 4 at `a` and `b` within the head, pairs [pair, pair + 4) turned.
struct RopeDims {
  int a, b, pair;
  bool turned;
};

template <bool kInterleaved>
__device__ __forceinline__ RopeDims rope_dims(int j, int pairs) {
  RopeDims d;
  d.pair = 4 * j;
  d.turned = 4 * j < pairs;
  d.a = (kInterleaved || !d.turned) ? 8 * j : 4 * j;
  d.b = (kInterleaved || !d.turned) ? 8 * j + 4 : pairs + 4 * j;
  return d;
}

// Position of token t of batch b; a position outside the table gives -1.
__device__ __forceinline__ long long rope_position(const RopeParams& p, int b, int t) {
  long long at = t;
  if (p.positions) {
    const long long i = (long long)b * p.position_stride + t;
    at = p.position_bytes == 8 ? static_cast<const long long*>(p.positions)[i]
                               : (long long)static_cast<const int*>(p.positions)[i];
  }
  return at >= 0 && at < p.table_rows ? at : -1;
}

// cos, sin of a turned lane's pairs; NaN for a position outside the table, from which nothing is read (the norm's
// factor is NaN there too, for the dims that are not turned).
__device__ __forceinline__ void rope_load(const RopeParams& p, const RopeDims& d, long long at, float (&c)[4],
                                          float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
  if (at >= 0 && d.turned) {
    const float4* src = reinterpret_cast<const float4*>(p.rope + at * p.table_stride + d.pair);
    const float4 u = src[0], v = src[1];
    c[0] = u.x, s[0] = u.y, c[1] = u.z, s[1] = u.w;
    c[2] = v.x, s[2] = v.y, c[3] = v.z, s[3] = v.w;
  }
}

template <bool kInterleaved>
__device__ __forceinline__ uint4 rope_ld(const __nv_bfloat16* head, const RopeDims& d) {
  if constexpr (kInterleaved) return *reinterpret_cast<const uint4*>(head + d.a);
  const uint2 u = *reinterpret_cast<const uint2*>(head + d.a), v = *reinterpret_cast<const uint2*>(head + d.b);
  return make_uint4(u.x, u.y, v.x, v.y);
}

__device__ __forceinline__ void rope_unpack(const uint4& u, float (&x)[8]) {
  x[0] = bf2_lo(u.x), x[1] = bf2_hi(u.x), x[2] = bf2_lo(u.y), x[3] = bf2_hi(u.y);
  x[4] = bf2_lo(u.z), x[5] = bf2_hi(u.z), x[6] = bf2_lo(u.w), x[7] = bf2_hi(u.w);
}

__device__ __forceinline__ float rope_squares(const uint4& u) {
  float x[8], s = 0.f;
  rope_unpack(u, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
  return s;
}

// x r w, turned, rounded and stored.  `w` as rope_ld laid it out.
template <bool kInterleaved>
__device__ __forceinline__ void rope_store(__nv_bfloat16* head, const RopeDims& d, const uint4& u, const float (&w)[8],
                                           float r, const float (&c)[4], const float (&s)[4]) {
  float x[8], y[8];
  rope_unpack(u, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= r * w[i];
  // Pairs inside the lane: (0,1)(2,3)(4,5)(6,7) interleaved, (0,4)(1,5)(2,6)(3,7) in halves.
  // An unturned lane's dims are no pairs: an infinity or NaN of one must not reach the other (0 x inf).
  // (Selects cost 0.3 us in the case above, a branch around the products 1.5.)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = kInterleaved ? 2 * i : i, b = kInterleaved ? 2 * i + 1 : i + 4;
    y[a] = d.turned ? x[a] * c[i] - x[b] * s[i] : x[a];
    y[b] = d.turned ? x[a] * s[i] + x[b] * c[i] : x[b];
  }
  const uint2 lo = make_uint2(bf2_pack(y[0], y[1]), bf2_pack(y[2], y[3]));
  const uint2 hi = make_uint2(bf2_pack(y[4], y[5]), bf2_pack(y[6], y[7]));
  if constexpr (kInterleaved) {
    *reinterpret_cast<uint4*>(head + d.a) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  } else {
    *reinterpret_cast<uint2*>(head + d.a) = lo;
    *reinterpret_cast<uint2*>(head + d.b) = hi;
  }
}

constexpr int kRopeThreads = 128;

// Norm of each head.  A group of D / 8 lanes takes up to kHeads heads of one
// token, all queries' or all keys' (one address and one weight for them), all
// loaded before the first is used.
template <int D, bool kInterleaved, int kHeads>
__global__ void __launch_bounds__(kRopeThreads) rope_head_kernel(const RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kRopeThreads / kLanes;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int q_chunks = (p.q.heads + kHeads - 1) / kHeads, chunks = q_chunks + (p.k.heads + kHeads - 1) / kHeads;
  const uint32_t item = blockIdx.x * kGroups + threadIdx.x / kLanes;
  const int b = blockIdx.y, t = item / uint32_t(chunks), chunk = int(item - uint32_t(t) * chunks);
  if (t >= p.rows) return;  // whole groups leave; the shuffles name their group
  const bool key = chunk >= q_chunks;
  const int heads = key ? p.k.heads : p.q.heads, h0 = (key ? chunk - q_chunks : chunk) * kHeads;
  const int n = min(kHeads, heads - h0);
  const __nv_bfloat16* src = (key ? p.k.x : p.q.x) + b * (key ? p.k.batch_stride : p.q.batch_stride) +
                             t * (key ? p.k.row_stride : p.q.row_stride) + h0 * D;
  __nv_bfloat16* dst = (key ? p.k.y : p.q.y) + (((long long)b * p.rows + t) * heads + h0) * D;
  const RopeDims d = rope_dims<kInterleaved>(threadIdx.x % kLanes, p.pairs);
  const long long at = p.rope ? rope_position(p, b, t) : 0;
  uint4 x[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) x[i] = i < n ? rope_ld<kInterleaved>(src + i * D, d) : make_uint4(0, 0, 0, 0);
  float c[4], s[4], w[8];
  rope_load(p, d, at, c, s);
  rope_unpack(rope_ld<kInterleaved>(key ? p.k.weight : p.q.weight, d), w);
  const uint32_t group = kLanes == 32 ? 0xffffffffu
                                      : ((1u << kLanes) - 1u) << ((threadIdx.x & 31) / kLanes * kLanes);
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (i >= n) break;  // the same for the whole group
    float sum = rope_squares(x[i]);
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) sum += __shfl_xor_sync(group, sum, o);
    const float r = at < 0 ? __int_as_float(0x7fffffff) : rsqrtf(sum * (1.0f / D) + p.eps);
    rope_store<kInterleaved>(dst + i * D, d, x[i], w, r, c, s);
  }
}

// Norm over the whole row.  One CTA a token, queries and keys together (one
// reduction step for both sums); a thread keeps kVec 8-dim vectors, a multiple
// of D / 8 threads apart so that its dims within the head never change.
template <int D, bool kInterleaved, int kVec>
__global__ void __launch_bounds__(512) rope_row_kernel(const RopeParams p) {
  constexpr int kLanes = D / 8;
  __shared__ float part[2][16];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int b = blockIdx.y, t = blockIdx.x;
  const long long token = (long long)b * p.rows + t;
  const RopeDims d = rope_dims<kInterleaved>(threadIdx.x % kLanes, p.pairs);
  const long long at = p.rope ? rope_position(p, b, t) : 0;
  const int heads = p.q.heads + p.k.heads;
  const int first = threadIdx.x / kLanes, step = blockDim.x / kLanes;
  uint4 x[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int h = first + i * step;
    const bool key = h >= p.q.heads;
    const __nv_bfloat16* base = key ? p.k.x + b * p.k.batch_stride + t * p.k.row_stride + (h - p.q.heads) * D
                                    : p.q.x + b * p.q.batch_stride + t * p.q.row_stride + h * D;
    x[i] = h < heads ? rope_ld<kInterleaved>(base, d) : make_uint4(0, 0, 0, 0);
  }
  float c[4], s[4];
  rope_load(p, d, at, c, s);
  float sq = 0.f, sk = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const float v = rope_squares(x[i]);
    if (first + i * step >= p.q.heads)
      sk += v;
    else
      sq += v;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sq += __shfl_xor_sync(0xffffffffu, sq, o);
    sk += __shfl_xor_sync(0xffffffffu, sk, o);
  }
  if ((threadIdx.x & 31) == 0) {
    part[0][threadIdx.x >> 5] = sq;
    part[1][threadIdx.x >> 5] = sk;
  }
  __syncthreads();
  sq = sk = 0.f;
  for (int w = 0; w < int(blockDim.x >> 5); ++w) {
    sq += part[0][w];
    sk += part[1][w];
  }
  const float bad = __int_as_float(0x7fffffff);
  const float rq = at < 0 ? bad : rsqrtf(sq / float(p.q.heads * D) + p.eps);
  const float rk = at < 0 ? bad : rsqrtf(sk / float(max(p.k.heads, 1) * D) + p.eps);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int h = first + i * step;
    if (h >= heads) break;
    const bool key = h >= p.q.heads;
    float w[8];
    rope_unpack(rope_ld<kInterleaved>(key ? p.k.weight + (h - p.q.heads) * D : p.q.weight + h * D, d), w);
    __nv_bfloat16* out = key ? p.k.y + (token * p.k.heads + (h - p.q.heads)) * D : p.q.y + (token * p.q.heads + h) * D;
    rope_store<kInterleaved>(out, d, x[i], w, key ? rk : rq, c, s);
  }
}

}  // namespace wamffn
