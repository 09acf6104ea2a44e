// Appending keys and values to a paged cache, with the per-head RMSNorm and the
// split-half rotation of K (and of Q beside it) on the way.
//
//   h = x / sqrt(mean(x^2) + eps) * w            (without a weight: h = x)
//   y[i]         = t00 h[i] + t01 h[i + r / 2]
//   y[i + r / 2] = t10 h[i] + t11 h[i + r / 2]   (i < r / 2);  y[i] = h[i] for i >= r
//   k_cache[slot / page_size, head, slot % page_size] = y_k, v likewise, q_out[token] = y_q
//
// Everything between the load and the store is fp32 and rounded once, at the
// store (the in-place norm-RoPE kernels of this library also round h, as the
// reference they reproduce does; nothing here has such a reference, and the
// second rounding would only cost accuracy).
//
// Layout: a half-warp owns one 128-wide head row as 16 lanes x 16 bytes. A
// lane's rotation partner is r / 16 lanes away; it sends its raw packed words
// (4 shuffles) and the receiver applies the norm to them, because the row's
// 1 / rms is known to both. A warp stays with one token for a run of its rows
// (Q heads, K heads, V heads in that order), so the token's slot, position and
// rotation coefficients are read once per run.
//
// Bound: HBM, each row read once and written once. A long prompt gives every
// token one warp. With few tokens the rows of a token are dealt out over more
// warps (down to one row per half-warp), since a call on one token is bound by
// the latency of one chain slot -> address -> store. What it takes to keep HBM busy is
// loads in flight: at 102 registers (5 CTAs an SM) 32,760 tokens of 72 rows take 268 us, at
// 80 (6 CTAs) with the first rows' loads ahead of the coefficients 219 us, with the rest of
// a run's Q or K rows prefetched into L2 205 us (6.06 TB/s, 93% of the measured copy). One
// step of prefetching ahead instead of the run's gives 209; Q, K and V rows of the token at
// once, or before its slot is known, 244.
#include <algorithm>

#include "attn_math.cuh"
#include "kernels.h"

namespace h3 {
namespace {

constexpr int kAppendThreads = 128;
constexpr int kAppendUnroll = 4;  // rows in flight per half-warp

struct AppendParams {
  const uint16_t* x[3];  // q, k, v
  int64_t xs_t[3], xs_h[3];
  uint16_t* q_out;
  int64_t qo_t, qo_h;
  uint16_t* cache[2];  // k, v
  int64_t c_page[2], c_head[2], c_row[2];
  int64_t slots;  // pages * page_size
  int64_t page_size;
  const void* slot_of;
  const void* position_of;
  int slot64, position64;
  const void* table;
  int table_dtype;
  int64_t table_rows, table_stride;
  const uint16_t* w[2];  // q, k norm weights or nullptr
  int64_t tokens;
  int heads, kv_heads, rot;
  int rows_per_warp, chunks;
  float eps;
};

__device__ __forceinline__ void prefetch_l2(const void* p, int bytes) {  // both multiples of 16
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes));
}

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? __ldg(static_cast<const long long*>(p) + i) : (int64_t)__ldg(static_cast<const int*>(p) + i);
}

// coefficients (own, partner) of 8 rotation pairs from `pair` on: row 0 of [[t00, t01], [t10, t11]]
// for the first half of the rotated dims (own t00, partner t01), row 1 for the second
// (own t11). Rows are at least 4 elements apart, so a pair's two values load as one word.
__device__ __forceinline__ void load_coefs(const void* table, int dtype, int64_t base, int pair, int second,
                                           float (&own)[8], float (&other)[8]) {
  const int64_t at = base + pair * 4 + second * 2;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a, b;
    if (dtype == 0) {
      const float2 v = __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(table) + at + 4 * i));
      a = v.x;
      b = v.y;
    } else {
      const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(table) + at + 4 * i));
      a = dtype == 1 ? Elem16<false>::lo(w) : Elem16<true>::lo(w);
      b = dtype == 1 ? Elem16<false>::hi(w) : Elem16<true>::hi(w);
    }
    own[i] = second ? b : a;
    other[i] = second ? a : b;
  }
}

// Rows [lo, hi) of the token's Q or K heads: y = rstd (A x + B x_partner) with the norm
// weights folded into the rotation coefficients A, B once per run.
template <bool F16>
__device__ __forceinline__ void turn_rows(const uint16_t* src, int64_t src_h, uint16_t* dst,
                                          int64_t dst_h, int lo, int hi, const uint16_t* w, float eps, bool rotated,
                                          int partner, const float (&ca)[8], const float (&cb)[8]) {
  using E = Elem16<F16>;
  const int half = (threadIdx.x >> 4) & 1, l = threadIdx.x & 15;
  uint4 x[kAppendUnroll];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      const int r = r0 + 2 * u + half;
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < hi) x[u] = ldg_v4(src + r * src_h);
    }
  };
  load(lo);  // on the way while the coefficients arrive
  // and the rest of the run on its way to L2, one row per lane
  for (int r = lo + 2 * kAppendUnroll + (threadIdx.x & 31); r < hi; r += 32)
    prefetch_l2(src - l * 8 + r * src_h, kHeadDim * 2);
  uint64_t a2[4], b2[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a0 = ca[2 * i], a1 = ca[2 * i + 1], b0 = cb[2 * i], b1 = cb[2 * i + 1];
    if (w != nullptr) {
      const uint32_t wo = __ldg(reinterpret_cast<const uint32_t*>(w + l * 8) + i);
      const uint32_t wp = __ldg(reinterpret_cast<const uint32_t*>(w + partner * 8) + i);
      a0 *= E::lo(wo);
      a1 *= E::hi(wo);
      b0 *= E::lo(wp);
      b1 *= E::hi(wp);
    }
    a2[i] = f2_pack(a0, a1);
    b2[i] = f2_pack(b0, b1);
  }
  for (int r0 = lo; r0 < hi; r0 += 2 * kAppendUnroll) {
    if (r0 > lo) load(r0);
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      if (r0 + 2 * u >= hi) break;  // warp-uniform: the shuffles below see both halves
      const int r = r0 + 2 * u + half;
      uint32_t own[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
      uint64_t f[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t other = __shfl_sync(0xFFFFFFFFu, own[i], partner, 16);
        if (!rotated) other = 0u;  // B is 0 there; 0 * inf must not be
        f[i] = f2_pack(E::lo(own[i]), E::hi(own[i]));
        y[i] = f2_fma(a2[i], f[i], f2_mul(b2[i], f2_pack(E::lo(other), E::hi(other))));
      }
      if (w != nullptr) {
        uint64_t s = 0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) s = f2_fma(f[i], f[i], s);
        float s0, s1;
        f2_unpack(s, s0, s1);
        s0 += s1;
#pragma unroll
        for (int i = 8; i > 0; i >>= 1) s0 += __shfl_xor_sync(0xFFFFFFFFu, s0, i, 16);
        const float rstd = rsqrtf(s0 * (1.0f / kHeadDim) + eps);
        const uint64_t rr = f2_pack(rstd, rstd);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = f2_mul(y[i], rr);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        f2_unpack(y[i], a, b);
        own[i] = E::pack(a, b);
      }
      if (r < hi) stg_v4(dst + r * dst_h, make_uint4(own[0], own[1], own[2], own[3]));
    }
  }
}

template <bool F16>
__global__ void __launch_bounds__(kAppendThreads, 6) append_paged_kv_kernel(const AppendParams p) {
  const int64_t warp = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int64_t token = warp / p.chunks;
  if (token >= p.tokens) return;
  const int chunk = (int)(warp - token * p.chunks);
  const int64_t slot = load_index(p.slot_of, p.slot64, token);
  int64_t position = token;
  if (p.position_of != nullptr) position = load_index(p.position_of, p.position64, token);
  if (slot < 0 || slot >= p.slots) return;  // padding: nothing of this token is written
  const int half = (threadIdx.x >> 4) & 1, l = threadIdx.x & 15;
  const int nq = p.q_out != nullptr ? p.heads : 0, nk = nq + p.kv_heads;
  const int begin = chunk * p.rows_per_warp, end = min(nk + p.kv_heads, begin + p.rows_per_warp);

  const int64_t page = slot / p.page_size, row_in_page = slot - page * p.page_size;
  if (begin < nk) {
    const int step = p.rot >> 4;  // lanes of half the rotated dims
    const bool rotated = l < 2 * step;
    const int second = l >= step ? 1 : 0;
    const int partner = rotated ? (second ? l - step : l + step) : l;
    float ca[8], cb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ca[i] = 1.0f;
      cb[i] = 0.0f;
    }
    if (rotated) {
      const int64_t row = position;
      const bool known = row >= 0 && row < p.table_rows;
      if (known)
        load_coefs(p.table, p.table_dtype, row * p.table_stride, (l - second * step) * 8, second, ca, cb);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) ca[i] = cb[i] = __int_as_float(0x7FC00000);  // NaN, not a wrong rotation
    }
    if (begin < nq)
      turn_rows<F16>(p.x[0] + token * p.xs_t[0] + l * 8, p.xs_h[0], p.q_out + token * p.qo_t + l * 8, p.qo_h, begin,
                     min(end, nq), p.w[0], p.eps, rotated, partner, ca, cb);
    if (end > nq)
      turn_rows<F16>(p.x[1] + token * p.xs_t[1] + l * 8, p.xs_h[1],
                     p.cache[0] + page * p.c_page[0] + row_in_page * p.c_row[0] + l * 8, p.c_head[0],
                     max(begin, nq) - nq, min(end, nk) - nq, p.w[1], p.eps, rotated, partner, ca, cb);
  }
  if (end > nk) {
    const uint16_t* src = p.x[2] + token * p.xs_t[2] + l * 8;
    uint16_t* dst = p.cache[1] + page * p.c_page[1] + row_in_page * p.c_row[1] + l * 8;
    for (int r0 = max(begin, nk) - nk; r0 < end - nk; r0 += 4 * kAppendUnroll) {
      uint4 x[2 * kAppendUnroll];
#pragma unroll
      for (int u = 0; u < 2 * kAppendUnroll; ++u)
        if (r0 + 2 * u + half < end - nk) x[u] = ldg_v4(src + (r0 + 2 * u + half) * p.xs_h[2]);
#pragma unroll
      for (int u = 0; u < 2 * kAppendUnroll; ++u)
        if (r0 + 2 * u + half < end - nk) stg_v4(dst + (r0 + 2 * u + half) * p.c_head[1], x[u]);
    }
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

cudaError_t launch_append_paged_kv(const AppendKvArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  AppendParams p;
  const void* xs[3] = {a.q, a.k, a.v};
  for (int i = a.q ? 0 : 1; i < 3; ++i)
    if (!aligned(xs[i]) || a.xs_t[i] % 8 || a.xs_h[i] % 8) return cudaErrorNotSupported;
  if (a.q && (!aligned(a.q_out) || a.qo_t % 8 || a.qo_h % 8)) return cudaErrorNotSupported;
  // a rotation pair's coefficients are read two at a time
  if (a.table && ((reinterpret_cast<uintptr_t>(a.table) & (a.table_dtype == 0 ? 7 : 3)) || a.table_stride % 2))
    return cudaErrorNotSupported;
  for (int i = 0; i < 2; ++i) {
    if (!aligned(a.cache[i]) || a.c_page[i] % 8 || a.c_head[i] % 8 || a.c_row[i] % 8 || !aligned(a.w[i]))
      return cudaErrorNotSupported;
    p.cache[i] = static_cast<uint16_t*>(a.cache[i]);
    p.c_page[i] = a.c_page[i]; p.c_head[i] = a.c_head[i]; p.c_row[i] = a.c_row[i];
    p.w[i] = static_cast<const uint16_t*>(a.w[i]);
  }
  for (int i = 0; i < 3; ++i) {
    p.x[i] = static_cast<const uint16_t*>(xs[i]);
    p.xs_t[i] = a.xs_t[i]; p.xs_h[i] = a.xs_h[i];
  }
  p.q_out = a.q ? static_cast<uint16_t*>(a.q_out) : nullptr;
  p.qo_t = a.qo_t; p.qo_h = a.qo_h;
  p.slots = a.pages * a.page_size;
  p.page_size = a.page_size;
  p.slot_of = a.slot_of; p.slot64 = a.slot64;
  p.position_of = a.position_of; p.position64 = a.position64;
  p.table = a.table; p.table_dtype = a.table_dtype; p.table_rows = a.table_rows; p.table_stride = a.table_stride;
  p.tokens = a.tokens; p.heads = (int)a.heads; p.kv_heads = (int)a.kv_heads; p.rot = (int)a.rot;
  p.eps = a.eps;
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t rows = (a.q ? a.heads : 0) + 2 * a.kv_heads;
  // Runs as long as the token (coefficients read once) when the tokens alone give every SM
  // 96 warps, four rounds of what it holds; shorter ones, down to one row per half-warp,
  // when they do not. 4,095 tokens x 168 rows: 82 us with 64 warps, 74 with 96, 78 with 128.
  const int64_t want = (int64_t)num_sms(dev) * 96;
  const int64_t chunks = std::min<int64_t>((rows + 1) / 2, std::max<int64_t>(1, (want + a.tokens - 1) / a.tokens));
  p.rows_per_warp = (int)(((rows + chunks - 1) / chunks + 1) / 2 * 2);
  p.chunks = (int)((rows + p.rows_per_warp - 1) / p.rows_per_warp);
  const int64_t warps = a.tokens * p.chunks;
  const int64_t blocks = (warps + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (blocks > 0x7FFFFFFF) return cudaErrorNotSupported;
  if (a.f16)
    append_paged_kv_kernel<true><<<(unsigned)blocks, kAppendThreads, 0, stream>>>(p);
  else
    append_paged_kv_kernel<false><<<(unsigned)blocks, kAppendThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace h3
