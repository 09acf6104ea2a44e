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
// the latency of one chain slot -> address -> store.
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

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? __ldg(static_cast<const long long*>(p) + i) : (int64_t)__ldg(static_cast<const int*>(p) + i);
}

// coefficients (own, partner) of rotation pair `pair`: row 0 of [[t00, t01], [t10, t11]] for
// the first half of the rotated dims (own t00, partner t01), row 1 for the second (own t11)
__device__ __forceinline__ void load_coef(const void* table, int dtype, int64_t base, int pair, int second, float& own,
                                          float& other) {
  const int64_t at = base + pair * 4 + second * 2;
  float a, b;
  if (dtype == 0) {
    a = __ldg(static_cast<const float*>(table) + at);
    b = __ldg(static_cast<const float*>(table) + at + 1);
  } else {
    const uint16_t* t = static_cast<const uint16_t*>(table) + at;
    const uint32_t w = (uint32_t)__ldg(t) | ((uint32_t)__ldg(t + 1) << 16);
    a = dtype == 1 ? Elem16<false>::lo(w) : Elem16<true>::lo(w);
    b = dtype == 1 ? Elem16<false>::hi(w) : Elem16<true>::hi(w);
  }
  own = second ? b : a;
  other = second ? a : b;
}

template <bool F16>
__global__ void __launch_bounds__(kAppendThreads) append_paged_kv_kernel(const AppendParams p) {
  using E = Elem16<F16>;
  const int64_t warp = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int64_t token = warp / p.chunks;
  if (token >= p.tokens) return;
  const int chunk = (int)(warp - token * p.chunks);
  const int64_t slot = load_index(p.slot_of, p.slot64, token);
  if (slot < 0 || slot >= p.slots) return;  // padding: nothing of this token is written
  const int half = (threadIdx.x >> 4) & 1, l = threadIdx.x & 15;
  const int nq = p.q_out != nullptr ? p.heads : 0;
  const int rows = nq + 2 * p.kv_heads;
  const int begin = chunk * p.rows_per_warp, end = min(rows, begin + p.rows_per_warp);
  if (begin >= end) return;

  const int step = p.rot >> 4;  // lanes of half the rotated dims
  const bool rotated = l < 2 * step;
  const int second = l >= step ? 1 : 0;
  const int partner = rotated ? (second ? l - step : l + step) : l;
  float ca[8], cb[8];
  if (rotated && begin < nq + p.kv_heads) {
    const int64_t row = p.position_of == nullptr ? token : load_index(p.position_of, p.position64, token);
    const bool known = row >= 0 && row < p.table_rows;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ca[i] = cb[i] = __int_as_float(0x7FC00000);  // a position outside the table: NaN, not a wrong rotation
      if (known) load_coef(p.table, p.table_dtype, row * p.table_stride, (l - second * step) * 8 + i, second, ca[i], cb[i]);
    }
  }
  const int64_t page = slot / p.page_size, row_in_page = slot - page * p.page_size;

  for (int r0 = begin; r0 < end; r0 += 2 * kAppendUnroll) {
    uint4 x[kAppendUnroll];
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      const int r = r0 + 2 * u + half;
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < end) {
        const int which = r < nq ? 0 : (r < nq + p.kv_heads ? 1 : 2);
        const int head = which == 0 ? r : r - nq - (which - 1) * p.kv_heads;
        x[u] = ldg_v4(p.x[which] + token * p.xs_t[which] + head * p.xs_h[which] + l * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < kAppendUnroll; ++u) {
      const int r = r0 + 2 * u + half;
      if (r0 + 2 * u >= end) break;  // warp-uniform: the shuffles below see both halves
      const int which = r < nq ? 0 : (r < nq + p.kv_heads ? 1 : 2);
      const int head = which == 0 ? r : r - nq - (which - 1) * p.kv_heads;
      uint32_t own[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, other[4];
      float f[8], g[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        other[i] = __shfl_sync(0xFFFFFFFFu, own[i], partner, 16);
        f[2 * i] = E::lo(own[i]);
        f[2 * i + 1] = E::hi(own[i]);
      }
      const uint16_t* w = which < 2 ? p.w[which] : nullptr;
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
      for (int i = 8; i > 0; i >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, i, 16);
      if (r >= end) continue;
      if (which < 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[2 * i] = E::lo(other[i]);
          g[2 * i + 1] = E::hi(other[i]);
        }
        if (w != nullptr) {
          const float rstd = rsqrtf(ss * (1.0f / kHeadDim) + p.eps);
          const uint4 wo = __ldg(reinterpret_cast<const uint4*>(w + l * 8));
          const uint4 wp = __ldg(reinterpret_cast<const uint4*>(w + partner * 8));
          const uint32_t wow[4] = {wo.x, wo.y, wo.z, wo.w}, wpw[4] = {wp.x, wp.y, wp.z, wp.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[2 * i] *= rstd * E::lo(wow[i]);
            f[2 * i + 1] *= rstd * E::hi(wow[i]);
            g[2 * i] *= rstd * E::lo(wpw[i]);
            g[2 * i + 1] *= rstd * E::hi(wpw[i]);
          }
        }
        if (rotated) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = fmaf(ca[i], f[i], cb[i] * g[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) own[i] = E::pack(f[2 * i], f[2 * i + 1]);
      }
      uint16_t* y;
      if (which == 0)
        y = p.q_out + token * p.qo_t + head * p.qo_h;
      else
        y = p.cache[which - 1] + page * p.c_page[which - 1] + head * p.c_head[which - 1] + row_in_page * p.c_row[which - 1];
      stg_v4(y + l * 8, make_uint4(own[0], own[1], own[2], own[3]));
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
  // runs as long as the token (coefficients read once) when the tokens alone give every
  // SM its 32 warps, shorter ones, down to one row per half-warp, when they do not
  const int64_t want = (int64_t)num_sms(dev) * 32;
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
