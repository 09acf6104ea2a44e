// Attention of one new token per sequence over a paged key / value cache.
//
//   s_j = scale q . k_j,  out = sum_j exp(s_j - m) v_j / l,  l = sum_j exp(s_j - m),  lse = m + ln l
//
// over the keys j < length of the sequence; key j is row j % page_size of page
// table[j / page_size]. A sequence without keys gives 0 and lse = -inf.
//
// Bound: HBM. Every key and value row is read once for the whole group of query
// heads that share it (groups of more than 16 heads load it once per 16 heads), 4 bytes
// per two multiply-adds and head, so the kernel only has to keep enough loads in flight. One warp takes 16 keys at a time and
// reads them straight into matrix-instruction operands; nothing is staged in
// shared memory:
//  * S^T = K Q^T (16 keys x 8 query heads, m16n8k16). The contraction index can
//    be permuted freely, so lane (g, t) reads 16 contiguous bytes of key g (dims
//    32 c + 8 t .. + 7) and uses them as two operand registers of two
//    instructions; Q is held in the same order.
//  * exp(S^T), rounded to 16 bits (the tensor core's operand type; the sum l
//    takes the unrounded values; in fp16 times 2^15, see WeightScale), is transposed in
//    registers (movmatrix).
//  * O^T += V^T P^T: lane (g, t) reads 16 contiguous bytes (dims 8 g .. + 7) of
//    keys 2t, 2t + 1, 2t + 8, 2t + 9 and pairs the keys with byte permutes. The
//    output rows are permuted accordingly; each lane ends with 8 consecutive dims.
// The small M of this work (the group's 1 to 16 heads) would leave a tcgen05
// tile of 128 rows almost empty, and staging through shared memory for it would
// cost what the direct loads save. Measured: 64 sequences of 8,192 keys, 8 key heads
// (2.15 GB): 336 us, 98% of the measured copy bandwidth; one of 250,001 keys, 4 key heads
// (0.51 GB): 85 to 89 us, 88 to 92%.
//
// The length of a sequence is split over CTAs, each with its own m, l and unnormalised O.
// Up to 8 splits are one cluster, where all CTAs fit on the GPU at once: they write theirs
// into the first CTA's shared memory, which joins them (one launch, no workspace). More
// splits (few sequences, long ones) or more CTAs go through a workspace and a second
// kernel: a cluster waits until the SMs of one GPC have room for all of it (64 x 8 key
// heads of 7,000 to 9,000 keys in 8 parts: 376 us in clusters, 338 us through the workspace). Both join in the order of the splits; there
// are no atomics, so the same inputs always give the same bits.
#include <algorithm>

#include "attn_math.cuh"
#include "kernels.h"

namespace h3 {
namespace {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = kDecWarps * 32;
template <bool F16>
using DecodeWeight = WeightScale<F16, 15>;  // the largest weight of a warp's keys so far is 1

struct DecodeParams {
  const uint16_t* q;
  int64_t q_b, q_h;
  const uint16_t* k;
  int64_t k_page, k_head, k_row;
  const uint16_t* v;
  int64_t v_page, v_head, v_row;
  const int32_t* table;
  int64_t t_b, t_h;
  int64_t pages, rows;  // pages of the pool; rows < pages * page_size: the last page is not full
  int width, page_size;
  const int32_t* lengths;
  uint16_t* out;
  int64_t o_b, o_h;
  float* lse;
  int64_t l_b, l_h;
  int heads, kv_heads, group, row_tiles;
  float scale, scale_log2;
  int splits, part_min;
  int clustered;          // the splits of an item are a cluster
  float* ws_acc;
  float2* ws_ml;
};

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ void st_cluster_v2(uint32_t addr, const float2& v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}

// Keys [begin, end) of split `s` of a sequence of `length` keys: even parts of at least
// part_min keys, in whole 16-key steps. Returns the number of parts that hold keys.
__device__ __forceinline__ int split_range(int length, int splits, int part_min, int s, int& begin, int& end) {
  const int n = max(1, min(splits, (length + part_min - 1) / part_min));
  const int per = max(16, ((length + n - 1) / n + 15) / 16 * 16);
  begin = min(length, s * per);
  end = min(length, begin + per);
  return max(1, (length + per - 1) / per);
}

__device__ __forceinline__ int sequence_length(const DecodeParams& p, int b) {
  const int cap = p.width * p.page_size;
  return p.lengths == nullptr ? cap : max(0, min(cap, __ldg(p.lengths + b)));
}

template <bool F16, int NT>
__global__ void __launch_bounds__(kDecThreads, NT == 1 ? 3 : 2) paged_decode_kernel(const DecodeParams p) {
  using E = Elem16<F16>;
  constexpr int R = 8 * NT;
  extern __shared__ __align__(16) float dec_smem[];
  float(*sm_acc)[R][kHeadDim] = reinterpret_cast<float(*)[R][kHeadDim]>(dec_smem);  // [warps]
  float(*sm_m)[R] = reinterpret_cast<float(*)[R]>(dec_smem + kDecWarps * R * kHeadDim);
  float(*sm_l)[R] = sm_m + kDecWarps;
  float(*cl_acc)[R][kHeadDim] = reinterpret_cast<float(*)[R][kHeadDim]>(&sm_l[kDecWarps][0]);  // [splits], clustered
  float2(*cl_ml)[R] = reinterpret_cast<float2(*)[R]>(&cl_acc[p.splits][0][0]);
  if (p.clustered) cluster_arrive();  // first phase: every CTA of the cluster has started
  launch_next();
  wait_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t item = blockIdx.x / p.splits;
  const int split = (int)(blockIdx.x - item * p.splits);
  const int rt = (int)(item % p.row_tiles);
  const int kvh = (int)((item / p.row_tiles) % p.kv_heads);
  const int b = (int)(item / ((int64_t)p.row_tiles * p.kv_heads));
  const int length = sequence_length(p, b);
  int begin, end;
  const int parts = split_range(length, p.splits, p.part_min, split, begin, end);
  if (split >= parts) {
    if (p.clustered) {
      cluster_wait();
      cluster_arrive();
    }
    return;
  }
  const int row0 = rt * R, rows = min(R, p.group - row0), head0 = kvh * p.group + row0;

  uint32_t qf[NT][16];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (n * 8 + g < rows) w = ldg_v4(p.q + b * p.q_b + (head0 + n * 8 + g) * p.q_h + c * 32 + t * 8);
      qf[n][4 * c] = w.x; qf[n][4 * c + 1] = w.y; qf[n][4 * c + 2] = w.z; qf[n][4 * c + 3] = w.w;
    }
  float acc[NT][8][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.0f;
  }
  const int32_t* table = p.table + b * p.t_b + kvh * p.t_h;
  const uint16_t* kb = p.k + kvh * p.k_head;
  const uint16_t* vb = p.v + kvh * p.v_head;

  // page ids of the two 8-key halves of a step (page sizes are multiples of 8), -1: no keys
  auto lookup = [&](int j) { return j < end ? table[j / p.page_size] : -1; };
  int id0 = lookup(begin + warp * 16), id1 = lookup(begin + warp * 16 + 8);
  for (int j = begin + warp * 16; j < end; j += kDecWarps * 16) {
    const int pid[2] = {id0, id1};
    id0 = lookup(j + kDecWarps * 16);
    id1 = lookup(j + kDecWarps * 16 + 8);
    int valid[2];       // keys of each half that exist
    int off[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int jj = j + 8 * h;
      off[h] = jj % p.page_size;
      valid[h] = min(8, end - jj);
      if (pid[h] < 0 || pid[h] >= p.pages)
        valid[h] = 0;  // no page of this pool: nothing is read
      else
        valid[h] = (int)min((int64_t)valid[h], p.rows - ((int64_t)pid[h] * p.page_size + off[h]));
    }
    uint4 kr[2][4], vr[2][2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        kr[h][c] = make_uint4(0u, 0u, 0u, 0u);
        if (g < valid[h]) kr[h][c] = ldg_stream_v4(kb + pid[h] * p.k_page + (off[h] + g) * p.k_row + c * 32 + t * 8);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          // keys that do not exist count as zero rows: 0 * (what lies there) could be NaN
          vr[h][e][d] = make_uint4(0u, 0u, 0u, 0u);
          if (2 * t + e < valid[h])
            vr[h][e][d] = ldg_stream_v4(vb + pid[h] * p.v_page + (off[h] + 2 * t + e) * p.v_row + d * 64 + g * 8);
        }
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        E::mma(s, kr[0][c].x, kr[1][c].x, kr[0][c].y, kr[1][c].y, qf[n][4 * c], qf[n][4 * c + 1]);
        E::mma(s, kr[0][c].z, kr[1][c].z, kr[0][c].w, kr[1][c].w, qf[n][4 * c + 2], qf[n][4 * c + 3]);
      }
      if (g >= valid[0]) s[0] = s[1] = -INFINITY;
      if (g >= valid[1]) s[2] = s[3] = -INFINITY;
      // Weights and rescaling are taken of differences to the maximum: with one fused
      // multiply-add of the score and the scaled maximum, the rounding of that maximum is
      // the largest weight's exponent, and fp16 overflows from scores of 1e7 on.
      float f[2], sub[2];
      bool grew = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(s[e], s[2 + e]);
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
        const float mn = fmaxf(m[n][e], mx);
        sub[e] = mn == -INFINITY ? 0.0f : mn;
        f[e] = mn == m[n][e] ? 1.0f : exp2f((m[n][e] - mn) * p.scale_log2);  // exp2(-inf) = 0 before the first key
        grew = grew || mn > m[n][e];
        m[n][e] = mn;
      }
      if (__any_sync(0xFFFFFFFFu, grew)) {
        l[n][0] *= f[0];
        l[n][1] *= f[1];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[n][i][0] *= f[0];
          acc[n][i][1] *= f[1];
          acc[n][i][2] *= f[0];
          acc[n][i][3] *= f[1];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = exp2f(fmaf(s[e] - sub[e & 1], p.scale_log2, DecodeWeight<F16>::log2));
        l[n][e & 1] += s[e];
      }
      pb[n][0] = movmatrix_trans(E::pack(s[0], s[1]));
      pb[n][1] = movmatrix_trans(E::pack(s[2], s[3]));
    }
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const uint32_t a[4] = {vr[0][0][d].x, vr[0][0][d].y, vr[0][0][d].z, vr[0][0][d].w};
      const uint32_t c[4] = {vr[0][1][d].x, vr[0][1][d].y, vr[0][1][d].z, vr[0][1][d].w};
      const uint32_t x[4] = {vr[1][0][d].x, vr[1][0][d].y, vr[1][0][d].z, vr[1][0][d].w};
      const uint32_t y[4] = {vr[1][1][d].x, vr[1][1][d].y, vr[1][1][d].z, vr[1][1][d].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a0 = __byte_perm(a[i], c[i], 0x5410), a1 = __byte_perm(a[i], c[i], 0x7632);
        const uint32_t a2 = __byte_perm(x[i], y[i], 0x5410), a3 = __byte_perm(x[i], y[i], 0x7632);
#pragma unroll
        for (int n = 0; n < NT; ++n) E::mma(acc[n][d * 4 + i], a0, a1, a2, a3, pb[n][0], pb[n][1]);
      }
    }
  }
  // join the warps: lane (g, t) holds dims 64 d + 8 g + 2 i + {0, 1} of queries 2 t, 2 t + 1
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = l[n][e];
      s += __shfl_xor_sync(0xFFFFFFFFu, s, 4);
      s += __shfl_xor_sync(0xFFFFFFFFu, s, 8);
      s += __shfl_xor_sync(0xFFFFFFFFu, s, 16);
      const int r = n * 8 + 2 * t + e;
      if (g == 0) {
        sm_m[warp][r] = m[n][e];
        sm_l[warp][r] = s;
      }
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 o = make_float4(acc[n][d * 4 + 2 * h][e], acc[n][d * 4 + 2 * h][2 + e],
                                       acc[n][d * 4 + 2 * h + 1][e], acc[n][d * 4 + 2 * h + 1][2 + e]);
          *reinterpret_cast<float4*>(&sm_acc[warp][r][d * 64 + g * 8 + 4 * h]) = o;
        }
    }
  __syncthreads();
  auto store = [&](int r, int d, const float4& o, float mx, float sum) {
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);  // NaN stays
    uint2 y;
    y.x = E::pack(o.x * inv, o.y * inv);
    y.y = E::pack(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(p.out + b * p.o_b + (head0 + r) * p.o_h + d) = y;
    if (d == 0 && p.lse != nullptr)
      p.lse[b * p.l_b + (head0 + r) * p.l_h] = sum == 0.0f ? -INFINITY : fmaf(mx, p.scale, logf(sum * DecodeWeight<F16>::inv));
  };
  if (p.clustered) cluster_wait();
  for (int i = threadIdx.x; i < rows * (kHeadDim / 4); i += kDecThreads) {
    const int r = i / (kHeadDim / 4), d = (i % (kHeadDim / 4)) * 4;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) mx = fmaxf(mx, sm_m[w][r]);
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float f = mx == -INFINITY ? 0.0f : exp2f((sm_m[w][r] - mx) * p.scale_log2);
      const float4 a = *reinterpret_cast<const float4*>(&sm_acc[w][r][d]);
      sum = fmaf(sm_l[w][r], f, sum);
      o.x = fmaf(a.x, f, o.x);
      o.y = fmaf(a.y, f, o.y);
      o.z = fmaf(a.z, f, o.z);
      o.w = fmaf(a.w, f, o.w);
    }
    if (p.clustered) {
      st_cluster_v4(mapa_shared(&cl_acc[split][r][d], 0), o);
      if (d == 0) st_cluster_v2(mapa_shared(&cl_ml[split][r], 0), make_float2(mx, sum));
    } else if (p.splits > 1) {
      const int64_t at = (item * p.splits + split) * R + r;
      *reinterpret_cast<float4*>(p.ws_acc + at * kHeadDim + d) = o;
      if (d == 0) p.ws_ml[at] = make_float2(mx, sum);
    } else {
      store(r, d, o, mx, sum);
    }
  }
  if (!p.clustered) return;
  cluster_arrive();        // second phase: every split is in the first CTA's shared memory
  if (split != 0) return;  // the cluster's CTAs are the item's splits in order
  cluster_wait();
  for (int i = threadIdx.x; i < rows * (kHeadDim / 4); i += kDecThreads) {
    const int r = i / (kHeadDim / 4), d = (i % (kHeadDim / 4)) * 4;
    float mx = -INFINITY;
    for (int s = 0; s < parts; ++s) mx = fmaxf(mx, cl_ml[s][r].x);
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < parts; ++s) {
      const float2 ml = cl_ml[s][r];
      const float f = mx == -INFINITY ? 0.0f : exp2f((ml.x - mx) * p.scale_log2);
      const float4 a = *reinterpret_cast<const float4*>(&cl_acc[s][r][d]);
      sum = fmaf(ml.y, f, sum);
      o.x = fmaf(a.x, f, o.x);
      o.y = fmaf(a.y, f, o.y);
      o.z = fmaf(a.z, f, o.z);
      o.w = fmaf(a.w, f, o.w);
    }
    store(r, d, o, mx, sum);
  }
}

// out = sum_s exp(m_s - m) O_s / sum_s exp(m_s - m) l_s of one (sequence, head) by W warps:
// warp w adds the splits w, w + W, ..., then the warps' sums are added in their order.
// One warp is enough for a few splits; a hundred of them (one long sequence) would be
// a chain of L2 latencies.
template <bool F16, int W>
__global__ void __launch_bounds__(256) decode_join_kernel(const DecodeParams p, int64_t total, int row_tile) {
  using E = Elem16<F16>;
  constexpr int kRows = 8 / W;
  __shared__ float4 sm_o[8][32];
  __shared__ float sm_sum[8], sm_max[8];
  wait_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp % W;
  const int64_t row = (int64_t)blockIdx.x * kRows + warp / W;
  const bool live = row < total;
  const int b = live ? (int)(row / p.heads) : 0, head = live ? (int)(row % p.heads) : 0;
  const int kvh = head / p.group, in_group = head % p.group;
  const int64_t item = ((int64_t)b * p.kv_heads + kvh) * p.row_tiles + in_group / row_tile;
  int begin, end;
  const int parts = live ? split_range(sequence_length(p, b), p.splits, p.part_min, 0, begin, end) : 0;
  const int64_t at = item * p.splits * row_tile + in_group % row_tile;
  float mx = -INFINITY;
  for (int s = w + W * lane; s < parts; s += W * 32) mx = fmaxf(mx, p.ws_ml[at + (int64_t)s * row_tile].x);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, i));
  float sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int s = w; s < parts; s += W) {
    const float2 ml = p.ws_ml[at + (int64_t)s * row_tile];
    const float4 a = *(reinterpret_cast<const float4*>(p.ws_acc + (at + (int64_t)s * row_tile) * kHeadDim) + lane);
    const float f = mx == -INFINITY ? 0.0f : exp2f((ml.x - mx) * p.scale_log2);
    sum = fmaf(ml.y, f, sum);
    o.x = fmaf(a.x, f, o.x);
    o.y = fmaf(a.y, f, o.y);
    o.z = fmaf(a.z, f, o.z);
    o.w = fmaf(a.w, f, o.w);
  }
  if constexpr (W > 1) {
    sm_o[warp][lane] = o;
    if (lane == 0) {
      sm_sum[warp] = sum;
      sm_max[warp] = mx;
    }
    __syncthreads();
    if (w != 0) return;
    float all = -INFINITY;
#pragma unroll
    for (int i = 0; i < W; ++i) all = fmaxf(all, sm_max[warp + i]);
    sum = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float f = all == -INFINITY ? 0.0f : exp2f((sm_max[warp + i] - all) * p.scale_log2);
      const float4 a = sm_o[warp + i][lane];
      sum = fmaf(sm_sum[warp + i], f, sum);
      o.x = fmaf(a.x, f, o.x);
      o.y = fmaf(a.y, f, o.y);
      o.z = fmaf(a.z, f, o.z);
      o.w = fmaf(a.w, f, o.w);
    }
    mx = all;
  }
  if (!live) return;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  uint2 y;
  y.x = E::pack(o.x * inv, o.y * inv);
  y.y = E::pack(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(p.out + b * p.o_b + head * p.o_h + lane * 4) = y;
  if (lane == 0 && p.lse != nullptr)
    p.lse[b * p.l_b + head * p.l_h] = sum == 0.0f ? -INFINITY : fmaf(mx, p.scale, logf(sum * DecodeWeight<F16>::inv));
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int kPartMin = 64;     // keys: one 16-key step of each warp
constexpr int kPartGood = 512;   // keys whose reading outweighs a part's own cost by far
// Parts of each sequence where the items alone fill the GPU: 64 x 8 key heads of 7,000 to
// 9,000 keys take 330 us in 4, 338 in 8, 358 in 12 parts; 48 x 8 of 0 to 6,000 keys 114,
// 113 and 123. The number of parts comes from the shape alone, so one long sequence
// among short ones runs on its few parts long after the others have ended: 250,001 keys
// beside 63 sequences of 100 to 2,000 take 1,476 us, where the bytes alone take 199.
constexpr int kTailParts = 4;
constexpr int kMaxSplits = 512;
constexpr int kClusterMax = 8;   // portable cluster size

int row_tile_of(int64_t group) { return group <= 8 ? 8 : 16; }

int64_t decode_items(int64_t batch, int64_t heads, int64_t kv_heads) {
  const int64_t group = heads / kv_heads, tile = row_tile_of(group);
  return batch * kv_heads * ((group + tile - 1) / tile);
}

bool clustered(int64_t items, int64_t splits, int sms) {
  return splits > 1 && splits <= kClusterMax && items * splits <= 2 * sms;
}

}  // namespace

int paged_decode_splits(int64_t batch, int64_t heads, int64_t kv_heads, int64_t max_keys, int sms) {
  const int64_t group = heads / kv_heads;
  const int64_t items = decode_items(batch, heads, kv_heads);
  const int64_t slots = (int64_t)sms * (row_tile_of(group) == 8 ? 3 : 2);  // CTAs the GPU holds at once
  // Few items: as many parts as fit at once (a part more would wait for a whole one), down
  // to one step per warp. Many items, of lengths only the GPU knows: parts short enough
  // that the last ones to finish are a small part of the work.
  const int64_t most = std::max<int64_t>(1, (max_keys + kPartMin - 1) / kPartMin);
  const int64_t good = std::min<int64_t>(kTailParts, std::max<int64_t>(1, max_keys / kPartGood));
  const int64_t n = std::min<int64_t>(kMaxSplits, std::min(most, std::max<int64_t>(slots / items, good)));
  // short sequences: a cluster's longer parts cost less than a second kernel
  return (int)(max_keys <= kClusterMax * kPartGood ? std::min<int64_t>(n, kClusterMax) : n);
}

int64_t paged_decode_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t max_keys, int sms) {
  const int64_t splits = paged_decode_splits(batch, heads, kv_heads, max_keys, sms);
  const int64_t items = decode_items(batch, heads, kv_heads);
  if (splits == 1 || clustered(items, splits, sms)) return 0;
  const int64_t rows = items * splits * row_tile_of(heads / kv_heads);
  return rows * (kHeadDim * 4 + 8);
}

cudaError_t check_paged_decode(const PagedDecodeArgs& a) {
  if (!aligned(a.q) || a.q_b % 8 || a.q_h % 8 || !aligned(a.k) || a.k_page % 8 || a.k_head % 8 || a.k_row % 8 ||
      !aligned(a.v) || a.v_page % 8 || a.v_head % 8 || a.v_row % 8 || !aligned(a.out) || a.o_b % 8 || a.o_h % 8)
    return cudaErrorNotSupported;
  int dev = 0;
  cudaGetDevice(&dev);
  const int splits = paged_decode_splits(a.batch, a.heads, a.kv_heads, a.width * a.page_size, num_sms(dev));
  return decode_items(a.batch, a.heads, a.kv_heads) * splits > 0x7FFFFFFF ? cudaErrorNotSupported : cudaSuccess;
}

cudaError_t launch_paged_decode(const PagedDecodeArgs& a, cudaStream_t stream) {
  if (a.batch <= 0) return cudaSuccess;
  const cudaError_t refused = check_paged_decode(a);
  if (refused != cudaSuccess) return refused;
  DecodeParams p;
  p.q = static_cast<const uint16_t*>(a.q); p.q_b = a.q_b; p.q_h = a.q_h;
  p.k = static_cast<const uint16_t*>(a.k); p.k_page = a.k_page; p.k_head = a.k_head; p.k_row = a.k_row;
  p.v = static_cast<const uint16_t*>(a.v); p.v_page = a.v_page; p.v_head = a.v_head; p.v_row = a.v_row;
  p.table = a.table; p.t_b = a.t_b; p.t_h = a.t_h;
  p.pages = a.pages; p.rows = a.rows; p.width = (int)a.width; p.page_size = (int)a.page_size;
  p.lengths = a.lengths;
  p.out = static_cast<uint16_t*>(a.out); p.o_b = a.o_b; p.o_h = a.o_h;
  p.lse = a.lse; p.l_b = a.l_b; p.l_h = a.l_h;
  p.heads = (int)a.heads; p.kv_heads = (int)a.kv_heads; p.group = (int)(a.heads / a.kv_heads);
  const int tile = row_tile_of(p.group);
  p.row_tiles = (p.group + tile - 1) / tile;
  p.scale = a.scale;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  int dev = 0;
  cudaGetDevice(&dev);
  p.splits = paged_decode_splits(a.batch, a.heads, a.kv_heads, a.width * a.page_size, num_sms(dev));
  p.part_min = kPartMin;
  const int64_t items = decode_items(a.batch, a.heads, a.kv_heads);
  p.clustered = clustered(items, p.splits, num_sms(dev));
  p.ws_acc = static_cast<float*>(a.workspace);
  p.ws_ml = reinterpret_cast<float2*>(p.ws_acc + items * p.splits * tile * kHeadDim);
  const unsigned grid = (unsigned)(items * p.splits);
  auto kernel = a.f16 ? (tile == 8 ? paged_decode_kernel<true, 1> : paged_decode_kernel<true, 2>)
                      : (tile == 8 ? paged_decode_kernel<false, 1> : paged_decode_kernel<false, 2>);
  const size_t warps_smem = (size_t)kDecWarps * tile * (kHeadDim + 2) * 4;
  const size_t smem = warps_smem + (p.clustered ? (size_t)p.splits * tile * (kHeadDim + 2) * 4 : 0);
  static bool attr_set[64][4] = {};
  bool* set = dev >= 0 && dev < 64 ? &attr_set[dev][(a.f16 ? 2 : 0) + (tile == 8 ? 0 : 1)] : nullptr;
  if (set == nullptr || !*set) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    if (e != cudaSuccess) return e;
    if (set) *set = true;
  }
  const cudaError_t e = launch_chained(kernel, grid, kDecThreads, smem, stream, a.chained, p.clustered ? p.splits : 1, p);
  if (e != cudaSuccess || p.splits == 1 || p.clustered) return e;
  const int64_t total = a.batch * a.heads;
  if (p.splits > 8)
    return launch_chained(a.f16 ? decode_join_kernel<true, 8> : decode_join_kernel<false, 8>, (unsigned)total, 256, 0,
                          stream, true, 1, p, total, tile);
  return launch_chained(a.f16 ? decode_join_kernel<true, 1> : decode_join_kernel<false, 1>, (unsigned)((total + 7) / 8),
                        256, 0, stream, true, 1, p, total, tile);
}

}  // namespace h3
