// Selection of key blocks for block-sparse attention: block means, scores, top-k.
//
//   m[h, b]     = fp32(mean of the rows of block b of head h)
//   score[i, j] = sum over the query heads h of a key head's group of m_q[h, i] . m_k[j]
//   the top_k highest scores of each row i; equal scores go to the lowest j; ascending output
//
// A selection is a whole-number result: two scores that differ in their last bits
// should not change places from one implementation (or one summation order) to
// another. Sums and products are therefore held in 64 bits. A block's sum of 16-bit
// values is exact there unless they span more than some 35 binary places, and the
// product of two fp32 means is exact; that of a sum over grouped heads is rounded. What
// is left is an error of about 1e-16 of the score's terms: scores closer than that can
// change places, those of equal means cannot (every block's are summed in one order). In
// 32 bits (1e-7) about one selection in 10^4 changes with the order of the sum.
//
// Measured (24 heads, 32,760 tokens, L2 full of written lines): means of 201 MB 57 us (3.5
// TB/s; 49 with sums in 32 bits, so most of it is the reads and the write-back beside them;
// prefetching the next CTA's rows, 8 CTAs per SM or shorter unrolls change nothing),
// 24 x 256 x 512 scores and the 64 best of each row 74 us (64-bit matrix instructions 20 us
// of it at their rate; the rest is loads and the descent through the keys' bits, latencies
// that the CTAs of an SM only partly hide).
// Beside the 1.5 ms of the attention they select for, both were left there.
//
// With `causal` (query row r stands at position r + keys - queries), a query
// block sees the key blocks that start no later than its last row. Those that
// hold one of its own positions, whose means cover keys behind some of its rows,
// are not scored: they come before all others.
#include <algorithm>

#include "attn_math.cuh"
#include "kernels.h"

namespace h3 {
namespace {

constexpr int kMeanThreads = 128;  // 8 half-warps, one block row each at a time
constexpr int kMeanUnroll = 8;     // rows in flight per half-warp

struct MeanSource {
  const uint16_t* x;
  int64_t x_t, x_h, tokens, blocks;
  int heads, block;
  float* means;
};

// One CTA per (block, head) of two tensors (the second may be empty). A half-warp reads
// a 256-byte row as 16 lanes x 16 bytes.
// HBM-bound in principle; the loads of a 64-key block are few, so what counts is how
// many small CTAs an SM holds. Consecutive CTAs take consecutive heads of the same tokens.
template <bool F16>
__global__ void __launch_bounds__(kMeanThreads, 6) block_means_kernel(const MeanSource first, const MeanSource second) {
  using E = Elem16<F16>;
  __shared__ double part[kMeanThreads / 32][kHeadDim];
  launch_next();
  const int hw = threadIdx.x >> 4, l = threadIdx.x & 15, warp = threadIdx.x >> 5;
  const int64_t ctas = first.blocks * first.heads;
  const bool of_first = (int64_t)blockIdx.x < ctas;
  const MeanSource& src_of = of_first ? first : second;
  const int64_t cta = of_first ? blockIdx.x : blockIdx.x - ctas;
  const int64_t b = cta / src_of.heads;
  const int h = (int)(cta - b * src_of.heads);
  const int64_t t0 = b * src_of.block, x_t = src_of.x_t;
  const int rows = (int)min((int64_t)src_of.block, src_of.tokens - t0);
  double s[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
  const uint16_t* src = src_of.x + h * src_of.x_h + t0 * x_t + l * 8;
  for (int r0 = hw; r0 < rows; r0 += kMeanThreads / 16 * kMeanUnroll) {
    uint4 v[kMeanUnroll];
#pragma unroll
    for (int u = 0; u < kMeanUnroll; ++u) {
      const int r = r0 + u * (kMeanThreads / 16);
      v[u] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) v[u] = ldg_nc_v4(src + r * x_t);
    }
#pragma unroll
    for (int u = 0; u < kMeanUnroll; ++u) {
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[2 * i] += (double)E::lo(w[i]);
        s[2 * i + 1] += (double)E::hi(w[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] += __shfl_xor_sync(0xFFFFFFFFu, s[i], 16);
  if ((threadIdx.x & 31) < 16) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) *reinterpret_cast<double2*>(&part[warp][l * 8 + i]) = make_double2(s[i], s[i + 1]);
  }
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kMeanThreads / 32; ++i) sum += part[i][threadIdx.x];
  src_of.means[((int64_t)h * src_of.blocks + b) * kHeadDim + threadIdx.x] = (float)(sum / (double)rows);
}
static_assert(kMeanThreads == kHeadDim, "one thread per dim finishes a mean");

constexpr int kSelThreads = 256;
constexpr int kSelHeld = 16;  // high words a lane keeps in registers during the descent (512 key blocks)
constexpr int kSelPad = kHeadDim + 2;  // doubles per staged query row: conflict-free 16-byte reads
constexpr int kSelRows = 8;  // query blocks per CTA: the M of one 64-bit matrix instruction; one warp each for the top-k

// c[8 x 8] += a[8 x 4] b[4 x 8] in 64 bits
__device__ __forceinline__ void mma_f64(double (&c)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
               : "+d"(c[0]), "+d"(c[1])
               : "d"(a), "d"(b));
}

__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// 64-bit key whose unsigned order is the order of the scores; 0 stands for "not to be
// selected". NaN scores rank below every number.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (!(s == s)) return 1ull << 32;
  if (s == 0.0) s = 0.0;  // -0 and +0 are equal
  const unsigned long long b = (unsigned long long)__double_as_longlong(s);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);  // -inf gives 0x000FF..F, above 1
}

// One CTA scores `rows` query blocks of one key head against all key blocks (64-bit
// products of the fp32 means, the query means summed over the group first), then one
// warp per query block finds the top_k-th highest key by descending through its bits
// and emits the selected blocks in ascending order.
//
// Scores: a warp takes 8 key blocks at a time, m8n8k4 in 64 bits. The contraction index
// is permuted so that lane (g, t) reads 16 contiguous bytes of key block g (dims
// 16 c + 4 t .. + 3) and uses them in four instructions; the 8 query rows are read from
// shared memory in the same order (in registers they would halve the CTAs per SM).
//
// Few query blocks leave most SMs idle, and one CTA takes as long for one row as for
// eight: then a cluster of `ctas` CTAs scores a row's key blocks, each a part of them,
// into the first CTA's shared memory.
//
// Keys are kept as their high and low words: the high ones (20 bits of the mantissa)
// nearly always decide alone.
__global__ void __launch_bounds__(kSelThreads) select_blocks_kernel(const float* qm,
                                                                    const float* km, int64_t km_h,
                                                                    int64_t km_b, int group,
                                                                    int64_t q_blocks, int k_blocks, int top_k,
                                                                    int rows_per_cta, int block, int64_t queries,
                                                                    int64_t keys, int causal,
                                                                    int32_t* __restrict__ out,
                                                                    int32_t* __restrict__ out_tiles,
                                                                    const uint16_t* __restrict__ q_row,
                                                                    int64_t q_row_h, int q_row_f16, int ctas) {
  extern __shared__ __align__(16) unsigned char sel_smem[];
  double* qs = reinterpret_cast<double*>(sel_smem);                          // [kSelRows][kSelPad]
  const int pitch = (k_blocks + 3) & ~3;
  uint32_t* key_hi = reinterpret_cast<uint32_t*>(qs + kSelRows * kSelPad);   // [rows][pitch], 0 behind the last block
  uint32_t* key_lo = key_hi + rows_per_cta * pitch;
  if (ctas > 1) cluster_arrive();  // first phase: every CTA of the cluster has started
  launch_next();
  wait_previous();
  const int64_t tiles = (q_blocks + rows_per_cta - 1) / rows_per_cta;
  const int64_t cta = blockIdx.x / ctas;
  const int rank = (int)(blockIdx.x - cta * ctas);
  const int64_t kvh = cta / tiles;
  const int64_t i0 = (cta - kvh * tiles) * rows_per_cta;
  const int rows = (int)min((int64_t)rows_per_cta, q_blocks - i0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  static_assert(kSelThreads == kSelRows * 32, "one warp sums a row's query heads");
  {
    double s[kHeadDim / 32] = {};
    if (warp < rows) {
#pragma unroll 4
      for (int g = 0; g < group; ++g) {
        const int64_t h = kvh * group + g;
        if (q_row != nullptr) {  // one query: it is its own mean
          const uint16_t* x = q_row + h * q_row_h + lane;
#pragma unroll
          for (int e = 0; e < kHeadDim / 32; ++e) {
            const uint32_t w = __ldg(x + 32 * e);
            s[e] += (double)(q_row_f16 ? Elem16<true>::lo(w) : Elem16<false>::lo(w));
          }
        } else {
          const float* x = qm + (h * q_blocks + i0 + warp) * kHeadDim + lane;
#pragma unroll
          for (int e = 0; e < kHeadDim / 32; ++e) s[e] += (double)x[32 * e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kHeadDim / 32; ++e) qs[warp * kSelPad + lane + 32 * e] = s[e];
  }
  for (int e = threadIdx.x; e < rows * (pitch - k_blocks); e += kSelThreads) {
    const int r = e / (pitch - k_blocks);
    key_hi[r * pitch + k_blocks + e - r * (pitch - k_blocks)] = 0u;
  }
  __syncthreads();
  {
    const int g = lane >> 2, t = lane & 3;
    const double2* a = reinterpret_cast<const double2*>(qs + g * kSelPad + 4 * t);
    const float* base = km + kvh * km_h + 4 * t;
    constexpr int warps = kSelThreads / 32;
    const uint32_t hi0 = ctas > 1 ? mapa_shared(key_hi, 0) : 0u, lo0 = ctas > 1 ? mapa_shared(key_lo, 0) : 0u;
    if (ctas > 1) cluster_wait();
    for (int j0 = (rank * warps + warp) * 8; j0 < k_blocks; j0 += ctas * warps * 8) {
      float4 v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        v[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (j0 + g < k_blocks) v[c] = *reinterpret_cast<const float4*>(base + (j0 + g) * km_b + 16 * c);
      }
      double s[2][2] = {{0.0, 0.0}, {0.0, 0.0}};  // two chains
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const double2 a0 = a[8 * c], a1 = a[8 * c + 1];
        mma_f64(s[0], a0.x, (double)v[c].x);
        mma_f64(s[1], a0.y, (double)v[c].y);
        mma_f64(s[0], a1.x, (double)v[c].z);
        mma_f64(s[1], a1.y, (double)v[c].w);
      }
      // lane (g, t): query block g, key blocks j0 + 2 t and j0 + 2 t + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + 2 * t + e;
        if (g >= rows || j >= k_blocks) continue;
        unsigned long long k = score_key(s[0][e] + s[1][e]);
        if (causal) {
          const int64_t first = (i0 + g) * kQueryBlock + keys - queries;
          const int64_t last = min((i0 + g + 1) * (int64_t)kQueryBlock, queries) - 1 + keys - queries;
          const int64_t start = (int64_t)j * block;
          if (start + block > first) k = ~0ull;
          if (start > last) k = 0ull;
        }
        if (ctas > 1) {
          st_cluster_u32(hi0 + (g * pitch + j) * 4, (uint32_t)(k >> 32));
          st_cluster_u32(lo0 + (g * pitch + j) * 4, (uint32_t)k);
        } else {
          key_hi[g * pitch + j] = (uint32_t)(k >> 32);
          key_lo[g * pitch + j] = (uint32_t)k;
        }
      }
    }
  }
  if (ctas > 1) {
    cluster_arrive();       // second phase: all keys are in the first CTA's shared memory
    if (rank != 0) return;
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp >= rows) return;
  const uint32_t* hi = key_hi + warp * pitch;
  const uint32_t* lo = key_lo + warp * pitch;
  int32_t* dst = out + (kvh * q_blocks + i0 + warp) * (int64_t)top_k;
  // th: the largest high word with at least top_k keys at or above it (1 when fewer keys
  // than that can be selected: a key of 0 cannot, and the high word of every other is not 0)
  uint32_t th = 1u;
  int above = 0;  // keys >= th
  uint32_t v[kSelHeld];  // the lane's high words, where there are few enough
  const bool held = k_blocks <= 32 * kSelHeld;
  if (held) {
#pragma unroll
    for (int e = 0; e < kSelHeld; ++e) v[e] = lane + 32 * e < k_blocks ? hi[lane + 32 * e] : 0u;
  }
  {
    uint32_t most = 0u, least = ~0u;
    if (held) {
#pragma unroll
      for (int e = 0; e < kSelHeld; ++e) {
        most = max(most, v[e]);
        least = min(least, lane + 32 * e < k_blocks ? v[e] : ~0u);
      }
    } else {
      for (int j = lane; j < k_blocks; j += 32) {
        most = max(most, hi[j]);
        least = min(least, hi[j]);
      }
    }
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    least = __reduce_min_sync(0xFFFFFFFFu, least);
    auto count = [&](uint32_t c) {  // keys with a high word >= c, c > 0
      int n = 0;
      if (held) {
#pragma unroll
        for (int e = 0; e < kSelHeld; ++e) n += v[e] >= c;
      } else {
#pragma unroll 4
        for (int j = lane * 4; j < pitch; j += 128) {
          const uint4 w = *reinterpret_cast<const uint4*>(hi + j);
          n += (w.x >= c) + (w.y >= c) + (w.z >= c) + (w.w >= c);
        }
      }
      return (int)__reduce_add_sync(0xFFFFFFFFu, (unsigned)n);
    };
    // bits that all keys share need no search
    uint32_t c = 0u;
    int bit = 31;
    if (top_k <= k_blocks) {
      bit = 31 - __clz((int)(most ^ least));  // -1: all equal
      c = bit >= 31 ? 0u : (most >> (bit + 1)) << (bit + 1);
    }
    for (; bit >= 0; --bit) {
      const int n = count(c | (1u << bit));
      if (n >= top_k) {
        c |= 1u << bit;
        if (n == top_k) break;  // exactly the selection: no lower bit changes it
      }
    }
    th = max(c, 1u);
    above = count(th);
  }
  uint32_t th_lo = 0u;
  int equal_left = top_k;  // keys equal to (th, th_lo) that are still to be taken, the first ones
  if (above > top_k) {
    auto count = [&](bool higher, uint32_t c) {  // keys above th, or equal to it with a low word >= c
      int n = 0;
      for (int j = lane; j < k_blocks; j += 32) n += hi[j] > th || (!higher && hi[j] == th && lo[j] >= c);
      return (int)__reduce_add_sync(0xFFFFFFFFu, (unsigned)n);
    };
    for (int bit = 31; bit >= 0; --bit)
      if (count(false, th_lo | (1u << bit)) >= top_k) th_lo |= 1u << bit;
    equal_left = top_k - (th_lo == ~0u ? count(true, 0u) : count(false, th_lo + 1u));
  }
  int at = 0;
#pragma unroll 4
  for (int j0 = 0; j0 < k_blocks; j0 += 32) {
    const int j = j0 + lane;
    const uint32_t h = j < k_blocks ? hi[j] : 0u;
    const unsigned lower = (1u << lane) - 1u;
    bool take = h >= th, same = false;
    if (above > top_k && h == th) {
      const uint32_t l = lo[j];
      take = l > th_lo;
      same = l == th_lo;
    }
    const unsigned equal = __ballot_sync(0xFFFFFFFFu, same);
    take = take || (same && __popc(equal & lower) < equal_left);
    const unsigned taken = __ballot_sync(0xFFFFFFFFu, take);
    if (take) dst[at + __popc(taken & lower)] = j;
    at += __popc(taken);
    equal_left -= __popc(equal & taken);
  }
  for (int j = at + lane; j < top_k; j += 32) dst[j] = -1;
  if (out_tiles != nullptr && lane == 0) out_tiles[kvh * q_blocks + i0 + warp] = list_tiles(at, block / 64);
}

}  // namespace

namespace {

int64_t mean_blocks(const BlockMeansArgs& m) {
  return m.tokens > 0 && m.heads > 0 ? (m.tokens + m.block - 1) / m.block : 0;
}

int64_t mean_ctas(const BlockMeansArgs& a, const BlockMeansArgs& b) {
  return mean_blocks(a) * a.heads + mean_blocks(b) * b.heads;
}

// query blocks of one CTA: fewer where so many rows of scores do not fit
int select_rows(const SelectBlocksArgs& a) {
  int rows = (int)std::min<int64_t>(kSelRows, a.q_blocks);
  while (rows > 1 && (int64_t)rows * (a.k_blocks + 4) > select_blocks_max()) rows = (rows + 1) / 2;
  return rows;
}

}  // namespace

cudaError_t check_block_means(const BlockMeansArgs& a, const BlockMeansArgs& b) {
  for (const BlockMeansArgs* m : {&a, &b})
    if (mean_blocks(*m) > 0 && ((reinterpret_cast<uintptr_t>(m->x) & 15) || m->x_t % 8 || m->x_h % 8))
      return cudaErrorNotSupported;
  return mean_ctas(a, b) > 0x7FFFFFFF ? cudaErrorNotSupported : cudaSuccess;
}

cudaError_t launch_block_means(const BlockMeansArgs& a, const BlockMeansArgs& b, bool f16, cudaStream_t stream) {
  const cudaError_t e = check_block_means(a, b);
  const int64_t ctas = mean_ctas(a, b);
  if (e != cudaSuccess || ctas == 0) return e;
  MeanSource src[2];
  for (int i = 0; i < 2; ++i) {
    const BlockMeansArgs& m = i ? b : a;
    src[i].x = static_cast<const uint16_t*>(m.x);
    src[i].x_t = m.x_t; src[i].x_h = m.x_h; src[i].tokens = m.tokens;
    src[i].heads = (int)m.heads; src[i].block = (int)m.block;
    src[i].blocks = mean_blocks(m);
    src[i].means = m.means;
  }
  return launch_chained(f16 ? block_means_kernel<true> : block_means_kernel<false>, (unsigned)ctas, kMeanThreads, 0,
                        stream, false, 1, src[0], src[1]);
}

int64_t select_blocks_max() { return (200 * 1024 - kSelRows * kSelPad * 8) / 8 - 4; }

cudaError_t check_select_blocks(const SelectBlocksArgs& a) {
  if (a.q_blocks <= 0 || a.kv_heads <= 0 || a.top_k <= 0) return cudaSuccess;
  if (a.k_blocks > select_blocks_max() || (reinterpret_cast<uintptr_t>(a.k_means) & 15) || a.km_h % 4 || a.km_b % 4)
    return cudaErrorNotSupported;
  const int rows = select_rows(a);
  return a.kv_heads * ((a.q_blocks + rows - 1) / rows) > 0x0FFFFFFF ? cudaErrorNotSupported : cudaSuccess;
}

cudaError_t launch_select_blocks(const SelectBlocksArgs& a, cudaStream_t stream) {
  if (a.q_blocks <= 0 || a.kv_heads <= 0 || a.top_k <= 0) return cudaSuccess;
  const cudaError_t refused = check_select_blocks(a);
  if (refused != cudaSuccess) return refused;
  const int rows = select_rows(a);
  const int smem = (int)(kSelRows * kSelPad * 8 + (int64_t)rows * ((a.k_blocks + 3) / 4 * 4) * 8);
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(select_blocks_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  const int64_t grid = a.kv_heads * ((a.q_blocks + rows - 1) / rows);
  // CTAs per row tile: while the GPU holds them all at once, and down to two steps of key
  // blocks per warp (24 rows of 512 key blocks: 22.5 us in one CTA each, 16.4 in clusters of
  // 4 and of 8; 56 tiles of 65 key blocks: 16.4 in one CTA each and in clusters of 2)
  const int64_t steps = (a.k_blocks + kSelThreads / 4 - 1) / (kSelThreads / 4);
  const int ctas = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(8, steps / 2), 3 * num_sms(dev) / grid));
  return launch_chained(select_blocks_kernel, (unsigned)(grid * ctas), kSelThreads, smem, stream, a.chained, ctas, a.q_means, a.k_means,
                        a.km_h, a.km_b, (int)(a.heads / a.kv_heads), a.q_blocks, (int)a.k_blocks, (int)a.top_k, rows,
                        (int)a.block, a.queries, a.keys, a.causal ? 1 : 0, a.out, a.tiles,
                        static_cast<const uint16_t*>(a.q_row), a.q_row_h, a.q_row_f16 ? 1 : 0, ctas);
}

}  // namespace h3
