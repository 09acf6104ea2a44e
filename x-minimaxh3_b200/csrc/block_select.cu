// Selection of key blocks for block-sparse attention: block means, scores, top-k.
//
//   m[h, b]     = fp32(mean of the rows of block b of head h)
//   score[i, j] = sum over the query heads h of a key head's group of m_q[h, i] . m_k[j]
//   the top_k highest scores of each row i; equal scores go to the lowest j; ascending output
//
// A selection is a whole-number result: two scores that differ in their last bits
// must not change places from one implementation (or one summation order) to
// another. Sums and products are therefore held in 64 bits: a block's sum of
// 16-bit values is exact there, and so is each product of two fp32 means, which
// leaves about 1e-16 of the score's terms as its error. In 32 bits (1e-7) about one
// selection in 10^4 changes with the order of the sum.
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

// One CTA per (block, head). A half-warp reads a 256-byte row as 16 lanes x 16 bytes.
// HBM-bound in principle; the loads of a 64-key block are few, so what counts is how
// many small CTAs an SM holds. Consecutive CTAs take consecutive heads of the same tokens.
template <bool F16>
__global__ void __launch_bounds__(kMeanThreads, 6) block_means_kernel(const uint16_t* __restrict__ x, int64_t x_t,
                                                                   int64_t x_h, int64_t tokens, int heads, int block,
                                                                   int64_t blocks, float* __restrict__ means) {
  using E = Elem16<F16>;
  __shared__ double part[kMeanThreads / 32][kHeadDim];
  const int hw = threadIdx.x >> 4, l = threadIdx.x & 15, warp = threadIdx.x >> 5;
  const int64_t b = blockIdx.x / heads;
  const int h = (int)(blockIdx.x - b * heads);
  const int64_t t0 = b * block;
  const int rows = (int)min((int64_t)block, tokens - t0);
  double s[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
  const uint16_t* src = x + h * x_h + t0 * x_t + l * 8;
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
  means[((int64_t)h * blocks + b) * kHeadDim + threadIdx.x] = (float)(sum / (double)rows);
}
static_assert(kMeanThreads == kHeadDim, "one thread per dim finishes a mean");

constexpr int kSelThreads = 512;
constexpr int kSelRows = 8;  // query blocks per CTA: the M of one 64-bit matrix instruction; one warp each for the top-k

// c[8 x 8] += a[8 x 4] b[4 x 8] in 64 bits
__device__ __forceinline__ void mma_f64(double (&c)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
               : "+d"(c[0]), "+d"(c[1])
               : "d"(a), "d"(b));
}

// 64-bit key whose unsigned order is the order of the scores; 0 stands for "not to be
// selected". NaN scores rank below every number.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (!(s == s)) return 1ull;
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
// 16 c + 4 t .. + 3) and uses them in four instructions; the 8 query rows stay in
// registers in the same order.
__global__ void __launch_bounds__(kSelThreads) select_blocks_kernel(const float* __restrict__ qm,
                                                                    const float* __restrict__ km, int64_t km_h,
                                                                    int64_t km_b, int group,
                                                                    int64_t q_blocks, int k_blocks, int top_k,
                                                                    int rows_per_cta, int block, int64_t queries,
                                                                    int64_t keys, int causal,
                                                                    int32_t* __restrict__ out,
                                                                    int32_t* __restrict__ out_tiles) {
  extern __shared__ __align__(16) unsigned char sel_smem[];
  double* qs = reinterpret_cast<double*>(sel_smem);                               // [rows][128]
  unsigned long long* key = reinterpret_cast<unsigned long long*>(qs + kSelRows * kHeadDim);  // [rows][k_blocks]
  const int64_t tiles = (q_blocks + rows_per_cta - 1) / rows_per_cta;
  const int64_t kvh = blockIdx.x / tiles;
  const int64_t i0 = (blockIdx.x - kvh * tiles) * rows_per_cta;
  const int rows = (int)min((int64_t)rows_per_cta, q_blocks - i0);
  for (int e = threadIdx.x; e < kSelRows * kHeadDim; e += kSelThreads) {
    const int r = e / kHeadDim, d = e % kHeadDim;
    double s = 0.0;
    if (r < rows)
      for (int g = 0; g < group; ++g) s += (double)__ldg(qm + ((kvh * group + g) * q_blocks + i0 + r) * kHeadDim + d);
    qs[e] = s;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  {
    const int g = lane >> 2, t = lane & 3;
    double a[32];
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) a[4 * c + e] = qs[g * kHeadDim + 16 * c + 4 * t + e];
    const float* base = km + kvh * km_h + 4 * t;
    for (int j0 = warp * 8; j0 < k_blocks; j0 += kSelThreads / 32 * 8) {
      float4 v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        v[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (j0 + g < k_blocks) v[c] = __ldg(reinterpret_cast<const float4*>(base + (j0 + g) * km_b + 16 * c));
      }
      double s[2][2] = {{0.0, 0.0}, {0.0, 0.0}};  // two chains
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        mma_f64(s[0], a[4 * c], (double)v[c].x);
        mma_f64(s[1], a[4 * c + 1], (double)v[c].y);
        mma_f64(s[0], a[4 * c + 2], (double)v[c].z);
        mma_f64(s[1], a[4 * c + 3], (double)v[c].w);
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
        key[(int64_t)g * k_blocks + j] = k;
      }
    }
  }
  __syncthreads();
  if (warp >= rows) return;
  const unsigned long long* mine = key + (int64_t)warp * k_blocks;
  int32_t* dst = out + (kvh * q_blocks + i0 + warp) * (int64_t)top_k;
  // largest threshold with at least top_k keys at or above it; 1 (everything) when fewer exist
  unsigned long long th = 0ull;
  int above = k_blocks;  // keys >= th
  bool enough = false;
  // bits that all keys share need no search: th starts as their common prefix
  unsigned long long hi = 0ull, lo = ~0ull;
  for (int j = lane; j < k_blocks; j += 32) {
    const unsigned long long k = mine[j];
    hi = max(hi, k);
    lo = min(lo, k);
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) {
    hi = max(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, i));
    lo = min(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, i));
  }
  int top_bit = 63;
  if (k_blocks > 0 && top_k <= k_blocks) {
    top_bit = 63 - __clzll((long long)(hi ^ lo));  // -1: all equal
    th = top_bit >= 63 ? 0ull : (hi >> (top_bit + 1)) << (top_bit + 1);
    enough = th != 0ull;                           // every key is at or above the prefix
  }
  for (int bit = top_bit; bit >= 0; --bit) {
    const unsigned long long c = th | (1ull << bit);
    int n = 0;
    for (int j = lane; j < k_blocks; j += 32) n += mine[j] >= c ? 1 : 0;
    n = (int)__reduce_add_sync(0xFFFFFFFFu, (unsigned)n);
    if (n >= top_k) {
      th = c;
      above = n;
      enough = true;
      if (n == top_k) break;  // exactly the selection: no lower bit changes it
    }
  }
  if (!enough || th == 0ull) th = 1ull;
  // keys above the threshold are all taken; of those equal to it the first ones
  int equal_left = top_k;
  if (enough && above > top_k) {
    int n = 0;
    for (int j = lane; j < k_blocks; j += 32) n += mine[j] > th ? 1 : 0;
    equal_left = top_k - (int)__reduce_add_sync(0xFFFFFFFFu, (unsigned)n);
  }
  int at = 0;
  for (int j0 = 0; j0 < k_blocks; j0 += 32) {
    const int j = j0 + lane;
    const unsigned long long k = j < k_blocks ? mine[j] : 0ull;
    const unsigned lower = (1u << lane) - 1u;
    const bool exact = above == top_k && enough;
    const unsigned equal = __ballot_sync(0xFFFFFFFFu, !exact && k == th);
    const bool take = k > th || (k == th && (exact || __popc(equal & lower) < equal_left));
    const unsigned taken = __ballot_sync(0xFFFFFFFFu, take);
    if (take) dst[at + __popc(taken & lower)] = j;
    at += __popc(taken);
    equal_left -= __popc(equal & taken);
  }
  for (int j = at + lane; j < top_k; j += 32) dst[j] = -1;
  if (out_tiles != nullptr && lane == 0) out_tiles[kvh * q_blocks + i0 + warp] = list_tiles(at, block / 64);
}

}  // namespace

cudaError_t launch_block_means(const void* x, int64_t x_t, int64_t x_h, int64_t tokens, int64_t heads, int64_t block,
                               bool f16, float* means, cudaStream_t stream) {
  const int64_t blocks = (tokens + block - 1) / block;
  if (blocks * heads == 0) return cudaSuccess;
  if ((reinterpret_cast<uintptr_t>(x) & 15) || x_t % 8 || x_h % 8 || blocks * heads > 0x7FFFFFFF)
    return cudaErrorNotSupported;
  const unsigned grid = (unsigned)(blocks * heads);
  if (f16)
    block_means_kernel<true><<<grid, kMeanThreads, 0, stream>>>(static_cast<const uint16_t*>(x), x_t, x_h, tokens,
                                                                (int)heads, (int)block, blocks, means);
  else
    block_means_kernel<false><<<grid, kMeanThreads, 0, stream>>>(static_cast<const uint16_t*>(x), x_t, x_h, tokens,
                                                                 (int)heads, (int)block, blocks, means);
  return cudaGetLastError();
}

int64_t select_blocks_max() { return (200 * 1024 - kSelRows * kHeadDim * 8) / 8; }

cudaError_t launch_select_blocks(const SelectBlocksArgs& a, cudaStream_t stream) {
  if (a.q_blocks <= 0 || a.kv_heads <= 0 || a.top_k <= 0) return cudaSuccess;
  if (a.k_blocks > select_blocks_max() || (reinterpret_cast<uintptr_t>(a.k_means) & 15) || a.km_h % 4 || a.km_b % 4)
    return cudaErrorNotSupported;
  int rows = kSelRows;
  while (rows > 1 && (int64_t)rows * a.k_blocks > select_blocks_max()) rows /= 2;
  const int smem = (int)(kSelRows * kHeadDim * 8 + (int64_t)rows * a.k_blocks * 8);
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
  if (grid > 0x7FFFFFFF) return cudaErrorNotSupported;
  select_blocks_kernel<<<(unsigned)grid, kSelThreads, smem, stream>>>(
      a.q_means, a.k_means, a.km_h, a.km_b, (int)(a.heads / a.kv_heads), a.q_blocks, (int)a.k_blocks, (int)a.top_k, rows, (int)a.block,
      a.queries, a.keys, a.causal ? 1 : 0, a.out, a.tiles);
  return cudaGetLastError();
}

}  // namespace h3
