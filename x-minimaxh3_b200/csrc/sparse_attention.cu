// Block-sparse attention of 128-row query blocks over selected key blocks (tcgen05).
//
//   out[r] = sum_j p_j v_j / l,  p_j = exp(scale q_r . k_j - m),  l = sum_j p_j,  lse = m + ln l
//
// over the keys j of the blocks that the query block's list names (with `causal`
// those at positions up to the row's own, r + keys - queries). A row that sees no
// key gives 0 and lse = -inf.
//
// A tile is 128 rows x 128 keys (two 64-key sub-blocks from anywhere, each read by
// its own TMA boxes; 128-key blocks are two neighbouring ones):
//  * S = Q K^T: Q and K in shared memory (K-major, 128-byte swizzle), fp32 in TMEM;
//  * softmax, one thread per row: the row's 128 scores come from TMEM, its maximum
//    and sum stay in the thread's registers, and P goes back, rounded to 16 bits
//    (the tensor core's operand type), into the columns S came from;
//  * O += P V: P read from TMEM, V from shared memory as an MN-major operand (the
//    keys are its contraction dim, so it is never transposed); fp32 in TMEM.
// O is rescaled only when a row's maximum grew by more than 2^8 since the last
// rescale (P then stays below 2^8, and l and O carry the same stale maximum, which
// cancels in O / l).
//
// A CTA runs two such streams (two query blocks) over one tensor pipe: while four
// warps do the softmax of one stream, the tensor core works on the other. Two
// query tiles, a ring of five 32 KB K/V tiles and 512 TMEM columns (2 S, 2 O) fill
// the SM, so there is one CTA per SM.
#include <algorithm>

#include "attn_math.cuh"
#include "kernels.h"

namespace h3 {

bool encode_tmap_3d_bf16(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1,
                         uint64_t s2, uint32_t b0, uint32_t b1, uint32_t b2, CUtensorMapSwizzle swizzle);

namespace {

constexpr int kSpThreads = 384;    // 2 x 4 softmax warps, two TMA warps (8, 11), one MMA warp per stream (9, 10)
constexpr int kSubKeys = 64;  // keys of one TMA box; a tile holds two
constexpr int kTileBytes = 128 * kHeadDim * 2;     // 32 KB: a Q, K or V tile
constexpr int kHalfBytes = kTileBytes / 2;         // dims 0..63 or 64..127 of 128 rows
constexpr int kRing = 5;
constexpr int kOffRing = 2 * kTileBytes;
constexpr int kOffBar = kOffRing + kRing * kTileBytes;
constexpr int kSpSmem = kOffBar + 512 + 1024;      // + barriers + alignment
constexpr unsigned kErrSpProd = 0x501, kErrSpMma = 0x502, kErrSpSoft = 0x503, kErrSpOut = 0x504, kErrSpDrain = 0x505;
constexpr float kRescaleLog2 = 8.0f;

struct SparseParams {
  const int32_t* blocks;  // [kv_heads, q_blocks, top_k]
  int top_k, block, k_blocks;
  int queries, keys, q_blocks, heads, group;
  int64_t items;
  int streams;            // 2: the CTA's items are 2 b and 2 b + 1; 1: item b alone
  int causal;
  float scale, scale_log2;
  uint16_t* out;
  int64_t o_t, o_h;
  float* lse;
  int64_t l_t, l_h;
};

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x,
                                            int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(smem_dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// MN-major operand (the contraction dim is the row index): 128-byte rows of 64 MN
// elements with 128-byte swizzle, 8-row groups 1024 bytes apart (SBO), the next 64 MN
// elements kHalfBytes further (LBO).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(kHalfBytes >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

// kind::f16, fp32 accumulator, A and B both bf16 or both fp16; B MN-major for P V
constexpr uint32_t idesc_f16kind(bool f16, bool b_mn) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? 1u << 16 : 0u) | ((128u >> 3) << 17) |
         ((128u >> 4) << 24);
}

// A from TMEM (128 lanes x 8 columns of packed pairs), B from shared memory
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// First key of sub-block `sub` of the list (64 keys from there), or -1: no such block.
__device__ __forceinline__ int sub_key(const SparseParams& p, const int32_t* list, int sub) {
  const int per = p.block / kSubKeys;
  const int e = sub / per;
  if (e >= p.top_k) return -1;
  const int id = __ldg(list + e);
  if (id < 0 || id >= p.k_blocks) return -1;
  return id * p.block + (sub - e * per) * kSubKeys;
}

// 32 lanes x 16 columns, as tmem_ld32 / tmem_st32
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

struct Stream {
  int64_t item;
  int head, q_block;
  const int32_t* list;
};

__device__ __forceinline__ Stream stream_of(const SparseParams& p, int s) {
  Stream st;
  st.item = p.streams == 2 ? (int64_t)blockIdx.x * 2 + s : (int64_t)blockIdx.x;
  st.head = (int)(st.item / p.q_blocks);
  st.q_block = (int)(st.item - (int64_t)st.head * p.q_blocks);
  st.list = p.blocks + ((int64_t)(st.head / p.group) * p.q_blocks + st.q_block) * p.top_k;
  return st;
}

template <bool F16>
__global__ void __launch_bounds__(kSpThreads, 1)
    sparse_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                            const __grid_constant__ CUtensorMap tm_v, const SparseParams p) {
  using E = Elem16<F16>;
  extern __shared__ uint8_t sp_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sp_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + kOffBar);  // [2]
  uint64_t* kv_full = q_full + 2;                                  // [kRing]
  uint64_t* kv_empty = kv_full + kRing;                            // [kRing]
  uint64_t* s_full = kv_empty + kRing;                             // [2] scores are in TMEM
  uint64_t* p_full = s_full + 2;                                   // [2][2] a half of P is in TMEM, O is rescaled
  uint64_t* o_full = p_full + 4;                                   // [2] O is complete
  uint64_t* turn = o_full + 2;                                     // [2] the stream's products of a tile are issued
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(turn + 2);
  int* tiles_of = reinterpret_cast<int*>(tmem_slot + 1);           // [2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 2);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);  // one arrival per softmax warp
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&turn[i], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&kv_full[i], 2);  // one arrival per TMA warp
      mbar_init(&kv_empty[i], 1);
    }
    fence_barrier_init();
    fence_proxy_async_shared();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 8) {
    // tiles of each stream: up to its last listed block
    for (int s = 0; s < 2; ++s) {
      int last = -1;
      if (s < p.streams && stream_of(p, s).item < p.items) {
        const int32_t* list = stream_of(p, s).list;
        for (int e = lane; e < p.top_k; e += 32) {
          const int id = __ldg(list + e);
          if (id >= 0 && id < p.k_blocks) last = e;
        }
      }
      last = __reduce_max_sync(0xFFFFFFFFu, last);
      if (lane == 0) tiles_of[s] = ((last + 1) * (p.block / kSubKeys) + 1) / 2;
    }
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n0 = tiles_of[0], n1 = tiles_of[1];
  const int nmax = max(n0, n1);

  if (warp == 8 || warp == 11) {
    if (lane == 0) {
      // ---------------- TMA producers: warp 8 loads the first 64 keys of each tile, 11 the second ----------------
      // (one thread issues a 64-row box every 237 clocks, 34 B/clk, whatever is in flight;
      // two threads reach 48 B/clk together). Both follow the order in which the MMA
      // warps consume.
      const int u = warp == 8 ? 0 : 1;
      int issued = 0;
      bool ok = true;
      const Stream st[2] = {stream_of(p, 0), stream_of(p, 1)};
      const int n[2] = {n0, n1};
      for (int s = 0; s < 2; ++s)
        if (n[s] > 0) {
          mbar_arrive_expect_tx(&q_full[s], kHalfBytes);
          tma_load_3d(smem + s * kTileBytes + u * kHalfBytes, &tm_q, &q_full[s], u * 64, st[s].q_block * kQueryBlock,
                      st[s].head);
        }
      auto load_tile = [&](int s, int i, const CUtensorMap* map) {
        const int slot = issued % kRing;
        const int key = sub_key(p, st[s].list, 2 * i + u);
        if (!mbar_wait(&kv_empty[slot], ((issued / kRing) & 1) ^ 1, kErrSpProd)) return false;
        uint8_t* dst = smem + kOffRing + slot * kTileBytes + u * (kSubKeys * 128);
        mbar_arrive_expect_tx(&kv_full[slot], kHalfBytes);
        for (int h = 0; h < 2; ++h)  // rows past the last key (and absent sub-blocks) arrive as zeros
          tma_load_3d(dst + h * kHalfBytes, map, &kv_full[slot], h * 64, key < 0 ? p.keys : key, st[s].head / p.group);
        ++issued;
        return true;
      };
      for (int s = 0; s < 2 && ok; ++s)
        if (n[s] > 0) ok = load_tile(s, 0, &tm_k);
      for (int i = 0; i < nmax && ok; ++i)
        for (int s = 0; s < 2 && ok; ++s) {
          if (i < n[s]) ok = load_tile(s, i, &tm_v);
          if (ok && i + 1 < n[s]) ok = load_tile(s, i + 1, &tm_k);
        }
      for (int s = 0; s < 2; ++s)  // issued copies land before exit
        if (n[s] > 0) mbar_wait(&q_full[s], 0, kErrSpDrain, 200000000ull);
      for (int j = (issued > kRing ? issued - kRing : 0); j < issued; ++j)
        mbar_wait(&kv_full[j % kRing], (j / kRing) & 1, kErrSpDrain, 200000000ull);
    }
  } else if (warp >= 9) {
    if (lane == 0) {
      // ---------------- MMA issuers: warp 9 + s serves stream s ----------------
      // An issuing thread is held until its instruction enters the (short) tensor queue,
      // so its waits for softmax and loads would leave the tensor core idle; with an
      // issuer per stream they run beside the other stream's products. The issuers take
      // turns (turn[s]: stream s has issued its i-th P V and next Q K^T): left to
      // themselves they interleave instruction by instruction, both softmaxes then start
      // together, and the exponentials of one no longer hide behind the products of the
      // other (2,126 us on the 21 x 39 x 40 grid, 24 heads, 64 of 512 blocks). Ring slots
      // keep the producer's order over both streams: an issuer counts past the other's tiles.
      constexpr uint32_t kIdescS = idesc_f16kind(F16, false), kIdescO = idesc_f16kind(F16, true);
      const int s = warp - 9, n = s ? n1 : n0, other = s ? n0 : n1;
      const uint32_t t_s = tmem + s * 128, t_o = tmem + 256 + s * 128;
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem + s * kTileBytes));
      const uint32_t ring = smem_u32(smem + kOffRing);
      int at = s == 1 && other > 0 ? 1 : 0;  // ring position of this stream's next tile
      auto scores = [&]() {
        const int slot = at % kRing;
        const uint64_t k_desc = umma_desc_sw128(ring + slot * kTileBytes);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
          umma_bf16(t_s, q_desc + off, k_desc + off, kIdescS, k > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[s]);
        umma_commit(&kv_empty[slot]);
      };
      bool ok = n > 0 && mbar_wait(&q_full[s], 0, kErrSpMma) &&
                mbar_wait(&kv_full[at % kRing], (at / kRing) & 1, kErrSpMma);
      if (ok) {
        tc_fence_after();
        scores();
      }
      at = (n0 > 0 ? 1 : 0) + (n1 > 0 ? 1 : 0) + (s == 1 ? (other > 0 ? 1 : 0) + (other > 1 ? 1 : 0) : 0);
      for (int i = 0; i < n && ok; ++i) {
        const int slot = at % kRing;
        ok = mbar_wait(&kv_full[slot], (at / kRing) & 1, kErrSpMma);
        if (i + 1 < n) ok = ok && mbar_wait(&kv_full[(at + 1) % kRing], ((at + 1) / kRing) & 1, kErrSpMma);
        ok = ok && mbar_wait(&p_full[2 * s], i & 1, kErrSpMma);
        const int before = s == 0 ? i - 1 : i;  // the other stream's tile whose turn comes first
        if (before >= 0 && before < other) ok = ok && mbar_wait(&turn[1 - s], before & 1, kErrSpMma);
        const uint64_t v_desc = umma_desc_mn_sw128(ring + slot * kTileBytes);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // the first half's product runs while the second half's P is computed
          if (h == 1) ok = ok && mbar_wait(&p_full[2 * s + 1], i & 1, kErrSpMma);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 4 * h; k < 4 * h + 4; ++k)
            umma_f16_ts(t_o, t_s + k * 8, v_desc + ((k * 16 * 128) >> 4), kIdescO, i > 0 || k > 0 ? 1u : 0u);
        }
        if (!ok) break;
        if (i + 1 < n) {
          ++at;
          scores();  // executes after the product above, which reads the columns it overwrites
          // then the other stream's V and next K: tile i of stream 1, tile i + 1 of stream 0
          const int j = s == 0 ? i : i + 1;
          at += 1 + (j < other ? 1 : 0) + (j + 1 < other ? 1 : 0);
        } else {
          umma_commit(&o_full[s]);
        }
        mbar_arrive(&turn[s]);
        umma_commit(&kv_empty[slot]);
      }
    }
  } else {
    // ---------------- softmax: thread = row ----------------
    const int s = warp >> 2;
    const int n = s ? n1 : n0;
    const Stream st = stream_of(p, s);
    const int row = st.q_block * kQueryBlock + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + s * 128 + lanes, t_o = tmem + 256 + s * 128 + lanes;
    const int limit = p.causal ? min(p.keys, row + 1 + p.keys - p.queries) : p.keys;  // keys this row may see
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    int key0 = -1, key1 = -1;
    if (n > 0) {
      key0 = sub_key(p, st.list, 0);
      key1 = sub_key(p, st.list, 1);
    }
    for (int i = 0; i < n; ++i) {
      const int v0 = key0 < 0 ? 0 : limit - key0, v1 = key1 < 0 ? 0 : limit - key1;  // visible keys of the halves
      if (i + 1 < n) {
        key0 = sub_key(p, st.list, 2 * i + 2);
        key1 = sub_key(p, st.list, 2 * i + 3);
      }
      if (!mbar_wait(&s_full[s], i & 1, kErrSpSoft)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, x[c]);
      tmem_wait_ld();
      if (!__all_sync(0xFFFFFFFFu, v0 >= kSubKeys && v1 >= kSubKeys)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((c & 1) * 32 + e >= (c < 2 ? v0 : v1)) x[c][e] = 0xFF800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = fmaxf(__uint_as_float(x[c][0]), __uint_as_float(x[c][1]));
#pragma unroll
        for (int e = 2; e < 32; e += 2) mx[c] = max3(mx[c], __uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grow = (top - m) * p.scale_log2 > kRescaleLog2;  // also the first finite score (m = -inf)
      if (i == 0) {
        m = top;
      } else if (__any_sync(0xFFFFFFFFu, grow)) {
        const float f = grow ? ex2_approx((m - top) * p.scale_log2) : 1.0f;
        if (grow) m = top;
        l *= f;
        // the product of the tile before is complete: its commit came before s_full's
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          uint32_t o[16];
          tmem_ld16(t_o + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st16(t_o + c * 16, o);
        }
      }
      const float sub = m == -INFINITY ? 0.0f : m * p.scale_log2;
      const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2), sub2 = f2_pack(-sub, -sub);
      uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float a, b;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1])), scale2, sub2), a, b);
          a = ex2_approx(a);
          b = ex2_approx(b);
          sum[e & 1] = f2_add(sum[e & 1], f2_pack(a, b));
          w[e] = E::pack(a, b);
        }
        tmem_st16(t_s + c * 16, w);  // over columns already read
        if (c & 1) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * s + (c >> 1)]);
        }
      }
      float s0, s1, s2, s3;
      f2_unpack(sum[0], s0, s1);
      f2_unpack(sum[1], s2, s3);
      l += (s0 + s1) + (s2 + s3);
    }
    if (st.item < p.items && s < p.streams && ok) {
      if (n > 0) ok = mbar_wait(&o_full[s], 0, kErrSpOut);
      tc_fence_after();
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays
      uint16_t* dst = p.out + (int64_t)row * p.o_t + (int64_t)st.head * p.o_h;
      if (ok) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld32(t_o + c * 32, o);
            tmem_wait_ld();
          }
          if (row < p.queries) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int at = e * 8 + 2 * j;
                w[j] = l == 0.0f ? 0u : E::pack(__uint_as_float(o[at]) * inv, __uint_as_float(o[at + 1]) * inv);
              }
              stg_v4(dst + c * 32 + e * 8, make_uint4(w[0], w[1], w[2], w[3]));
            }
          }
          __syncwarp();
        }
        if (row < p.queries && p.lse != nullptr)
          p.lse[(int64_t)row * p.l_t + (int64_t)st.head * p.l_h] = l == 0.0f ? -INFINITY : fmaf(m, p.scale, logf(l));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

bool map_view(CUtensorMap* map, const void* base, int64_t rows, int64_t heads, int64_t st, int64_t sh, int box_rows) {
  // a dim of one element has no stride that matters; the encoder still checks it
  if (rows == 1) st = kHeadDim;
  if (heads == 1) sh = kHeadDim;
  if ((reinterpret_cast<uintptr_t>(base) & 15) || st <= 0 || sh <= 0 || st % 8 || sh % 8) return false;
  return encode_tmap_3d_bf16(map, base, kHeadDim, (uint64_t)rows, (uint64_t)heads, (uint64_t)st * 2, (uint64_t)sh * 2,
                             64, (uint32_t)box_rows, 1, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool F16>
cudaError_t launch_sparse(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const SparseParams& p,
                          unsigned grid, int dev, cudaStream_t stream) {
  static bool attr_set[64] = {false};
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(sparse_attention_kernel<F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSpSmem);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  sparse_attention_kernel<F16><<<grid, kSpThreads, kSpSmem, stream>>>(q, k, v, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_block_sparse_attention(const SparseAttnArgs& a, cudaStream_t stream) {
  if (a.queries <= 0 || a.heads <= 0) return cudaSuccess;
  SparseParams p;
  p.q_blocks = (int)((a.queries + kQueryBlock - 1) / kQueryBlock);
  p.items = a.heads * p.q_blocks;
  if (a.queries > 0x7FFFFF00 || a.keys > 0x7FFFFF00 || p.items > 0x7FFFFFFF || a.block % kSubKeys || a.o_t % 8 ||
      a.o_h % 8 || (reinterpret_cast<uintptr_t>(a.out) & 15))
    return cudaErrorNotSupported;
  CUtensorMap q, k, v;
  if (!map_view(&q, a.q, a.queries, a.heads, a.q_t, a.q_h, kQueryBlock) ||
      !map_view(&k, a.k, a.keys, a.kv_heads, a.k_t, a.k_h, kSubKeys) ||
      !map_view(&v, a.v, a.keys, a.kv_heads, a.v_t, a.v_h, kSubKeys))
    return cudaErrorNotSupported;
  p.blocks = a.blocks; p.top_k = (int)a.top_k; p.block = (int)a.block;
  p.k_blocks = (int)((a.keys + a.block - 1) / a.block);
  p.queries = (int)a.queries; p.keys = (int)a.keys; p.heads = (int)a.heads; p.group = (int)(a.heads / a.kv_heads);
  p.causal = a.causal ? 1 : 0;
  p.scale = a.scale; p.scale_log2 = a.scale * 1.4426950408889634f;
  p.out = static_cast<uint16_t*>(a.out); p.o_t = a.o_t; p.o_h = a.o_h;
  p.lse = a.lse; p.l_t = a.l_t; p.l_h = a.l_h;
  int dev = 0;
  cudaGetDevice(&dev);
  p.streams = p.items > num_sms(dev) ? 2 : 1;  // a second stream only where every SM has a first one
  const unsigned grid = (unsigned)((p.items + p.streams - 1) / p.streams);
  return a.f16 ? launch_sparse<true>(q, k, v, p, grid, dev, stream) : launch_sparse<false>(q, k, v, p, grid, dev, stream);
}

}  // namespace h3
