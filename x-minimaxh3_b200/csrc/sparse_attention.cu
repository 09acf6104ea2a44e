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
// rescale (P then stays below 2^8, in fp16 times 2^7 (WeightScale), and l and O carry the
// same stale maximum, which cancels in O / l).
//
// A CTA runs two such streams over one tensor pipe: while four warps do the softmax of
// one stream, the tensor core works on the other. Two query tiles, a ring of five 32 KB
// K/V tiles and 512 TMEM columns (2 S, 2 O) fill the SM, so there is one CTA per SM,
// persistent: stream s of CTA b takes the items b + G (s + 2 r). With few query blocks
// a list is split into parts, which a second kernel joins in their order.
//
// Bound: the tensor core in principle (1,024 clocks a tile of both products at the issue
// rate). 24 heads, 32,760 tokens, 64 of 512 blocks (1.65 TFLOP): 1.52 ms, 1,085 TFLOP/s,
// 66% of the measured bf16 burst, in isolation; 1.77 ms back to back, where the power
// limit takes the SM clock from 1.70 to 1.47 GHz. A pair of tiles takes about 3,600 clocks
// against 2,048: scores to weights 2,000 (exponentials at half the rate of their unit,
// two warps per scheduler), then both products and three hand-overs. Shortening the
// issuers' code, a deeper or shallower ring, passing the turn earlier or later and four
// TMA warps changed the time by less than 3% either way: fewer clocks came with a lower
// clock. The end of an item costs 5,800 clocks of a pair (rows stored a sector per lane,
// the next item's queries), which is what short lists pay.
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
constexpr int kSpSmem = kOffBar + 1024 + 1024;     // + barriers and notes + alignment
constexpr unsigned kErrSpProd = 0x501, kErrSpMma = 0x502, kErrSpSoft = 0x503, kErrSpOut = 0x504, kErrSpDrain = 0x505;
constexpr float kRescaleLog2 = 8.0f;
template <bool F16>
using SparseWeight = WeightScale<F16, 7>;  // weights count from a maximum that may be 2^8 too low
// One pair of exponentials of kPolyOf is computed on the FMA pipe: the special-function
// unit gives 16 a clock and SM, 1,024 clocks a tile, as long as the tile's products take.
constexpr int kPolyOf = 8;

struct SparseParams {
  const int32_t* blocks;  // [kv_heads, q_blocks, top_k]
  const int32_t* tiles;   // [kv_heads, q_blocks]: tiles up to the list's last block
  int top_k, block, k_blocks;
  int queries, keys, q_blocks, heads, group;
  int items, parts;       // items = heads * q_blocks * parts: a list is split into `parts` runs of tiles
  int causal;
  float* ws_acc;          // parts > 1: unnormalised fp32 rows [items][128][128] and their (m, l)
  float2* ws_ml;
  float scale, scale_log2;
  uint16_t* out;
  int64_t o_t, o_h;
  int out32;              // rows of out are 32-byte aligned
  float* lse;
  int64_t l_t, l_h;
};

// one 32-byte sector per lane
__device__ __forceinline__ void stg_v8(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f,
                                       uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e),
               "r"(f), "r"(g), "r"(h)
               : "memory");
}

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

// Item `idx`: tiles [first, first + n) of the list of one query block of one head.
struct Work {
  int head, q_block, part, first, n;
  const int32_t* list;
};

__device__ __forceinline__ Work work_of(const SparseParams& p, int idx) {
  Work w;
  const int row = idx / p.parts;
  w.part = idx - row * p.parts;
  w.head = row / p.q_blocks;
  w.q_block = row - w.head * p.q_blocks;
  if (p.causal) w.q_block = p.q_blocks - 1 - w.q_block;  // the longest lists first
  const int at = (w.head / p.group) * p.q_blocks + w.q_block;
  w.list = p.blocks + (int64_t)at * p.top_k;
  const int total = p.tiles[at];
  const int per = (total + p.parts - 1) / p.parts;
  w.first = min(total, w.part * per);
  w.n = min(total - w.first, per);
  return w;
}

// What the producers tell the other warps through shared memory (they run ahead by less
// than the ring, so kNotes entries of each kind cannot be overtaken; the loads' barriers order them).
constexpr int kNotes = 8;
struct ItemNote {
  int head, q_block, part, n;
};

template <bool F16>
__global__ void __launch_bounds__(kSpThreads, 1)
    sparse_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                            const __grid_constant__ CUtensorMap tm_v, const SparseParams p) {
  using E = Elem16<F16>;
  extern __shared__ uint8_t sp_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sp_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + kOffBar);  // [2]
  uint64_t* q_empty = q_full + 2;                                  // [2] the item's last scores are computed
  uint64_t* kv_full = q_empty + 2;                                 // [kRing]
  uint64_t* kv_empty = kv_full + kRing;                            // [kRing]
  uint64_t* s_full = kv_empty + kRing;                             // [2] scores are in TMEM
  uint64_t* p_full = s_full + 2;                                   // [2][2] a half of P is in TMEM, O is rescaled
  uint64_t* o_full = p_full + 4;                                   // [2] the item's O is complete
  uint64_t* turn = o_full + 2;                                     // [2] the stream's products of a tile are issued
  uint64_t* h_done = turn + 2;                                     // [2] the product of P's first half is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(h_done + 2);
  int* tiles_of = reinterpret_cast<int*>(tmem_slot + 1);           // [2] tiles of each stream
  int* empty_of = tiles_of + 2;                                    // [2] whether it has items without tiles
  ItemNote* item_note = reinterpret_cast<ItemNote*>(smem + kOffBar + 384);  // [2][kNotes] items that have tiles
  int2* key_note = reinterpret_cast<int2*>(item_note + 2 * kNotes);         // [2][kNotes] first keys of a tile's halves
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 2);  // one arrival per TMA warp
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);  // one arrival per softmax warp
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&turn[i], 1);
      mbar_init(&h_done[i], 1);
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
  launch_next();
  wait_previous();  // lists and tile counts
  if (warp == 8 || warp == 9) {
    const int s = warp - 8;
    int tiles = 0;
    bool empty = false;
    for (int idx = blockIdx.x + gridDim.x * (s + 2 * lane); idx < p.items; idx += 2 * 32 * gridDim.x) {
      const int n = work_of(p, idx).n;
      tiles += n;
      empty = empty || n == 0;
    }
    tiles = (int)__reduce_add_sync(0xFFFFFFFFu, (unsigned)tiles);
    empty = __any_sync(0xFFFFFFFFu, empty);
    if (lane == 0) {
      tiles_of[s] = tiles;
      empty_of[s] = empty ? 1 : 0;
    }
  }
  if (warp == 10) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n0 = tiles_of[0], n1 = tiles_of[1];

  if (warp == 8 || warp == 11) {
    // ---------------- TMA producers: warp 8 loads the first 64 keys of each tile, 11 the second ----------------
    // (one thread issues a 64-row box every 237 clocks, 34 B/clk, whatever is in flight;
    // two threads reach 48 B/clk together). Both follow the order in which the MMA
    // warps consume. The whole warp walks the lists, one lane per tile, so that an
    // item costs one list read and a tile none.
    const int u = warp == 8 ? 0 : 1;
    int issued = 0;
    bool ok = true;
    struct Feed {  // one stream
      int s, base;                             // lane e of the batch: item base + e of the stream
      int b_head, b_block, b_part, b_first, b_n;
      int pos;                                 // the batch's next item
      int n_head, n_block, n_part, n_first, n_n, n_ids0, n_ids1;  // the item after the current one (n_n 0: none)
      int head, block, part, first, n;         // the item whose K tiles are being loaded (n 0: none)
      int ids0, ids1;                          // lane e: block ids of its tile i0 + e, i0 = i rounded down to 32
      int i, item, tile, v_key, v_head;
      bool pending;                            // V of the last K tile is not loaded yet
    } a, o;
    auto refill = [&](Feed& t) {
      const int64_t idx = blockIdx.x + (int64_t)gridDim.x * (t.s + 2 * (int64_t)(t.base + lane));
      t.b_n = -1;
      if (idx < p.items) {
        const Work w = work_of(p, (int)idx);
        t.b_head = w.head; t.b_block = w.q_block; t.b_part = w.part; t.b_first = w.first; t.b_n = w.n;
      }
      t.pos = 0;
    };
    // Lane e: block ids of tile i + e. Nothing looks at them before key_of, an item (or a
    // tile) later: the warp would stand still for the length of the load.
    const int per = p.block / kSubKeys;
    auto read_ids = [&](int head, int block, int first, int n, int i, int& ids0, int& ids1) {
      ids0 = ids1 = -1;
      if (i + lane < n) {
        const int32_t* list = p.blocks + (int64_t)((head / p.group) * p.q_blocks + block) * p.top_k;
        const int e0 = 2 * (first + i + lane) / per, e1 = (2 * (first + i + lane) + 1) / per;
        if (e0 < p.top_k) ids0 = list[e0];
        if (e1 < p.top_k) ids1 = list[e1];
      }
    };
    auto key_of = [&](int id, int half) {  // first of the 64 keys, or -1: no such block
      return id < 0 || id >= p.k_blocks ? -1 : id * p.block + (per == 2 ? half * kSubKeys : 0);
    };
    auto advance = [&](Feed& t) {  // the next item becomes the current one; the one after it is looked up
      t.head = t.n_head; t.block = t.n_block; t.part = t.n_part; t.first = t.n_first; t.n = t.n_n;
      t.ids0 = t.n_ids0; t.ids1 = t.n_ids1;
      t.i = 0;
      t.n_n = 0;
      for (;;) {
        if (t.pos == 32) {
          t.base += 32;
          refill(t);
        }
        const int n = __shfl_sync(0xFFFFFFFFu, t.b_n, t.pos);
        if (n < 0) return;  // behind the last item
        if (n > 0) break;
        ++t.pos;
      }
      t.n_n = __shfl_sync(0xFFFFFFFFu, t.b_n, t.pos);
      t.n_head = __shfl_sync(0xFFFFFFFFu, t.b_head, t.pos);
      t.n_block = __shfl_sync(0xFFFFFFFFu, t.b_block, t.pos);
      t.n_part = __shfl_sync(0xFFFFFFFFu, t.b_part, t.pos);
      t.n_first = __shfl_sync(0xFFFFFFFFu, t.b_first, t.pos);
      ++t.pos;
      read_ids(t.n_head, t.n_block, t.n_first, t.n_n, 0, t.n_ids0, t.n_ids1);  // used an item later
    };
    auto start = [&](Feed& t, int s) {
      t.s = s;
      t.base = 0;
      t.item = t.tile = 0;
      t.pending = false;
      refill(t);
      t.n_n = 0;
      advance(t);
      advance(t);
    };
    auto load_tile = [&](int key, int kv_head, const CUtensorMap* map) {
      const int slot = issued % kRing;
      if (!mbar_wait_warp(&kv_empty[slot], ((issued / kRing) & 1) ^ 1, kErrSpProd)) return false;
      if (lane == 0) {
        uint8_t* dst = smem + kOffRing + slot * kTileBytes + u * (kSubKeys * 128);
        mbar_arrive_expect_tx(&kv_full[slot], kHalfBytes);
        for (int h = 0; h < 2; ++h)  // rows past the last key (and absent sub-blocks) arrive as zeros
          tma_load_3d(dst + h * kHalfBytes, map, &kv_full[slot], h * 64, key < 0 ? p.keys : key, kv_head);
      }
      ++issued;
      return true;
    };
    auto load_k = [&](Feed& t) {
      if (t.i == 0) {  // a new item: its queries, once the item before has used the buffer
        if (!mbar_wait_warp(&q_empty[t.s], (t.item & 1) ^ 1, kErrSpProd)) return false;
        if (lane == 0) {
          if (u == 0) item_note[t.s * kNotes + t.item % kNotes] = ItemNote{t.head, t.block, t.part, t.n};
          mbar_arrive_expect_tx(&q_full[t.s], kHalfBytes);
          tma_load_3d(smem + t.s * kTileBytes + u * kHalfBytes, &tm_q, &q_full[t.s], u * 64, t.block * kQueryBlock,
                      t.head);
        }
        ++t.item;
      }
      const int key0 = key_of(__shfl_sync(0xFFFFFFFFu, t.ids0, t.i & 31), 0);
      const int key1 = key_of(__shfl_sync(0xFFFFFFFFu, t.ids1, t.i & 31), 1);
      if (u == 0 && lane == 0) key_note[t.s * kNotes + t.tile % kNotes] = make_int2(key0, key1);
      ++t.tile;
      t.v_key = u == 0 ? key0 : key1;
      t.v_head = t.head / p.group;
      t.pending = true;
      if (!load_tile(t.v_key, t.v_head, &tm_k)) return false;
      if (++t.i == t.n)
        advance(t);
      else if ((t.i & 31) == 0)
        read_ids(t.head, t.block, t.first, t.n, t.i, t.ids0, t.ids1);
      return true;
    };
    start(a, 0);
    start(o, 1);
    // K of both streams' first tiles, then V and the next K of one stream after the other
#pragma unroll 1
    while (ok && (a.pending || a.n > 0 || o.pending || o.n > 0)) {
      if (a.pending) {
        a.pending = false;
        ok = load_tile(a.v_key, a.v_head, &tm_v);
      }
      if (ok && a.n > 0) ok = load_k(a);
      const Feed t = a;
      a = o;
      o = t;
    }
#pragma unroll 1
    for (int j = 0; j < 2; ++j) {  // issued copies land before exit
      const Feed& t = j ? o : a;
      if (t.item > 0) mbar_wait(&q_full[t.s], (t.item - 1) & 1, kErrSpDrain, 200000000ull);
    }
#pragma unroll 1
    for (int j = (issued > kRing ? issued - kRing : 0); j < issued; ++j)
      mbar_wait(&kv_full[j % kRing], (j / kRing) & 1, kErrSpDrain, 200000000ull);
  } else if (warp >= 9) {
    if (lane == 0) {
      // ---------------- MMA issuers: warp 9 + s serves stream s ----------------
      // An issuing thread is held until its instruction enters the (short) tensor queue,
      // so its waits for softmax and loads would leave the tensor core idle; with an
      // issuer per stream they run beside the other stream's products. The issuers take
      // turns (turn[s]: stream s has issued its t-th P V and next Q K^T): left to
      // themselves they interleave instruction by instruction, both softmaxes then start
      // together, and the exponentials of one no longer hide behind the products of the
      // other (2,126 us on the 21 x 39 x 40 grid, 24 heads, 64 of 512 blocks). Ring slots
      // keep the producers' order over both streams: an issuer counts past the other's tiles.
      constexpr uint32_t kIdescS = idesc_f16kind(F16, false), kIdescO = idesc_f16kind(F16, true);
      const int s = warp - 9, n = s ? n1 : n0, other = s ? n0 : n1;
      const uint32_t t_s = tmem + s * 128, t_o = tmem + 256 + s * 128;
      const uint64_t q_desc = umma_desc_sw128(smem_u32(smem + s * kTileBytes));
      const uint32_t ring = smem_u32(smem + kOffRing);
      int at = s == 1 && other > 0 ? 1 : 0;  // ring position of this stream's next tile
      int item = 0;                          // items whose scores have begun
      int opens = 1, left_s = 0;             // the next scores open an item; its tiles whose scores are to come
      auto loaded = [&](int pos) { return mbar_wait(&kv_full[pos % kRing], (pos / kRing) & 1, kErrSpMma); };
      auto queries_loaded = [&]() {
        if (!opens) return true;
        ++item;
        return mbar_wait(&q_full[s], (item - 1) & 1, kErrSpMma);
      };
      // scores of the next tile from ring position pos; `pass`: hand the turn over on the way
      auto scores = [&](int pos, bool pass) {
        const int slot = pos % kRing;
        if (opens) left_s = item_note[s * kNotes + (item - 1) % kNotes].n;
        opens = --left_s == 0;
        const uint64_t k_desc = umma_desc_sw128(ring + slot * kTileBytes);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
          umma_bf16(t_s, q_desc + off, k_desc + off, kIdescS, k > 0 ? 1u : 0u);
          if (pass && k == 5) mbar_arrive(&turn[s]);  // the other issuer wakes while the last ones run
        }
        umma_commit(&s_full[s]);
        umma_commit(&kv_empty[slot]);
        if (opens) umma_commit(&q_empty[s]);  // the item's last scores
      };
      bool ok = n > 0 && queries_loaded() && loaded(at);
      int left = 0;  // tiles of the current item whose P V is not issued
      if (ok) {
        tc_fence_after();
        scores(at, false);
        left = left_s + 1;
      }
      at = (n0 > 0 ? 1 : 0) + (n1 > 0 ? 1 : 0) + (s == 1 ? (other > 0 ? 1 : 0) + (other > 1 ? 1 : 0) : 0);
      bool first = true;  // of its item
      for (int i = 0; i < n && ok; ++i) {
        const int slot = at % kRing;
        const bool more = i + 1 < n;
        ok = loaded(at);
        if (more) ok = ok && queries_loaded() && loaded(at + 1);
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
            umma_f16_ts(t_o, t_s + k * 8, v_desc + ((k * 16 * 128) >> 4), kIdescO, !first || k > 0 ? 1u : 0u);
          if (h == 0) umma_commit(&h_done[s]);
        }
        if (!ok) break;
        first = --left == 0;  // the next tile opens an item
        if (first) umma_commit(&o_full[s]);
        if (more) {
          scores(at + 1, true);  // executes after the product above, which reads the columns it overwrites
          if (first) left = left_s + 1;
          // V and next K of this tile, then the other stream's: its tile i (stream 1) or i + 1 (stream 0)
          const int j = s == 0 ? i : i + 1;
          at += 2 + (j < other ? 1 : 0) + (j + 1 < other ? 1 : 0);
        } else {
          mbar_arrive(&turn[s]);
        }
        umma_commit(&kv_empty[slot]);
      }
    }
  } else {
    // ---------------- softmax: thread = row ----------------
    const int s = warp >> 2;
    const int row_in = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + s * 128 + lanes, t_o = tmem + 256 + s * 128 + lanes;
    const int total = s ? n1 : n0;
    ItemNote it;
    int i = 0, item = 0, row = 0, limit = 0;  // limit: keys this row may see
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int t = 0; t < total; ++t) {
      if (!mbar_wait_warp(&s_full[s], t & 1, kErrSpSoft)) {
        ok = false;
        break;
      }
      if (i == 0) {
        it = item_note[s * kNotes + item % kNotes];
        row = it.q_block * kQueryBlock + row_in;
        limit = p.causal ? min(p.keys, row + 1 + p.keys - p.queries) : p.keys;
        m = -INFINITY;
        l = 0.0f;
      }
      const int2 key = key_note[s * kNotes + t % kNotes];
      const int v0 = key.x < 0 ? 0 : limit - key.x, v1 = key.y < 0 ? 0 : limit - key.y;  // visible keys of the halves
      tc_fence_after();
      if (!__all_sync(0xFFFFFFFFu, v0 >= kSubKeys && v1 >= kSubKeys)) {
        // keys this row may not see: -inf, written back
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int seen = (c < 2 ? v0 : v1) - (c & 1) * 32;
          uint32_t x[32];
          tmem_ld32(t_s + c * 32, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (e >= seen) x[e] = 0xFF800000u;
          tmem_st32(t_s + c * 32, x);
        }
        tmem_wait_st();
      }
      if (i == 0) {  // the item's first maximum
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t x[32];
          tmem_ld32(t_s + c * 32, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mx[k] = max3(mx[k], __uint_as_float(x[e + 2 * k]), __uint_as_float(x[e + 2 * k + 1]));
        }
        m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      }
      // The weights of a half are computed with the maximum so far while its own maximum
      // is found beside them; only where that is more than 2^8 higher (or the first finite
      // score) are the sums so far rescaled and the half computed again.
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        uint32_t x[2][32], w[32];
        tmem_ld32(t_s + h * 64, x[0]);
        tmem_ld32(t_s + h * 64 + 32, x[1]);
        tmem_wait_ld();
        uint64_t sum[2];
#pragma unroll 1
        for (;;) {
          // in fp16 rounded down: from scores of 1e7 on, rounding to nearest is whole powers
          // of 2, which must not lift the largest weight over 65,504
          const float shift = m == -INFINITY ? SparseWeight<F16>::log2
                              : F16          ? __fmaf_rd(-m, p.scale_log2, SparseWeight<F16>::log2)
                                             : -(m * p.scale_log2);
          const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2), shift2 = f2_pack(shift, shift);
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          sum[0] = sum[1] = 0ull;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float y0 = __uint_as_float(x[e >> 4][2 * (e & 15)]), y1 = __uint_as_float(x[e >> 4][2 * (e & 15) + 1]);
            const uint64_t z = f2_fma(f2_pack(y0, y1), scale2, shift2);
            float a, b;
            if (e % kPolyOf == kPolyOf - 1) {
              exp2_poly2(z, a, b);
            } else {
              f2_unpack(z, a, b);
              a = ex2_approx(a);
              b = ex2_approx(b);
            }
            mx[e & 3] = max3(mx[e & 3], y0, y1);
            sum[e & 1] = f2_add(sum[e & 1], f2_pack(a, b));
            w[e] = E::pack(a, b);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const bool grow = (top - m) * p.scale_log2 > kRescaleLog2;
          if (!__any_sync(0xFFFFFFFFu, grow)) break;
          const float f = grow ? ex2_approx((m - top) * p.scale_log2) : 1.0f;
          if (grow) m = top;
          l *= f;
          // O holds what is complete: the tiles before (their commit came before s_full's)
          // and, for the second half, the first half's product
          if (h == 1) ok = mbar_wait_warp(&h_done[s], t & 1, kErrSpSoft) && ok;
          if (i > 0 || h == 1) {
            tc_fence_after();
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
        }
        float s0, s1, s2, s3;
        f2_unpack(sum[0], s0, s1);
        f2_unpack(sum[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
        tmem_st32(t_s + h * 32, w);  // over columns already read
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * s + h]);
      }
      if (++i < it.n) continue;
      // the item's last tile: its rows
      if (!mbar_wait_warp(&o_full[s], item & 1, kErrSpOut)) {
        ok = false;
        break;
      }
      tc_fence_after();
      i = 0;
      ++item;
      if (p.parts > 1) {
        const int64_t at = ((int64_t)(it.head * p.q_blocks + it.q_block) * p.parts + it.part) * kQueryBlock + row_in;
        if (row < p.queries) p.ws_ml[at] = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tmem_wait_ld();
          if (row < p.queries) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              stg_v8(p.ws_acc + at * kHeadDim + c * 32 + e, o[e], o[e + 1], o[e + 2], o[e + 3], o[e + 4], o[e + 5],
                     o[e + 6], o[e + 7]);
          }
          __syncwarp();
        }
      } else {
        const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays
        uint16_t* dst = p.out + (int64_t)row * p.o_t + (int64_t)it.head * p.o_h;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32], w[16];
          tmem_ld32(t_o + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            w[j] = l == 0.0f ? 0u : E::pack(__uint_as_float(o[2 * j]) * inv, __uint_as_float(o[2 * j + 1]) * inv);
          if (row < p.queries) {
            if (p.out32) {
              stg_v8(dst + c * 32, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
              stg_v8(dst + c * 32 + 16, w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15]);
            } else {
#pragma unroll
              for (int e = 0; e < 16; e += 4) stg_v4(dst + c * 32 + 2 * e, make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]));
            }
          }
          __syncwarp();
        }
        if (row < p.queries && p.lse != nullptr)
          p.lse[(int64_t)row * p.l_t + (int64_t)it.head * p.l_h] = l == 0.0f ? -INFINITY : fmaf(m, p.scale, logf(l * SparseWeight<F16>::inv));
      }
    }
    if (ok && empty_of[s]) {  // query blocks without any key
      for (int idx = blockIdx.x + gridDim.x * s; idx < p.items; idx += 2 * gridDim.x) {
        const Work w = work_of(p, idx);
        const int r = w.q_block * kQueryBlock + row_in;
        if (w.n > 0 || r >= p.queries) continue;
        if (p.parts > 1) {  // a part without tiles: l is 0, and the join reads no row
          p.ws_ml[((int64_t)(w.head * p.q_blocks + w.q_block) * p.parts + w.part) * kQueryBlock + row_in] =
              make_float2(-INFINITY, 0.0f);
          continue;
        }
        uint16_t* dst = p.out + (int64_t)r * p.o_t + (int64_t)w.head * p.o_h;
        for (int c = 0; c < kHeadDim; c += 8) stg_v4(dst + c, make_uint4(0u, 0u, 0u, 0u));
        if (p.lse != nullptr) p.lse[(int64_t)r * p.l_t + (int64_t)w.head * p.l_h] = -INFINITY;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 10) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// tiles[row] of each list: up to its last block that exists
__global__ void __launch_bounds__(128) count_tiles_kernel(const int32_t* blocks, int64_t rows, int top_k, int k_blocks,
                                                          int subs_per_block, int32_t* tiles) {
  launch_next();
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  int last = -1;
  for (int e = lane; e < top_k; e += 32) {
    const int id = __ldg(blocks + row * top_k + e);
    if (id >= 0 && id < k_blocks) last = e;
  }
  last = __reduce_max_sync(0xFFFFFFFFu, last);
  if (lane == 0) tiles[row] = list_tiles(last + 1, subs_per_block);
}

// Joins the parts of a query row: one warp per (row, head), in the order of the parts.
template <bool F16>
__global__ void __launch_bounds__(128) sparse_join_kernel(const SparseParams p) {
  using E = Elem16<F16>;
  wait_previous();
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (at >= (int64_t)p.heads * p.queries) return;
  const int lane = threadIdx.x & 31;
  const int head = (int)(at / p.queries), row = (int)(at - (int64_t)head * p.queries);
  const int64_t first = ((int64_t)(head * p.q_blocks + row / kQueryBlock) * p.parts) * kQueryBlock + row % kQueryBlock;
  float mx = -INFINITY;
  for (int s = lane; s < p.parts; s += 32) mx = fmaxf(mx, p.ws_ml[first + (int64_t)s * kQueryBlock].x);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, i));
  float sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s = 0; s < p.parts; ++s) {
    const float2 ml = p.ws_ml[first + (int64_t)s * kQueryBlock];
    if (ml.y == 0.0f) continue;  // no keys: nothing was written
    const float f = ex2_approx((ml.x - mx) * p.scale_log2);
    const float4 a = *(reinterpret_cast<const float4*>(p.ws_acc + (first + (int64_t)s * kQueryBlock) * kHeadDim) + lane);
    sum = fmaf(ml.y, f, sum);
    o.x = fmaf(a.x, f, o.x);
    o.y = fmaf(a.y, f, o.y);
    o.z = fmaf(a.z, f, o.z);
    o.w = fmaf(a.w, f, o.w);
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  uint2 y;
  y.x = E::pack(o.x * inv, o.y * inv);
  y.y = E::pack(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(p.out + (int64_t)row * p.o_t + (int64_t)head * p.o_h + lane * 4) = y;
  if (lane == 0 && p.lse != nullptr)
    p.lse[(int64_t)row * p.l_t + (int64_t)head * p.l_h] = sum == 0.0f ? -INFINITY : fmaf(mx, p.scale, logf(sum * SparseWeight<F16>::inv));
}

// Token and head strides as a tensor map takes them: a dim of one element has no stride that
// matters, but the encoder still checks it.
int64_t map_stride(int64_t count, int64_t stride) { return count == 1 ? kHeadDim : stride; }

bool view_maps(const void* base, int64_t rows, int64_t heads, int64_t st, int64_t sh) {
  for (const int64_t s : {map_stride(rows, st), map_stride(heads, sh)})
    if (s <= 0 || s % 8 || s * 2 >= (1ll << 40)) return false;  // a broadcast dim (stride 0) has no map
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0;
}

bool map_view(CUtensorMap* map, const void* base, int64_t rows, int64_t heads, int64_t st, int64_t sh, int box_rows) {
  st = map_stride(rows, st);
  sh = map_stride(heads, sh);
  return encode_tmap_3d_bf16(map, base, kHeadDim, (uint64_t)rows, (uint64_t)heads, (uint64_t)st * 2, (uint64_t)sh * 2,
                             64, (uint32_t)box_rows, 1, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool F16>
cudaError_t launch_sparse(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const SparseParams& p,
                          unsigned grid, int dev, bool chained, cudaStream_t stream) {
  static bool attr_set[64] = {false};
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(sparse_attention_kernel<F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSpSmem);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  const cudaError_t e =
      launch_chained(sparse_attention_kernel<F16>, grid, kSpThreads, kSpSmem, stream, chained, 1, q, k, v, p);
  if (e != cudaSuccess || p.parts == 1) return e;
  const int64_t warps = (int64_t)p.heads * p.queries;
  return launch_chained(sparse_join_kernel<F16>, (unsigned)((warps + 3) / 4), 128, 0, stream, true, 1, p);
}

// Runs a list is split into: as many as fill the streams of all SMs, of at least two tiles.
int64_t list_parts(int64_t items, int64_t tiles, int sms) {
  return std::max<int64_t>(1, std::min<int64_t>(tiles / 2, 2 * sms / items));
}

struct SparseShape {
  int64_t q_blocks, items, tiles, parts, tiles_bytes, acc_bytes, ml_bytes;
};
SparseShape sparse_shape(int64_t queries, int64_t heads, int64_t kv_heads, int64_t top_k, int64_t block, int sms) {
  SparseShape s;
  s.q_blocks = (queries + kQueryBlock - 1) / kQueryBlock;
  s.items = heads * s.q_blocks;
  s.tiles = (top_k * block + 127) / 128;
  s.parts = list_parts(s.items, s.tiles, sms);
  const int64_t rows = s.parts > 1 ? s.items * s.parts * kQueryBlock : 0;
  s.tiles_bytes = (kv_heads * s.q_blocks * 4 + 255) / 256 * 256;
  s.acc_bytes = rows * kHeadDim * 4;
  s.ml_bytes = rows * 8;
  return s;
}

}  // namespace

int64_t block_sparse_workspace_bytes(int64_t queries, int64_t heads, int64_t kv_heads, int64_t top_k, int64_t block,
                                     int sms) {
  const SparseShape s = sparse_shape(queries, heads, kv_heads, top_k, block, sms);
  return s.tiles_bytes + s.acc_bytes + s.ml_bytes;
}

cudaError_t check_block_sparse_attention(const SparseAttnArgs& a) {
  int dev = 0;
  cudaGetDevice(&dev);
  const SparseShape sh = sparse_shape(a.queries, a.heads, a.kv_heads, a.top_k, a.block, num_sms(dev));
  if (a.queries > (1 << 30) || a.keys > (1 << 30) || sh.items * sh.parts > (1 << 30) || a.block % kSubKeys ||
      a.o_t % 8 || a.o_h % 8 || (reinterpret_cast<uintptr_t>(a.out) & 15))
    return cudaErrorNotSupported;
  return view_maps(a.q, a.queries, a.heads, a.q_t, a.q_h) && view_maps(a.k, a.keys, a.kv_heads, a.k_t, a.k_h) &&
                 view_maps(a.v, a.keys, a.kv_heads, a.v_t, a.v_h)
             ? cudaSuccess
             : cudaErrorNotSupported;
}

cudaError_t launch_block_sparse_attention(const SparseAttnArgs& a, cudaStream_t stream) {
  if (a.queries <= 0 || a.heads <= 0) return cudaSuccess;
  const cudaError_t refused = check_block_sparse_attention(a);
  if (refused != cudaSuccess) return refused;
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = num_sms(dev);
  const SparseShape sh = sparse_shape(a.queries, a.heads, a.kv_heads, a.top_k, a.block, sms);
  CUtensorMap q, k, v;
  if (!map_view(&q, a.q, a.queries, a.heads, a.q_t, a.q_h, kQueryBlock) ||
      !map_view(&k, a.k, a.keys, a.kv_heads, a.k_t, a.k_h, kSubKeys) ||
      !map_view(&v, a.v, a.keys, a.kv_heads, a.v_t, a.v_h, kSubKeys))
    return cudaErrorNotSupported;
  SparseParams p;
  p.q_blocks = (int)sh.q_blocks;
  p.parts = (int)sh.parts;
  p.items = (int)(sh.items * sh.parts);
  p.blocks = a.blocks; p.top_k = (int)a.top_k; p.block = (int)a.block;
  p.k_blocks = (int)((a.keys + a.block - 1) / a.block);
  p.queries = (int)a.queries; p.keys = (int)a.keys; p.heads = (int)a.heads; p.group = (int)(a.heads / a.kv_heads);
  p.causal = a.causal ? 1 : 0;
  p.scale = a.scale; p.scale_log2 = a.scale * 1.4426950408889634f;
  p.out = static_cast<uint16_t*>(a.out); p.o_t = a.o_t; p.o_h = a.o_h;
  p.out32 = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.o_t * 2) | (uintptr_t)(a.o_h * 2)) & 31) == 0;
  p.lse = a.lse; p.l_t = a.l_t; p.l_h = a.l_h;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.ws_acc = reinterpret_cast<float*>(ws + sh.tiles_bytes);
  p.ws_ml = reinterpret_cast<float2*>(ws + sh.tiles_bytes + sh.acc_bytes);
  p.tiles = a.tiles;
  bool chained = a.chained;
  if (p.tiles == nullptr) {
    int32_t* tiles = reinterpret_cast<int32_t*>(ws);
    const int64_t rows = a.kv_heads * sh.q_blocks;
    const cudaError_t e =
        launch_chained(count_tiles_kernel, (unsigned)((rows + 3) / 4), 128, 0, stream, false, 1, a.blocks, rows, p.top_k,
                       p.k_blocks, p.block / kSubKeys, tiles);
    if (e != cudaSuccess) return e;
    chained = true;
    p.tiles = tiles;
  }
  // one persistent CTA per SM; a second stream only where every SM has a first one
  const unsigned grid = (unsigned)std::min<int64_t>(sms, p.items);
  return a.f16 ? launch_sparse<true>(q, k, v, p, grid, dev, chained, stream)
               : launch_sparse<false>(q, k, v, p, grid, dev, chained, stream);
}

}  // namespace h3
