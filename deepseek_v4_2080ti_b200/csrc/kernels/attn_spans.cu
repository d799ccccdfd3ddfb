// Attention over the paged bf16 cache (head width 128) in which every query row sees a span of keys of its own, sm_100a.
//
//   s_ij = scale q_i . k_j, with a cap c > 0: s = c tanh(s / c); o_i = sum_j softmax_j(s_ij) v_j over lo_i <= j < hi_i
//
// in three forms over one kernel: prompt rows (b200_attn_spans: packed documents, prefixes, blocks of an image that see each
// other, windows, causal rows after a context), one row per sequence where groups of sequences hold the same leading pages
// (b200_attn_shared: those keys are read and multiplied once for the whole group) and the rows of a drafted tree (b200_attn_tree: the
// context, and of the tree's own keys, the last of the sequence, those whose bit is set in the row's mask).  A row that sees nothing is
// zero; a masked key takes no part whatever its bits are.
//
// Work is a list of items, a block of the launch each: as many as there are SMs run, and one that is ready for more cancels a block that
// has not begun and takes its item (cluster launch control; against a fixed deal 16 ragged portions take 126 us instead of 163, 8192 causal
// rows 627 instead of 636; asking one item ahead would cost 1 to 7 %): 256 rows (token, head of one kv head) - all query
// heads of a kv head are packed into the rows, so a tile is full however few tokens there are - times a range of key tiles of
// 128.  A row's result comes from one item, or from several whose partial sums (fp32) the second kernel here, or the one over
// the sequences' own keys, joins.
//
// Two streams of 128 rows keep the tensor core and the exponential units busy in turn.  An item of at most 128 rows gives both
// streams the same rows and every other key tile, and joins them at its end.  Warp roles:
//   warps 0-3, 4-7: softmax of stream 0 and 1 - one row per thread, online maximum / sum in the exp2 domain (fp32), P rounded to
//             bf16 for the product (2^-8 of a weight at most; the sum adds the weights before they are rounded) into the tensor
//             memory its scores came from, lazy rescale of the stream's O (when a maximum grows by 2^8); then the item's rows;
//   warp 8  : items - which rows and keys are next, up to four ahead of the slowest role - and their loads: key and value tiles
//             gathered page by page through the block table into one ring (TMA), running ahead into the next item;
//   warp 9  : tcgen05.mma issuer - step u: P V of step u, scores of step u + 2 (steps alternate between the streams);
//   warp 10 : value check of tiles with masked keys - rows that are not there (behind the last key) or not finite are set to
//             zero, because 0 x inf in a product would reach rows that do not see them; rows that do see a key with values that
//             are not finite add it themselves;
//   warp 11 : nothing (a warpgroup gives its registers up as a whole).
// Tensor memory: S0 | S1 | O0 | O1, 128 columns each.  All mbarrier waits are bounded and unwind through the common exit.
//
// What bounds it (8192 causal rows of 40 heads over 8 kv heads, gated: 628 us, 1.1 PFLOP/s): 256 rows times 128 keys cost 2048
// cycles of the tensor core and about 2100 of each scheduler's softmax warps, and take 3500 together, because a stream's scores,
// weights and products follow each other through tensor memory and two streams do not hide all of that; an item's start and end
// take another 10 %.  Packed documents of 4000 rows of 48 heads, capped: 110 us, a third of it the start and end of items, and of the
// rest most masked tiles (6000 cycles).
// Shared keys of 40 heads over 8, in one item a block: 64 rows over 32768 keys 44 us, 32 over 8192 15 us.
// Trees of 40 heads over 8: 32 of 64 nodes over 8192 keys 475 to 571 us, where the second row tile of 64 rows reads the keys from DRAM
// once more (2.2 GB; begun beside the first it gains nothing) and 512 items are 3.5 rounds of blocks; 32 of 25 nodes 193 to 199 us, 5.4 to 5.6
// TB/s; one of 16 over 32768 keys 37 us, 20 of them the keys.  The smallest, 7 nodes over 350 keys, is a chain of 18 thousand cycles: the item 2.8,
// queries 1.5, first scores 1, three tiles 7.5 (the last one masked), the rows' way out 5.2.
#include <cuda_bf16.h>
#include "per_device.h"
#include "../ptx/sm100.cuh"
#include "score_cap.cuh"
#include "tma_host.h"
#include "launch.h"
#include "ops.h"

namespace b200 {
namespace spans {

constexpr int D = 128;
constexpr int BQ = 128;           // rows per stream
constexpr int BKV = 128;          // keys per tile
constexpr int ATOM = 16384;       // bytes of one [128 x 64] bf16 swizzled slab
constexpr int TILE = 2 * ATOM;
constexpr int STAGES = 5;
constexpr int EMULATED = 2;       // of 8 pairs of exponentials: those on the arithmetic units (0 / 1 / 2 / 3: 641 / 639 / 624 / 626 us for 8192 causal rows)
constexpr int ITEMS = 4;          // items the producer may be ahead of the slowest role
constexpr int NTHREADS = 384;
constexpr int SMEM_BYTES = 1024 + (2 + STAGES) * TILE + 2048;
static_assert(SMEM_BYTES <= 232448, "shared memory of a block");

struct Params {
  const __nv_bfloat16* q;         // [T, Hq, 128]
  const __nv_bfloat16* gate;      // optional [T, Hq, 128]
  __nv_bfloat16* out;             // [T, Hq, 128]
  const __nv_bfloat16* v_cache;
  const int* block_table;         // [B, max_blocks]
  const int* kv_len;              // [B]
  // prompt rows
  const int* q_start;             // [B]
  const int* q_len;               // [B]
  const int* lo;                  // optional [T]
  const int* hi;                  // optional [T]
  const uint32_t* tree;           // rows of a tree: [T, tree_words], bit i: node i is seen
  int tree_words;
  // one row per sequence
  const int* group_start;         // [n_groups + 1]
  const int* shared_len;          // [n_groups]
  int n_groups;
  float* part_o;                  // [slots, T, Hq, 128], null: every row has one item
  float* part_ml;                 // [slots, T, Hq, 2]
  int batch, T, max_blocks, num_blocks, bs, bs_log2, Hq, Hkv, G;
  int row_tiles;                  // of a sequence, at most (prompt rows)
  // Prompt rows: the items of one sequence after those of another, with no places for tiles that a sequence does not have; else by their place
  // in the sequences, the last first - long ones before short ones, neighbours of different sequences.  8 sequences of 1000 rows, 40
  // heads: 166 / 146 us; 16 of 7 to 757: 135 / 126; one of 2000 beside 63 single rows: 91 / 161, which decides where more than
  // half of the places would be empty.
  int by_sequence;
  int splits;                     // key ranges per row tile
  int n_items;
  float scale_log2;               // scale * log2(e)
  float cap_in, cap_out;          // scale / cap, cap * log2(e)
  float cap_small;                // scores to which cap_c reach: half of cap / scale, 0 where the powers of scale / cap leave 32 bits
  float4 cap_c;                   // tanh(cap_in s) = s (c.x + c.y s^2 + c.z s^4 + c.w s^6)
  int* status;
};

// MN-major operand, 128-byte swizzle: 64-element MN atoms LBO bytes apart, 8-row K groups SBO bytes apart.
__device__ __forceinline__ uint64_t desc_mn_sw128(const void* p, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_u32(p) & 0x3FFFF) >> 4);
  d |= (uint64_t)(lbo >> 4) << 16;
  d |= (uint64_t)(sbo >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t idesc_qk = umma_idesc_bf16(128, 128);
constexpr uint32_t idesc_pv = umma_idesc_bf16(128, 128) | (1u << 16);   // B is MN-major

__device__ __forceinline__ void tmem_ld_32x2(uint32_t taddr, uint32_t& v, uint32_t& w) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(v), "=r"(w) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_32x2(uint32_t taddr, uint32_t v, uint32_t w) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(taddr), "r"(v), "r"(w) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x1(uint32_t taddr, uint32_t& v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
}
// mbar_wait for a whole warp, each lane on a barrier of its own if it likes: no lane leaves the loop before the others, so that the
// warp stays converged (its addresses and ring places are in uniform registers).  false: not all phases have come in time.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  uint64_t t0 = 0;
  for (uint32_t n = 1;; ++n) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((n & 255) == 0) {
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (__any_sync(0xffffffffu, now - t0 > B200_WAIT_BUDGET_NS)) return false;
    }
  }
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      :
      : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// The launch's blocks that have not begun are the list of items that are left: a block takes the next one by cancelling it.  The answer
// comes into 16 bytes of shared memory and completes a phase of `bar`; a block whose request found none left makes no other.
__device__ __forceinline__ void request_block(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int requested_block(const void* answer) {           // -1: none was left
  uint64_t a, b;
  int x;
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(smem_u32(answer)) : "memory");
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred got;\n\tmov.b128 h, {%1, %2};\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 got, h;\n\t"
      "mov.s32 %0, -1;\n\t"
      "@got clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}"
      : "=r"(x)
      : "l"(a), "l"(b));
  return x;
}
__device__ __forceinline__ void l2_prefetch(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy16_async(void* smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(src) : "memory");
}
// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of two numbers below 128 on the arithmetic units: 2^round(x) by the exponent bits, 2^f of the rest, |f| <= 1/2, by a cubic with
// constant term 1 (fitted to the relative error, 1e-4: P is rounded to 2^-8).  From -127 down the result is exactly zero.  Not for NaN.
__device__ __forceinline__ void exp2_fma(float& a, float& b) {
  constexpr float BIG = 12582912.f;                          // 1.5 2^23: the sum's low bits are the rounded integer
  constexpr float E1 = 0.693282961845398f, E2 = 0.24221111834049225f, E3 = 0.05500898137688637f;
  const uint64_t x = pack2(fmaxf(a, -127.f), fmaxf(b, -127.f));
  const uint64_t r = add2(x, pack2(BIG, BIG));
  const uint64_t f = add2(x, fma2(r, pack2(-1.f, -1.f), pack2(BIG, BIG)));
  uint64_t y = fma2(f, pack2(E3, E3), pack2(E2, E2));
  y = fma2(y, f, pack2(E1, E1));
  y = fma2(y, f, pack2(1.f, 1.f));
  float r0, r1, y0, y1;
  unpack2(r, r0, r1);
  unpack2(y, y0, y1);
  a = __int_as_float(__float_as_int(y0) + (__float_as_int(r0) << 23));
  b = __int_as_float(__float_as_int(y1) + (__float_as_int(r1) << 23));
}

// One piece of work; the same in every thread of a warp.
struct Item {
  int n_rows;            // rows of the tile that are there (0: the list has ended)
  int r0;                // first of them among the packed rows of base_tok
  int base_tok;          // q row of packed row 0
  int kvh, trow, slot;   // kv head; row of the block table; slot of the partial sums
  int t0, t1;            // key tiles
  int lo_max, hi_min;    // keys in [lo_max, hi_min) are seen by every row
  int k_end;             // first key that no row sees
  int kv_end;            // keys of the sequence
  int own_hi;            // shared keys: end of the rows' span; trees: position of node 0
  int delta;             // position of a token minus its q row (prompt rows)
  int tok0, tok1;        // tokens of the rows
  __device__ __forceinline__ bool dual() const { return n_rows <= BQ; }
  __device__ __forceinline__ int steps() const { return dual() ? t1 - t0 : 2 * (t1 - t0); }
};

enum Form { SPANS, SHARED_KEYS, TREE_ROWS };

template <Form FORM>
__device__ __forceinline__ void span_of(const Params& p, const Item& it, int tok, int& lo, int& hi) {
  if (FORM == SHARED_KEYS) {
    lo = 0;
    hi = max(0, min(it.own_hi, min(p.kv_len[tok], p.max_blocks * p.bs)));
  } else {
    lo = p.lo ? max(0, p.lo[tok]) : 0;
    hi = FORM == TREE_ROWS ? it.kv_end : max(0, min(p.hi ? p.hi[tok] : tok + it.delta + 1, it.kv_end));    // (differences of these fit 32 bits)
  }
}

// Which of the 32 keys from `key` on a tree's row sees by its mask, node 0 lying at position `first`: all in the context.
__device__ __forceinline__ uint32_t tree_bits(const uint32_t* words, int n_words, int key, int first) {
  const int at = key - first;
  if (at <= -32) return 0xffffffffu;
  auto word = [&](int i) { return i >= 0 && i < n_words ? words[i] : i < 0 ? 0xffffffffu : 0u; };
  return __funnelshift_r(word(at >> 5), word((at >> 5) + 1), at & 31);
}

// Item `idx` of the list; false: there is nothing to do.  Called by whole warps.
template <Form FORM>
__device__ __forceinline__ bool get_item(const Params& p, int idx, int lane, Item& it) {
  it.n_rows = 0;
  int split, splits;
  int rows_all;
  if (FORM == SHARED_KEYS) {
    // A group's rows are whole tiles and a rest; a rest of at most 128 rows takes half the time per key (both streams work on it), so its
    // keys are cut into half as many items.
    const int few = (p.splits + 1) / 2;
    int y = idx, b0 = 0, rows = -1, shared = 0;
    for (int base = 0; base < p.n_groups && rows < 0; base += 32) {      // a group per lane
      const int g = base + lane;
      int first = 0, n = 0, sh = 0;
      if (g < p.n_groups) {
        first = max(0, min(p.batch, p.group_start[g]));
        n = max(0, min(p.batch, p.group_start[g + 1]) - first) * p.G;
        sh = p.shared_len[g];
      }
      const int rest = n % (2 * BQ), tiles = n / (2 * BQ) + (rest > BQ);
      const int items = sh > 0 ? p.Hkv * (tiles * p.splits + (rest > 0 && rest <= BQ ? few : 0)) : 0;
      int upto = items;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int before = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += before;
      }
      const uint32_t here = __ballot_sync(0xffffffffu, y < upto);
      if (here) {
        const int src = __ffs(here) - 1;
        b0 = __shfl_sync(0xffffffffu, first, src);
        rows = __shfl_sync(0xffffffffu, n, src);
        shared = __shfl_sync(0xffffffffu, sh, src);
        y -= __shfl_sync(0xffffffffu, upto - items, src);
      } else {
        y -= __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (rows < 0) return false;
    const int tiles = rows / (2 * BQ) + (rows % (2 * BQ) > BQ), whole = p.Hkv * tiles * p.splits;
    const bool last = y >= whole;                          // the rest
    splits = last ? few : p.splits;
    if (last) y -= whole;
    const uint32_t z = (uint32_t)y / (uint32_t)splits, head = z / (uint32_t)p.Hkv;       // (unsigned: a third of the code)
    split = y - (int)z * splits;
    it.kvh = (int)(z - head * p.Hkv);
    const int tile = last ? tiles : (int)head;
    it.slot = split;
    it.base_tok = it.trow = b0;
    it.r0 = tile * 2 * BQ;
    rows_all = rows;
    it.own_hi = shared;
    it.kv_end = p.max_blocks * p.bs;
    it.delta = 0;
  } else {
    splits = p.splits;
    int y = idx, b = -1, q0 = 0, n = 0, kv = 0, len = 0, tile = -1;
    if (p.by_sequence) {
      for (int base = 0; base < p.batch && b < 0; base += 32) {              // a sequence per lane
        int q0_ = 0, n_ = 0, kv_ = 0, len_ = 0;
        if (base + lane < p.batch) {
          q0_ = p.q_start[base + lane];
          n_ = p.q_len[base + lane];
          kv_ = p.kv_len[base + lane];
          len_ = q0_ < 0 ? 0 : max(0, min(n_, p.T - q0_));
        }
        const int items = (len_ * p.G + 2 * BQ - 1) / (2 * BQ) * p.Hkv * splits;
        int upto = items;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int before = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += before;
        }
        const uint32_t here = __ballot_sync(0xffffffffu, y < upto);
        if (here) {
          const int src = __ffs(here) - 1;
          b = base + src;
          q0 = __shfl_sync(0xffffffffu, q0_, src);
          n = __shfl_sync(0xffffffffu, n_, src);
          kv = __shfl_sync(0xffffffffu, kv_, src);
          len = __shfl_sync(0xffffffffu, len_, src);
          y -= __shfl_sync(0xffffffffu, upto - items, src);
        } else {
          y -= __shfl_sync(0xffffffffu, upto, 31);
        }
      }
      if (b < 0) return false;
    } else {
      const uint32_t x = (uint32_t)idx / (uint32_t)(splits * p.Hkv), z = x / (uint32_t)p.batch;
      b = (int)(x - z * p.batch);
      y = idx - (int)x * splits * p.Hkv;
      tile = FORM == TREE_ROWS ? (int)z : p.row_tiles - 1 - (int)z;        // long contexts first; of a tree's rows, which all see the context, full tiles
      q0 = p.q_start[b];
      n = p.q_len[b];
      kv = p.kv_len[b];
      len = q0 < 0 ? 0 : max(0, min(n, p.T - q0));
    }
    rows_all = len * p.G;
    const uint32_t x = (uint32_t)y / (uint32_t)splits, z = x / (uint32_t)p.Hkv;
    split = y - (int)x * splits;
    it.kvh = (int)(x - z * p.Hkv);
    it.slot = split;
    it.r0 = (!p.by_sequence ? tile : FORM == TREE_ROWS ? (int)z : (rows_all + 2 * BQ - 1) / (2 * BQ) - 1 - (int)z) * 2 * BQ;
    it.trow = b;
    it.base_tok = q0;
    it.kv_end = max(0, min(kv, p.max_blocks * p.bs));
    it.delta = kv - n - q0;
    it.own_hi = kv - n;
  }
  it.n_rows = min(2 * BQ, rows_all - it.r0);
  if (it.n_rows <= 0) return false;
  const int tok0 = it.base_tok + (int)((uint32_t)it.r0 / (uint32_t)p.G), tok1 = it.base_tok + (int)((uint32_t)(it.r0 + it.n_rows - 1) / (uint32_t)p.G);
  it.tok0 = tok0;
  it.tok1 = tok1;
  int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = 0;
  for (int t = tok0 + lane; t <= tok1; t += 32) {
    int lo, hi;
    span_of<FORM>(p, it, t, lo, hi);
    lo_max = max(lo_max, lo);
    hi_min = min(hi_min, hi);
    if (lo < hi) {
      lo_min = min(lo_min, lo);
      hi_max = max(hi_max, hi);
    }
  }
  lo_min = __reduce_min_sync(0xffffffffu, lo_min);
  it.lo_max = __reduce_max_sync(0xffffffffu, lo_max);
  it.hi_min = __reduce_min_sync(0xffffffffu, hi_min);
  if (FORM == TREE_ROWS) it.hi_min = min(it.hi_min, it.own_hi);            // (of the tree's keys every row sees its own)
  it.k_end = __reduce_max_sync(0xffffffffu, hi_max);
  it.t0 = it.t1 = 0;
  if (it.k_end > lo_min) {
    // Ranges by the keys that are there, not by what the host knows of them: a captured step's bound, or the table's width, is often far above its
    // contexts, and a window leaves few keys of them.  (16 nodes over 4000 keys with a bound of 4016 / 32768 / 131072: 16.2 / 17.1 / 17.0 us, with ranges
    // of a length that follows from the bound 16.1 / 25.3 / 42.6; over 32768 keys in a window of 4096: 16.6, and 26.6.  Ranges of at least 2, 3 or 4
    // tiles gain nothing.)
    const int a = lo_min / BKV, n = (it.k_end + BKV - 1) / BKV - a, per = (int)((uint32_t)(n + splits - 1) / (uint32_t)splits);
    it.t0 = a + min(n, split * per);
    it.t1 = a + min(n, (split + 1) * per);
  }
  return true;
}

static_assert(sizeof(Item) == 64, "copied as four 16-byte words");

template <int N>
struct Int {
  static constexpr int value = N;
};

struct Ring {
  int st;
  uint32_t ph;
  __device__ __forceinline__ void next() {
    if (++st == STAGES) { st = 0; ph ^= 1; }
  }
  __device__ __forceinline__ void skip(int n) {
    const int s = st + n, w = s / STAGES;
    st = s - w * STAGES;
    ph ^= w & 1;
  }
  __device__ __forceinline__ void two() {
    st += 2;
    if (st >= STAGES) { st -= STAGES; ph ^= 1; }
  }
};

template <Form FORM, bool CAP>
__global__ void __launch_bounds__(NTHREADS, 1)
spans_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_base[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_base) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                       // [2 streams] tiles; then gates and results
  uint8_t* sR = smem + 2 * TILE;                            // ring of key and value tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(sR + STAGES * TILE);
  // Stages are given back by place in the ring, but filled by tile: a stage holds keys and values in turn, loads finish in any order, and
  // a role that waits for the values alone would take the phase of two loads ago for the one it waits for.
  uint64_t* r_empty = bars;
  uint64_t* k_full = bars + STAGES;                         // by tile, modulo STAGES (never more than three tiles are on their way)
  uint64_t* v_full = bars + 2 * STAGES;
  uint64_t* v_ok = bars + 3 * STAGES;                       // values checked
  uint64_t* q_full = bars + 4 * STAGES;                     // per stream: queries there, O zero
  uint64_t* s_full = q_full + 2;
  uint64_t* p_half = q_full + 4;                            // P of the tile's first 64 keys
  uint64_t* p_full = q_full + 6;
  uint64_t* o_full = q_full + 8;
  uint64_t* j_full = q_full + 10;                           // per stream, where both have a part of every row: its part is ready,
  uint64_t* j_empty = q_full + 12;                          // and it has read the other's
  uint64_t* i_full = q_full + 14;                           // items
  uint64_t* i_empty = i_full + ITEMS;
  uint64_t* pv_half = i_empty + ITEMS;                      // per stream: the product with the values of a tile's first 64 keys
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_half + 2);
  uint64_t* next_full = pv_half + 3;                        // the block that was asked for
  uint4* s_next = reinterpret_cast<uint4*>(bars + 48);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(bars + 52); // [STAGES][4] keys with values that are not finite
  Item* s_item = reinterpret_cast<Item*>(bars + 62);        // [ITEMS]

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform: the issuer depends on it
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&r_empty[i], 1);
      mbar_init(&v_ok[i], 1);
    }
    for (int m = 0; m < 2; ++m) {
      mbar_init(&q_full[m], 4);
      mbar_init(&s_full[m], 1);
      mbar_init(&p_half[m], 4);
      mbar_init(&p_full[m], 4);
      mbar_init(&o_full[m], 1);
    }
    for (int i = 0; i < ITEMS; ++i) {
      mbar_init(&i_full[i], 1);
      mbar_init(&i_empty[i], 10);
    }
    for (int m = 0; m < 2; ++m) mbar_init(&pv_half[m], 1);
    mbar_init(next_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&j_full[i], 4);
      mbar_init(&j_empty[i], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_wait();
  pdl_launch_dependents();                                  // (after the wait: the kernel that joins shared keys begins with what this one reads)

  Item it;
  // The next item, in shared memory: every role but the producer, which has put it there.
  int i_at = 0;
  uint32_t i_ph = 0;
  auto next_item = [&]() -> bool {
    bool ok = warp_wait(&i_full[i_at], i_ph) && !*abort_flag;
    if (!ok) return false;
    const int4* src = reinterpret_cast<const int4*>(s_item + i_at);
    int4* dst = reinterpret_cast<int4*>(&it);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = src[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(&i_empty[i_at]);
    if (++i_at == ITEMS) { i_at = 0; i_ph ^= 1; }
    return true;
  };
  // registers per thread at launch: 168 (3 x 168 = 2 x 224 + 56)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    Ring r = {0, 0}, c = {0, 0};                           // a stage; a tile
    bool ok = true;
    if (warp == 8) {
      const int rows = min(p.bs, BKV), rows_log2 = 31 - __clz(rows), per_tile = BKV >> rows_log2;              // pages (or parts of one) in a tile
      const uint32_t sub_bytes = rows * 128;                               // one 64-column half of one
      if (lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
      }
      r.ph = 1;
      auto hand_out = [&]() {
        ok = warp_wait(&i_empty[i_at], i_ph ^ 1) && !*abort_flag;
        if (!ok) return;
        if (lane == 0) {
          int4* dst = reinterpret_cast<int4*>(s_item + i_at);
          const int4* src = reinterpret_cast<const int4*>(&it);
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[i] = src[i];
          mbar_arrive(&i_full[i_at]);
        }
        if (++i_at == ITEMS) { i_at = 0; i_ph ^= 1; }
      };
      int idx = blockIdx.x;
      uint32_t ph_next = 0;
      auto next_block = [&]() {                            // cancels a block that has not begun; idx: its number, -1 if there is none
        idx = -1;
        if (lane == 0) {
          mbar_expect_tx(next_full, 16);
          request_block(s_next, next_full);
        }
        __syncwarp();
        if (!warp_wait(next_full, ph_next)) return false;
        ph_next ^= 1;
        idx = requested_block(s_next);
        fence_proxy_async_smem();                          // read before the next answer is written
        __syncwarp();
        return true;
      };
      while (idx >= 0) {
        if (get_item<FORM>(p, idx, lane, it)) {
        const int* bt = p.block_table + (size_t)it.trow * p.max_blocks;
        const int last_page = (it.k_end - 1) >> p.bs_log2;
        auto page_row = [&](int tile) {                                    // cache row where this lane's part of a tile begins
          const int key = tile * BKV + (lane << rows_log2);
          const int page = min(key >> p.bs_log2, last_page);
          if (tile >= it.t1 || lane >= per_tile) return 0;
          // a page that is not there (an entry before the first key that is seen, or a bad one) lies behind the cache: it reads as zeros
          const int id = min((unsigned)bt[page], (unsigned)p.num_blocks);
          return ((id * p.Hkv + it.kvh) << p.bs_log2) + (key & (p.bs - 1));
        };
        int row = page_row(it.t0);                         // (on its way while the item is handed out)
        hand_out();
        for (int t = it.t0; ok && t < it.t1; ++t) {
          const int n = min(per_tile, (it.k_end - t * BKV + rows - 1) >> rows_log2);
          const int next_row = page_row(t + 1);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok = warp_wait(&r_empty[r.st], r.ph) && !*abort_flag;
            if (!ok) break;
            uint64_t* full = (kv ? v_full : k_full) + c.st;
            if (lane == 0) mbar_expect_tx(full, n * 2 * sub_bytes);
            __syncwarp();
            if (lane < n) {
              uint8_t* dst = sR + r.st * TILE + lane * sub_bytes;
              tma_load_2d(dst, kv ? &tmV : &tmK, full, 0, row);
              tma_load_2d(dst + ATOM, kv ? &tmV : &tmK, full, 64, row);
            }
            r.next();
          }
          row = next_row;
          c.next();
          if (t == it.t0) {                                // queries and gate of items ahead on their way to L2
            for (int y = it.tok0 + lane; y <= it.tok1; y += 32) {
              const size_t at = ((size_t)y * p.Hq + it.kvh * p.G) * D;
              l2_prefetch(p.q + at, p.G * D * 2);
              if (p.gate && !p.part_o) l2_prefetch(p.gate + at, p.G * D * 2);
            }
          }
        }
        }
        // the next one only now, when this one's tiles are all on their way: blocks that are ahead take more
        if (!ok || !(ok = next_block())) break;
      }
      if (ok) {
        it.n_rows = 0;
        hand_out();
      }
      // A launch whose waits have run out ends: its blocks that have not begun are cancelled, so that they do not wait as well.  (The error
      // word does not tell: it is the device's, and may hold what another kernel has reported.)
      if (!ok) {
        if (lane == 0) { atomicExch(p.status, ERR_WAIT_STAGE); *abort_flag = 1; }
        while (idx >= 0 && next_block()) {}
      }
    } else if (warp == 9) {
      // The whole warp walks the loop, so that addresses and descriptors stay warp-uniform, and one elected lane issues.  What a step
      // costs beside the products is as long as they are if it is not kept short: even lanes wait for one barrier while odd lanes
      // wait for another, and what the streams share is waited for once.
      const uint32_t on = elect_one();
      auto wait2 = [&](uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
        ok = warp_wait(lane & 1 ? b : a, lane & 1 ? pb : pa);
        return ok;
      };
      const uint64_t dq0 = umma_desc_sw128(sQ), dk = umma_desc_sw128(sR), dv = desc_mn_sw128(sR, ATOM, 1024);
      uint32_t ph_q[2] = {0, 0}, ph_p[2] = {0, 0};
      Ring k = {0, 0}, v = {1, 0}, kt = {0, 0};            // stages of the next key tile and the next value tile; the next key tile
      for (;;) {
        if (ok) ok = next_item();
        if (!ok || it.n_rows == 0) break;
        const int steps = it.steps();
        if (steps == 0) continue;
        const bool dual = it.dual();
        auto scores = [&](const int m) {                   // of the tile at k, which is there
          const uint64_t a = dq0 + (dual ? 0 : m * (TILE >> 4)), b = dk + k.st * (TILE >> 4);
#pragma unroll
          for (int s = 0; s < 8; ++s)
            umma_bf16_ss_warp(on, tmem + m * 128, a + (s >> 2) * (ATOM >> 4) + 2 * (s & 3), b + (s >> 2) * (ATOM >> 4) + 2 * (s & 3), idesc_qk,
                              s ? 1u : 0u);
          umma_commit_warp(on, &s_full[m]);
          if (dual || m) {
            umma_commit_warp(on, &r_empty[k.st]);
            k.two();
            kt.next();
          }
        };
#pragma unroll
        for (int m = 0; m < 2; ++m)
          if (ok && m < steps && wait2(&q_full[m], ph_q[m], &k_full[kt.st], kt.ph)) {
            ph_q[m] ^= 1;
            tc_fence_after();
            scores(m);
          }
        for (int u0 = 0; ok && u0 < steps; u0 += 2) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const int u = u0 + m;
            if (!ok || u >= steps) break;
            if (!wait2(&p_half[m], ph_p[m], &v_ok[c.st], c.ph)) break;
            tc_fence_after();
            const uint64_t b = dv + v.st * (TILE >> 4);
#pragma unroll
            for (int s = 0; s < 4; ++s) umma_bf16_ts_warp(on, tmem + 256 + m * 128, tmem + m * 128 + s * 8, b + s * 128, idesc_pv, 1u);
            umma_commit_warp(on, &pv_half[m]);
            const bool more = u + 2 < steps;
            if (!wait2(&p_full[m], ph_p[m], more ? &k_full[kt.st] : &p_full[m], more ? kt.ph : ph_p[m])) break;
            ph_p[m] ^= 1;
            tc_fence_after();
#pragma unroll
            for (int s = 4; s < 8; ++s) umma_bf16_ts_warp(on, tmem + 256 + m * 128, tmem + m * 128 + s * 8, b + s * 128, idesc_pv, 1u);
            if (dual || m) {
              umma_commit_warp(on, &r_empty[v.st]);
              v.two();
              c.next();
            }
            if (more) scores(m);
            else umma_commit_warp(on, &o_full[m]);
          }
        }
      }
      if (!ok && lane == 0) { atomicExch(p.status, ERR_WAIT_TMA); *abort_flag = 1; }
    } else if (warp == 10) {
      for (;;) {
        if (ok) ok = next_item();
        if (!ok || it.n_rows == 0) break;
        for (int t = it.t0; ok && t < it.t1; ++t) {
          r.next();
          ok = warp_wait(&v_full[c.st], c.ph) && !*abort_flag;
          if (!ok) break;
          const int key0 = t * BKV;
          if (key0 < it.lo_max || key0 + BKV > it.hi_min) {
            bool wrote = false;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
              const int key = i * 32 + lane;
              uint8_t* row = sR + r.st * TILE + key * 128;
              const bool there = key0 + key < it.k_end;
              uint32_t acc = 0;
              if (there) {
#pragma unroll 8
                for (int d = 0; d < 16; ++d) {
                  const uint4 x = *reinterpret_cast<const uint4*>(row + (d >> 3) * ATOM + (((d & 7) ^ (key & 7)) << 4));
                  // bit 15 / 31 where an exponent is all ones
                  acc |= ((x.x & 0x7F807F80u) + 0x00800080u) | ((x.y & 0x7F807F80u) + 0x00800080u) | ((x.z & 0x7F807F80u) + 0x00800080u) |
                         ((x.w & 0x7F807F80u) + 0x00800080u);
                }
              }
              const bool bad = (acc & 0x80008000u) != 0;
              const uint32_t mask = __ballot_sync(0xffffffffu, bad);
              if (lane == 0) s_bad[c.st * 4 + i] = mask;
              if (bad || !there) {
                wrote = true;
#pragma unroll
                for (int d = 0; d < 16; ++d) *reinterpret_cast<uint4*>(row + (d >> 3) * ATOM + ((d & 7) << 4)) = make_uint4(0, 0, 0, 0);
              }
            }
            if (wrote) fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ok[c.st]);
          r.next();
          c.next();
        }
      }
      if (!ok && lane == 0) { atomicExch(p.status, ERR_WAIT_STAGE); *abort_flag = 1; }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int m = warp >> 2;                               // stream
    const int lr = threadIdx.x & 127;                      // row of the stream == TMEM lane
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + m * 128 + lane_off, tO = tmem + 256 + m * 128 + lane_off;
    uint32_t ph_s = 0, ph_o = 0, ph_j = 0;
    Ring checks = {0, 0};
    bool alive = true;
    for (;;) {
      if (alive) alive = next_item();
      if (!alive || it.n_rows == 0) break;
      const bool dual = it.dual();
      const int steps = it.steps();
      const int row = dual ? lr : threadIdx.x;             // of the item
      const bool row_ok = row < it.n_rows;
      const bool warp_on = __any_sync(0xffffffffu, row_ok);
      const int rr = it.r0 + min(row, it.n_rows - 1);
      const uint32_t rt = (uint32_t)rr / (uint32_t)p.G;
      const int tok = it.base_tok + (int)rt;
      const uint32_t at = (uint32_t)tok * p.Hq + it.kvh * p.G + (rr - rt * p.G);         // row of q and out
      int lo, hi;
      span_of<FORM>(p, it, tok, lo, hi);
      float m_run = -INFINITY, l_run = 0.f;
      const int my_steps = (steps - m + 1) / 2;
      if (my_steps > 0) {
        if (warp_on) {
          if (!(dual && m)) {
            // half a warp per row: whole lines on both sides
            uint4 x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              x[i] = reinterpret_cast<const uint4*>(p.q + (size_t)__shfl_sync(0xffffffffu, at, 2 * i + (lane >> 4)) * D)[lane & 15];
            uint8_t* dst = sQ + m * TILE + ((lane >> 3) & 1) * ATOM + (warp & 3) * 4096;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int r = 2 * i + (lane >> 4);
              *reinterpret_cast<uint4*>(dst + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = x[i];
            }
            fence_proxy_async_smem();
          }
          uint32_t z[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) z[i] = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_st_32x32(tO + c * 32, z);
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[m]);
      }
      for (int j = 0; j < my_steps; ++j) {
        const int t = dual ? 2 * j + m : j;                // tile of the item
        const int key0 = (it.t0 + t) * BKV;
        const bool edge = key0 < it.lo_max || key0 + BKV > it.hi_min;
        uint32_t in_tree[4];                               // keys of the tile that a tree's row sees (on their way while the scores are)
        if (FORM == TREE_ROWS && edge)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int x = min(32, max(0, lo - key0 - c * 32)), y = min(32, max(0, hi - key0 - c * 32));
            in_tree[c] = tree_bits(p.tree + (size_t)tok * p.tree_words, p.tree_words, key0 + c * 32, it.own_hi) & (uint32_t)((1ull << y) - 1) &
                         ~(uint32_t)((1ull << x) - 1);
          }
        if (!(alive = warp_wait(&s_full[m], ph_s) && !*abort_flag)) break;
        ph_s ^= 1;
        if (warp_on) {
          tc_fence_after();
          // The tile's scores in halves of 64, each a step of the online softmax.
          const float scale = CAP ? p.cap_out : p.scale_log2;
          const uint64_t sc2 = pack2(scale, scale);
          auto load = [&](int h, uint32_t (&sv)[2][32]) {
            tmem_ld_32x32(tS + h * 64, sv[0]);
            tmem_ld_32x32(tS + h * 64 + 32, sv[1]);
          };
          auto max_of = [&](const uint32_t (&sv)[2][32]) { // independent chains
            float mx[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(sv[0][i]);
#pragma unroll
            for (int i = 4; i < 60; i += 8)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                mx[x] = max3(mx[x], __uint_as_float(sv[(i + 2 * x) >> 5][(i + 2 * x) & 31]), __uint_as_float(sv[(i + 2 * x + 1) >> 5][(i + 2 * x + 1) & 31]));
            return max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], __uint_as_float(sv[1][28]), __uint_as_float(sv[1][29])),
                        max3(__uint_as_float(sv[1][29]), __uint_as_float(sv[1][30]), __uint_as_float(sv[1][31])));
          };
          // A cap on the arithmetic units, as two exponential units' steps per score would cost as much as both products: where
          // |k s| <= 1/2 for a half's scores, as almost always, tanh(k s) = s (c0 + c1 s^2 + c2 s^4 + c3 s^6), an interpolation at
          // Chebyshev points off by 6e-7 of itself at most, five steps a pair of scores that are taken between the exponentials.  Else
          // it is taken in place in tensor memory, to keep the code short, and the polynomial that follows is s.
          uint64_t cap_c[4];
          auto cap = [&](int h, uint32_t (&sv)[2][32], float top) {
            float mn[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mn[i] = __uint_as_float(sv[0][i]);
#pragma unroll
            for (int i = 4; i < 64; i += 2)
              mn[(i >> 1) & 3] = min3(mn[(i >> 1) & 3], __uint_as_float(sv[i >> 5][i & 31]), __uint_as_float(sv[i >> 5][(i & 31) + 1]));
            const float low = min3(min3(mn[0], mn[1], mn[2]), mn[3], mn[3]);
            cap_c[0] = pack2(p.cap_c.x, p.cap_c.x);
            cap_c[1] = pack2(p.cap_c.y, p.cap_c.y);
            cap_c[2] = pack2(p.cap_c.z, p.cap_c.z);
            cap_c[3] = pack2(p.cap_c.w, p.cap_c.w);
            if (__all_sync(0xffffffffu, top <= p.cap_small && low >= -p.cap_small)) return;        // (NaN: no)
            const bool below_1 = __all_sync(0xffffffffu, top * p.cap_in <= 1.f && low * p.cap_in >= -1.f);
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t v[16];
              tmem_ld_32x16(tS + h * 64 + c * 16, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float x = __uint_as_float(v[i]);
                v[i] = __float_as_uint(below_1 ? score_cap_small(x, p.cap_in) : score_cap(x, p.cap_in));
              }
              tmem_st_32x16(tS + h * 64 + c * 16, v);
            }
            tmem_st_wait();
            load(h, sv);
            tmem_ld_wait();
            cap_c[0] = pack2(1.f, 1.f);
            cap_c[1] = cap_c[2] = cap_c[3] = 0;
          };
          // What the weights of scores up to `top` are taken relative to: that score's own, so that its weight, which often outweighs the
          // others, is 1 and not rounded.  (Scores that are larger by less than 2^8 do not move the maximum: their weights are up to 2^8 and
          // rounded like the others.)
          auto level = [&](float top) { return scale * (CAP ? score_cap(top, p.cap_in) : top); };
          // The running maximum up to that of new scores, where it is far enough behind; false: the product that last added to O has not
          // finished in time.  The tile before's has, as it was issued before the scores that arrived; `half`: the first half's may be on its way.
          auto raise = [&](float m_tile, bool half) {
            // a score of NaN or +inf makes the whole row NaN, whatever the exponentials below give
            if (!(m_tile < INFINITY)) l_run = __int_as_float(0x7fffffff);
            const float m_new = fmaxf(m_run, m_tile);
            const bool grow = m_new > m_run + 8.f;         // (the first visible key: from -inf)
            const float m_next = grow ? m_new : m_run;
            if (__any_sync(0xffffffffu, grow && l_run != 0.f)) {
              if (half && !warp_wait(&pv_half[m], ph_s ^ 1)) return false;
              tc_fence_after();
              const float alpha = !grow ? 1.f : exp2f(m_run - m_next);
              l_run *= alpha;
#pragma unroll 1
              for (int c = 0; c < 8; ++c) {
                uint32_t v[16];
                tmem_ld_32x16(tO + c * 16, v);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                tmem_st_32x16(tO + c * 16, v);
              }
            }
            m_run = m_next;
            return true;
          };
          // The weights of half h, as packed pairs over the first half's scores.  seen: not 0 for the scores that count, if not all do.
          auto weigh = [&](int h, const uint32_t (&sv)[2][32], auto masked, const uint32_t (&seen)[2]) {
            const float m_use = m_run == -INFINITY ? 0.f : m_run;        // (nothing visible yet: every exponential is zero)
            const uint64_t nm2 = pack2(-m_use, -m_use);
            uint64_t sum2[4] = {0, 0, 0, 0};
            uint32_t w[32];
            float e[2][16];
#pragma unroll
            for (int c = 0; c < 5; ++c) {                  // 16 exponentials, then the sums and packing of the 16 before
              if (c < 4) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  float &x = e[c & 1][2 * i], &y = e[c & 1][2 * i + 1];
                  uint64_t s2 = pack2(__uint_as_float(sv[c >> 1][(c & 1) * 16 + 2 * i]), __uint_as_float(sv[c >> 1][(c & 1) * 16 + 2 * i + 1]));
                  if (CAP) {
                    const uint64_t u = mul2(s2, s2);
                    s2 = mul2(fma2(fma2(fma2(u, cap_c[3], cap_c[2]), u, cap_c[1]), u, cap_c[0]), s2);
                  }
                  unpack2(fma2(s2, sc2, nm2), x, y);
                  if (i >= 8 - (CAP ? 0 : EMULATED)) {
                    exp2_fma(x, y);
                  } else {
                    x = exp2f(x);
                    y = exp2f(y);
                  }
                  if (masked.value) {
                    if (!(seen[c >> 1] & (1u << ((c & 1) * 16 + 2 * i)))) x = 0.f;
                    if (!(seen[c >> 1] & (2u << ((c & 1) * 16 + 2 * i)))) y = 0.f;
                  }
                }
              }
              if (c > 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float x = e[(c - 1) & 1][2 * i], y = e[(c - 1) & 1][2 * i + 1];
                  sum2[i & 3] = add2(sum2[i & 3], pack2(x, y));
                  const __nv_bfloat162 z = __floats2bfloat162_rn(x, y);
                  w[(c - 1) * 8 + i] = *reinterpret_cast<const uint32_t*>(&z);
                }
              }
            }
            tmem_st_32x32(tS + h * 32, w);
            tmem_st_wait();
            float l0, l1;
            unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), l0, l1);
            l_run += l0 + l1;
          };
          if (!edge) {
            // The second half is loaded and its maximum found under the exponentials of the first, and the products with the first half's
            // values begin before the second is done.  Cycles a tile of one warp alone / two warps of a scheduler, without
            // the products: 1977 / 2853 in one piece, 1396 / 2314 in halves, 1197 / 2098 with a quarter of the exponentials
            // on the arithmetic units; with a cap and none there: 2448 / 4064 with the polynomial before the weights, 1711 / 2981 with
            // its steps between their exponentials.
            uint32_t sa[2][32], sb[2][32];
            load(0, sa);
            tmem_ld_wait();
            if (!CAP) load(1, sb);                         // (with a cap the registers hold its polynomial instead)
            const uint32_t all[2] = {};
            const float top_a = max_of(sa);
            if (CAP) cap(0, sa, top_a);
            if (!(alive = raise(level(top_a), false))) break;
            weigh(0, sa, Int<0>(), all);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[m]);
            if (CAP) load(1, sb);
            tmem_ld_wait();
            const float top_b = max_of(sb);
            if (CAP) cap(1, sb, top_b);
            if (!(alive = raise(level(top_b), true))) break;
            weigh(1, sb, Int<0>(), all);
          } else {
            // With masked keys the products wait for the check of the values, so that O must not be rescaled between the halves' weights:
            // both halves' maximum comes first (of the scores themselves: a cap keeps their order).  Halves that no row of the warp sees cost
            // nothing; a loop keeps the code short.
            uint32_t sv[2][32];
            auto sees = [&](int h, int& a, int& b) {       // keys [a, b) of the half's 64
              a = lo - key0 - h * 64;
              b = hi - key0 - h * 64;
              if (FORM == TREE_ROWS) return (bool)__any_sync(0xffffffffu, (h ? in_tree[2] | in_tree[3] : in_tree[0] | in_tree[1]) != 0);
              return (bool)__any_sync(0xffffffffu, max(a, 0) < min(b, 64));
            };
            uint32_t seen[2];
            auto bits = [&](int h, int a, int b) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int x = min(32, max(0, a - c * 32)), y = min(32, max(0, b - c * 32));
                seen[c] = FORM == TREE_ROWS ? h ? in_tree[2 + c] : in_tree[c] : (uint32_t)((1ull << y) - 1) & ~(uint32_t)((1ull << x) - 1);
              }
            };
            auto mask = [&](int h, int a, int b) {
              if (FORM != TREE_ROWS && __all_sync(0xffffffffu, a <= 0 && b >= 64)) return;
              bits(h, a, b);
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(seen[c] & (1u << i))) sv[c][i] = 0xff800000u;      // -inf
            };
            float m_edge = -INFINITY;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              int a, b;
              if (!sees(h, a, b)) continue;
              load(h, sv);
              tmem_ld_wait();
              mask(h, a, b);
              const float x = max_of(sv);
              m_edge = max3(m_edge, x, x);
            }
            const bool some = FORM == TREE_ROWS ? (in_tree[0] | in_tree[1] | in_tree[2] | in_tree[3]) != 0 : max(lo, key0) < min(hi, key0 + BKV);
            raise(some ? level(m_edge) : -INFINITY, false);
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              int a, b;
              if (sees(h, a, b)) {
                load(h, sv);
                tmem_ld_wait();
                if (CAP) {                                 // (the weights are masked: a polynomial of -inf is not -inf)
                  cap(h, sv, max_of(sv));
                  bits(h, a, b);
                } else {
                  mask(h, a, b);
                }
                weigh(h, sv, Int<CAP>(), seen);
              } else {
                uint32_t z[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) z[i] = 0;
                tmem_st_32x32(tS + h * 32, z);
                tmem_st_wait();
              }
            }
          }
          if (!alive) break;
          if (edge) {
            Ring v = checks;
            v.skip(t);
            if (!(alive = warp_wait(&v_ok[v.st], v.ph))) break;
            auto in_tree_word = [&](int part) { return part < 2 ? part ? in_tree[1] : in_tree[0] : part == 2 ? in_tree[2] : in_tree[3]; };
            uint4 none;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(none.x), "=r"(none.y), "=r"(none.z), "=r"(none.w) : "r"(smem_u32(s_bad + v.st * 4)) : "memory");
            for (int part = 0; part < 4 && (none.x | none.y | none.z | none.w); ++part)
              for (uint32_t bad = *(volatile uint32_t*)(s_bad + v.st * 4 + part); bad; bad &= bad - 1) {
                // a key with values that are not finite: its row in shared memory is zero, the rows that see it add it here
                const int kx = part * 32 + __ffs(bad) - 1, key = key0 + kx;
                uint32_t w;
                tmem_ld_32x1(tS + (kx >> 1), w);
                tmem_ld_wait();
                const float pv = __uint_as_float(kx & 1 ? w & 0xFFFF0000u : w << 16);
                if (key >= it.k_end) continue;
                const bool seen = FORM == TREE_ROWS ? in_tree_word(part) >> (kx & 31) & 1 : key >= lo && key < hi;       // (also where its weight is zero: 0 x NaN is NaN, as in the products)
                const size_t vrow = ((size_t)p.block_table[(size_t)it.trow * p.max_blocks + (key >> p.bs_log2)] * p.Hkv + it.kvh) * p.bs + (key & (p.bs - 1));
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                  uint32_t o[32];
                  tmem_ld_32x32(tO + c * 32, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (seen) o[i] = __float_as_uint(fmaf(pv, __bfloat162float(p.v_cache[vrow * D + c * 32 + i]), __uint_as_float(o[i])));
                  tmem_st_32x32(tO + c * 32, o);
                  tmem_st_wait();
                }
              }
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          if (edge || !warp_on) mbar_arrive(&p_half[m]);
          mbar_arrive(&p_full[m]);
        }
      }
      if (!alive) break;
      checks.skip(it.t1 - it.t0);
      const bool joined = dual && steps > 1;               // both streams have a part of every row
      const bool writer = warp_on && !(dual && m);
      const size_t row0 = (size_t)it.slot * p.T * p.Hq;    // of the partial sums
      const int rows_here = min(32, it.n_rows - (row - lane));             // of this warp
      uint8_t* own = sQ + m * TILE + (warp & 3) * 4096;    // this warp's 32 rows of the two slabs, which held its queries
      auto load_gate = [&]() {                             // half a warp per row, as the queries lay
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          const int r = 2 * i + (lane >> 4);
          copy16_async(own + ((lane >> 3) & 1) * ATOM + r * 128 + (((lane & 7) ^ (r & 7)) << 4),
                       p.gate + (size_t)__shfl_sync(0xffffffffu, at, r) * D + (lane & 15) * 8);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      const bool gated = p.gate && !p.part_o && writer;
      // ---- a joined item's results: each stream reads both streams' parts where they are - rows lie in the same lanes - and takes half of the
      // columns, through the half of the shared memory that is its own; maxima and sums pass through the scores' columns, which are free.  (One
      // stream alone, with the other's part handed to it through shared memory, took 9200 cycles for 35 rows instead of 5200: 7 nodes over
      // 350 keys 14.3 us instead of 11.9.)
      if (joined) {
        uint8_t* half = sQ + m * TILE + (warp & 3) * 4096;                 // this warp's 32 rows of 64 columns
        const bool with_gate = p.gate && !p.part_o && warp_on;
        uint4 g[8];                                        // (on their way; the other stream's products may still read the queries that lie in the half)
        if (with_gate) {
#pragma unroll
          for (int i = 0; i < 8; ++i)                      // a quarter warp per row
            g[i] = reinterpret_cast<const uint4*>(p.gate + (size_t)__shfl_sync(0xffffffffu, at, 4 * i + (lane >> 3)) * D + m * 64)[lane & 7];
        }
        if (!(alive = warp_wait(&o_full[m], ph_o))) break;
        ph_o ^= 1;
        tc_fence_after();
        if (warp_on) {
          tmem_st_32x2(tS, __float_as_uint(m_run), __float_as_uint(l_run));
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&j_full[m]);
        if (!(alive = warp_wait(&j_full[m ^ 1], ph_j))) break;
        tc_fence_after();
        if (warp_on) {
          uint32_t other_m, other_l;
          tmem_ld_32x2(tmem + (m ^ 1) * 128 + lane_off, other_m, other_l);
          tmem_ld_wait();
          const float m0 = m ? __uint_as_float(other_m) : m_run, m1 = m ? m_run : __uint_as_float(other_m);
          const float l0 = m ? __uint_as_float(other_l) : l_run, l1 = m ? l_run : __uint_as_float(other_l), mm = fmaxf(m0, m1);
          float w0 = m0 == -INFINITY ? 0.f : exp2f(m0 - mm), w1 = m1 == -INFINITY ? 0.f : exp2f(m1 - mm);
          const float l = (l0 == 0.f ? 0.f : l0 * w0) + (l1 == 0.f ? 0.f : l1 * w1);
          if (p.part_o) {
            if (row_ok && m == 0) *reinterpret_cast<float2*>(p.part_ml + (row0 + at) * 2) = make_float2(mm, l);
          } else {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            w0 *= inv;
            w1 *= inv;
          }
          if (with_gate) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = 4 * i + (lane >> 3);
              *reinterpret_cast<uint4*>(half + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = g[i];
            }
            __syncwarp();
          }
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {                    // 32 columns
            uint32_t v[32], x[32];
            tmem_ld_32x32(tmem + 256 + lane_off + m * 64 + c * 32, v);
            tmem_ld_32x32(tmem + 384 + lane_off + m * 64 + c * 32, x);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float o = __uint_as_float(v[i]) * w0;
              v[i] = __float_as_uint(fmaf(__uint_as_float(x[i]), w1, o));
            }
            if (p.part_o) {
              float4* room = reinterpret_cast<float4*>(half);              // four columns of a row at place (column / 4, row ^ column / 4)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                room[i * 32 + (lane ^ i)] =
                    make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 8; ++i) {                // a quarter warp per row
                const int r = 4 * i + (lane >> 3);
                const size_t prow = row0 + __shfl_sync(0xffffffffu, at, r);
                if (r < rows_here) reinterpret_cast<float4*>(p.part_o + prow * D + m * 64 + c * 32)[lane & 7] = room[(lane & 7) * 32 + (r ^ (lane & 7))];
              }
              __syncwarp();
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint4* place = reinterpret_cast<uint4*>(half + lane * 128 + (((c * 4 + i) ^ (lane & 7)) << 4));
                float o[8];
#pragma unroll
                for (int y = 0; y < 8; ++y) o[y] = __uint_as_float(v[8 * i + y]);
                if (with_gate) {
                  const uint4 here = *place;
                  const __nv_bfloat162* gh = reinterpret_cast<const __nv_bfloat162*>(&here);
#pragma unroll
                  for (int y = 0; y < 4; ++y) {
                    const float2 gf = __bfloat1622float2(gh[y]);
                    o[2 * y] = __fdividef(o[2 * y], 1.f + __expf(-gf.x));
                    o[2 * y + 1] = __fdividef(o[2 * y + 1], 1.f + __expf(-gf.y));
                  }
                }
                uint4 u4;
                __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&u4);
#pragma unroll
                for (int y = 0; y < 4; ++y) h2[y] = __floats2bfloat162_rn(o[2 * y], o[2 * y + 1]);
                *place = u4;
              }
            }
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&j_empty[m]);           // this stream has read the other's part
        if (warp_on && !p.part_o) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {                    // a quarter warp per row
            const int r = 4 * i + (lane >> 3);
            const uint4 u4 = *reinterpret_cast<const uint4*>(half + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
            const size_t to = __shfl_sync(0xffffffffu, at, r);
            if (r < rows_here) reinterpret_cast<uint4*>(p.out + to * D + m * 64)[lane & 7] = u4;
          }
          __syncwarp();
        }
        if (!(alive = warp_wait(&j_empty[m ^ 1], ph_j))) break;
        tc_fence_after();
        ph_j ^= 1;
        continue;
      }
      // (this stream's score products have all finished: the scores of its last tile have arrived)
      if (gated) load_gate();
      if (my_steps > 0) {
        if (!(alive = warp_wait(&o_full[m], ph_o))) break;
        ph_o ^= 1;
        tc_fence_after();
      }
      // ---- results of the item: O / l through the gate, or O with (m, l) for the join of several items.  A warp's rows go through
      // the shared memory that held its queries, so that whole lines are stored: as bf16 over the gate, or in fp32
      // 32 columns at a time, four columns of a row at place (column / 4, row ^ column / 4).
      if (!writer) continue;                               // (a stream without a part, or without rows: the others write)
      float w_own = 1.f;
      auto staged = [&](int stream, int slot, int c4, int r) -> float4* {
        return reinterpret_cast<float4*>(sQ + stream * TILE + slot * ATOM + (warp & 3) * 4096 + ((c4 * 32 + (r ^ c4)) << 4));
      };
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {                        // 32 columns
        uint32_t v[32];
        if (my_steps > 0) {
          tmem_ld_32x32(tO + c * 32, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        auto four = [&](int i) {
          return make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
        };
        if (c == 0) {
          if (p.part_o) {
            if (row_ok) *reinterpret_cast<float2*>(p.part_ml + (row0 + at) * 2) = make_float2(m_run, l_run);
          } else {
            w_own = l_run == 0.f ? 0.f : 1.f / l_run;
            if (gated) {
              asm volatile("cp.async.wait_all;" ::: "memory");
              __syncwarp();
            }
          }
        }
        if (!p.part_o)
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * w_own);
        if (p.part_o) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *staged(m, 0, i, lane) = four(i);
          __syncwarp();
          if (steps) {
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = *staged(m, 0, lane & 7, 4 * i + (lane >> 3));               // a quarter warp per row
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const size_t prow = row0 + __shfl_sync(0xffffffffu, at, 4 * i + (lane >> 3));
              if (4 * i + (lane >> 3) < rows_here) reinterpret_cast<float4*>(p.part_o + prow * D + c * 32)[lane & 7] = x[i];
            }
          }
        } else {
          auto put = [&](auto with_gate) {              // (one look at the gate, not four)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4* place = reinterpret_cast<uint4*>(own + (c >> 1) * ATOM + lane * 128 + ((((c & 1) * 4 + i) ^ (lane & 7)) << 4));
              float o[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) o[x] = __uint_as_float(v[8 * i + x]);
              if (with_gate.value) {
                const uint4 g = *place;
                const __nv_bfloat162* gh = reinterpret_cast<const __nv_bfloat162*>(&g);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const float2 gf = __bfloat1622float2(gh[x]);
                  o[2 * x] = __fdividef(o[2 * x], 1.f + __expf(-gf.x));
                  o[2 * x + 1] = __fdividef(o[2 * x + 1], 1.f + __expf(-gf.y));
                }
              }
              uint4 u4;
              __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&u4);
#pragma unroll
              for (int x = 0; x < 4; ++x) h2[x] = __floats2bfloat162_rn(o[2 * x], o[2 * x + 1]);
              *place = u4;
            }
          };
          if (p.gate) put(Int<1>());
          else put(Int<0>());
        }
        __syncwarp();
      }
      if (!p.part_o) {
#pragma unroll 4
        for (int i = 0; i < (rows_here + 1) / 2; ++i) {    // half a warp per row
          const int r = 2 * i + (lane >> 4);
          const uint4 u4 = *reinterpret_cast<const uint4*>(own + ((lane >> 3) & 1) * ATOM + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          const size_t to = __shfl_sync(0xffffffffu, at, r);
          if (r < rows_here) reinterpret_cast<uint4*>(p.out + to * D)[lane & 15] = u4;
        }
        __syncwarp();
      }
      tc_fence_before();
    }
    if (!alive) {
      if (lane == 0) atomicExch(p.status, ERR_WAIT_ACC);
      *abort_flag = 1;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins a prompt row's partial sums; one warp per row of one head, lane: four columns.
__global__ void __launch_bounds__(256)
spans_join_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const size_t at = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (size_t)p.T * p.Hq;
  if (at >= rows) return;
  pdl_wait();
  const int tok = (int)(at / p.Hq);
  // the first 32 slots' maxima and sums and the gate are on their way while the row's sequence is looked for
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < p.splits) ml = *reinterpret_cast<const float2*>(p.part_ml + (lane * rows + at) * 2);
  uint2 gate = make_uint2(0, 0);
  if (p.gate) gate = *reinterpret_cast<const uint2*>(p.gate + at * D + lane * 4);
  int mine = 0;                                            // rows of no sequence stay as they are
  for (int b = lane; b < p.batch; b += 32) mine |= p.q_start[b] >= 0 && tok >= p.q_start[b] && tok - p.q_start[b] < p.q_len[b];
  if (!__any_sync(0xffffffffu, mine)) return;
  float M = ml.x;
  for (int s = lane + 32; s < p.splits; s += 32) M = fmaxf(M, p.part_ml[(s * rows + at) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < p.splits; s0 += 32) {              // a slot's maximum and sum per lane, then its part, eight on their way at a time
    if (s0 > 0) ml = s0 + lane < p.splits ? *reinterpret_cast<const float2*>(p.part_ml + ((s0 + lane) * rows + at) * 2) : make_float2(-INFINITY, 0.f);
    const float w_all = ml.y == 0.f ? -1.f : exp2f(ml.x - M);              // (below 0: nothing seen, the item may not have written its sums)
    for (int s1 = 0; s1 < min(32, p.splits - s0); s1 += 8) {
      float4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = __shfl_sync(0xffffffffu, w_all, s1 + i);
        if (!(w < 0.f)) x[i] = *reinterpret_cast<const float4*>(p.part_o + ((s0 + s1 + i) * rows + at) * D + lane * 4);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = __shfl_sync(0xffffffffu, w_all, s1 + i), l = __shfl_sync(0xffffffffu, ml.y, s1 + i);
        if (w < 0.f) continue;
        L += w * l;
        o[0] += w * x[i].x; o[1] += w * x[i].y; o[2] += w * x[i].z; o[3] += w * x[i].w;
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] *= inv;
  if (p.gate) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&gate);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      o[2 * i] *= 1.f / (1.f + __expf(-f.x));
      o[2 * i + 1] *= 1.f / (1.f + __expf(-f.y));
    }
  }
  uint2 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
  h[0] = __floats2bfloat162_rn(o[0], o[1]);
  h[1] = __floats2bfloat162_rn(o[2], o[3]);
  *reinterpret_cast<uint2*>(p.out + at * D + lane * 4) = u;
}

template <Form FORM, bool CAP>
int launch_as(const CUtensorMap& tmK, const CUtensorMap& tmV, const Params& p, cudaStream_t stream) {
  static PerDeviceOnce once_;
  bool& configured = once_.slot();
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(spans_kernel<FORM, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  cudaError_t e = launch_pdl(spans_kernel<FORM, CAP>, dim3(p.n_items), dim3(NTHREADS), SMEM_BYTES, stream, tmK, tmV, p);
  if (e != cudaSuccess || FORM == SHARED_KEYS || !p.part_o) return (int)e;
  return (int)launch_pdl(spans_join_kernel, dim3((unsigned)(((size_t)p.T * p.Hq + 7) / 8)), dim3(256), 0, stream, p);
}

template <Form FORM>
int launch(Params& p, const SpansCall& a) {
  const int bs = a.block_size;
  const bool pow2 = bs >= 16 && bs <= 256 && !(bs & (bs - 1));
  if (!pow2 || a.n_q_heads % a.n_kv_heads || a.batch < 1 || a.T < 1 || a.max_blocks < 1 || a.num_blocks < 1 || !(a.scale > 0.f) || !(a.cap >= 0.f) ||
      (long long)a.max_blocks * bs > 0x7fffff00ll || ((long long)a.num_blocks + 1) * a.n_kv_heads * bs > 0x7fffff00ll ||
      ((FORM == SHARED_KEYS || a.splits > 1) && !a.workspace))
    return -ERR_BAD_ARG;
  p.q = reinterpret_cast<const __nv_bfloat16*>(a.q);
  p.gate = FORM == SHARED_KEYS ? nullptr : reinterpret_cast<const __nv_bfloat16*>(a.gate);
  p.out = reinterpret_cast<__nv_bfloat16*>(a.out);
  p.v_cache = reinterpret_cast<const __nv_bfloat16*>(a.v_cache);
  p.block_table = a.block_table;
  p.kv_len = a.kv_len;
  p.batch = a.batch; p.T = a.T; p.max_blocks = a.max_blocks; p.num_blocks = a.num_blocks; p.bs = bs;
  while ((1 << p.bs_log2) < bs) ++p.bs_log2;
  p.Hq = a.n_q_heads; p.Hkv = a.n_kv_heads; p.G = a.n_q_heads / a.n_kv_heads;
  p.splits = a.splits;
  const size_t rows = (size_t)a.T * a.n_q_heads;
  const bool parts = FORM == SHARED_KEYS || p.splits > 1;
  p.part_o = parts ? a.workspace : nullptr;
  p.part_ml = parts ? a.workspace + rows * p.splits * D : nullptr;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.cap_in = a.cap > 0.f ? a.scale / a.cap : 0.f;
  p.cap_out = a.cap * 1.4426950408889634f;
  if (p.cap_in > 1e-5f && p.cap_in < 1e5f) {
    const double k = p.cap_in, k3 = k * k * k;
    p.cap_small = (float)(0.5 / k);
    p.cap_c = make_float4((float)(0.999999463558197 * k), (float)(-0.3332628309726715 * k3), (float)(0.1318994015455246 * k3 * k * k),
                          (float)(-0.0443927384912968 * k3 * k3 * k));
  }
  p.status = a.status;
  CUtensorMap tmK, tmV;
  const uint64_t kv_rows = (uint64_t)a.num_blocks * a.n_kv_heads * bs;
  const uint32_t box = bs < BKV ? bs : BKV;
  if (!make_tmap_2d(&tmK, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.k_cache, kv_rows, D, D * 2, box, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&tmV, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.v_cache, kv_rows, D, D * 2, box, 64, CU_TENSOR_MAP_SWIZZLE_128B))
    return -ERR_BAD_ARG;
  return a.cap > 0.f ? launch_as<FORM, true>(tmK, tmV, p, a.stream) : launch_as<FORM, false>(tmK, tmV, p, a.stream);
}

}  // namespace spans
}  // namespace b200

using namespace b200;

// Prompt rows.  Sequence b: rows [q_start, q_start + q_len) and the first kv_len keys of table row b.  Row t sees the keys
// lo[t] <= j < min(hi[t], kv_len); without lo from 0, without hi up to its own position kv_len - q_len + i.  splits: items a
// row's keys are cut into.  Rows of no sequence are left as they are.
template <spans::Form FORM>
static int prompt_rows(const SpansCall& a) {
  if (a.bytes != (int)sizeof(a) || a.max_q_len < 1 || a.max_q_len > a.T || a.splits < 1 || a.n_kv_heads < 1 || a.n_q_heads < a.n_kv_heads)
    return -ERR_BAD_ARG;
  spans::Params p = {};
  p.q_start = a.q_start; p.q_len = a.q_len; p.lo = a.lo; p.hi = a.hi;
  const long long g = a.n_q_heads / a.n_kv_heads, each = (a.max_q_len * g + 2 * spans::BQ - 1) / (2 * spans::BQ);
  const long long places = each * a.batch, real = a.T * g / (2 * spans::BQ) + a.batch;       // a sequence ends in at most one that is not full
  p.by_sequence = places > 2 * real;
  const long long tiles = p.by_sequence ? real : places;
  if (each > 0x7fffff || tiles * a.n_kv_heads * a.splits > 0x7fffffffll) return -ERR_BAD_ARG;
  p.row_tiles = (int)each;
  p.n_items = (int)(tiles * a.n_kv_heads * a.splits);
  if (FORM == spans::TREE_ROWS) {
    p.tree = a.tree;
    p.tree_words = a.tree_words;
  }
  return spans::launch<FORM>(p, a);
}
extern "C" int b200_attn_spans(const SpansCall* call) { return prompt_rows<spans::SPANS>(*call); }

// Rows of drafted trees: the last q_len[b] of sequence b's kv_len[b] keys are its tree's nodes.  Row t sees the context before them from
// lo[t] on, and the nodes whose bits are set in its tree_words words of `tree`.  splits: items that the keys a row tile sees are
// cut into at most.
extern "C" int b200_attn_tree(const SpansCall* call) {
  if (call->bytes != (int)sizeof(SpansCall) || !call->tree || call->tree_words < 1 || call->hi) return -ERR_BAD_ARG;
  return prompt_rows<spans::TREE_ROWS>(*call);
}

// One row per sequence: partial sums over the keys that groups of sequences share, for b200_attn_own_rows.  The sequences
// group_start[g] <= b < group_start[g + 1] hold the same first shared_len[g] keys in the same pages (those of the group's first row
// of the table); sequence b sees kv_len[b] of them.  splits: items the keys are cut into.
extern "C" int b200_attn_shared(const SpansCall* call) {
  const SpansCall& a = *call;
  if (a.bytes != (int)sizeof(a) || a.n_groups < 1 || a.splits < 1 || a.n_kv_heads < 1 || a.n_q_heads < a.n_kv_heads || a.T != a.batch)
    return -ERR_BAD_ARG;
  spans::Params p = {};
  p.group_start = a.group_start; p.shared_len = a.shared_len; p.n_groups = a.n_groups;
  const long long rows = (long long)a.batch * (a.n_q_heads / a.n_kv_heads), tiles = rows / (2 * spans::BQ) + a.n_groups;
  if (tiles * a.splits * a.n_kv_heads > 0x7fffffffll) return -ERR_BAD_ARG;
  p.n_items = (int)(tiles * a.splits * a.n_kv_heads);
  return spans::launch<spans::SHARED_KEYS>(p, a);
}
