// Attention over the paged bf16 cache (head width 128) in which every query row sees a span of keys of its own, sm_100a.
//
//   s_ij = scale q_i . k_j, with a cap c > 0: s = c tanh(s / c); o_i = sum_j softmax_j(s_ij) v_j over lo_i <= j < hi_i
//
// in two forms over one kernel: prompt rows (b200_attn_spans: packed documents, prefixes, blocks of an image that see each
// other, windows, causal rows after a context) and one row per sequence where groups of sequences hold the same leading pages
// (b200_attn_shared: those keys are read and multiplied once for the whole group).  A row that sees nothing is zero; a masked
// key takes no part whatever its bits are.
//
// Work is a list of items that as many CTAs as there are SMs walk in turn: 256 rows (token, head of one kv head) - all query
// heads of a kv head are packed into the rows, so a tile is full however few tokens there are - times a range of key tiles of
// 128.  A row's result comes from one item, or from several whose partial sums the second kernel joins.
//
// Two streams of 128 rows keep the tensor core and the exponential units busy in turn.  An item of at most 128 rows gives both
// streams the same rows and every other key tile, and joins them at its end.  Warp roles:
//   warps 0-3, 4-7: softmax of stream 0 and 1 - one row per thread, online maximum / sum in the exp2 domain, P as bf16 back
//             into the tensor memory its scores came from, lazy rescale of the stream's O (when a maximum grows by 2^8);
//   warp 8  : TMA producer - key and value tiles gathered page by page through the block table into one ring, running ahead
//             into the next item;
//   warp 9  : tcgen05.mma issuer - step u: P V of step u, scores of step u + 2 (steps alternate between the streams);
//   warps 10, 11: value check of tiles with masked keys - rows that are not there (behind the last key) or not finite are
//             set to zero, because 0 x inf in a product would reach rows that do not see them; rows that do see a key
//             with values that are not finite add it themselves.
// Tensor memory: S0 | S1 | O0 | O1, 128 columns each.  All mbarrier waits are bounded and unwind through the common exit.
#include <cuda_bf16.h>
#include "per_device.h"
#include "../ptx/sm100.cuh"
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
  // one row per sequence
  const int* group_start;         // [n_groups + 1]
  const int* shared_len;          // [n_groups]
  int n_groups;
  float* part_o;                  // [slots, T, Hq, 128], null: every row has one item
  float* part_ml;                 // [slots, T, Hq, 2]
  int batch, T, max_blocks, bs, Hq, Hkv, G;
  int row_tiles;                  // row tiles per sequence (prompt rows), over all groups (shared keys)
  int splits, own_splits;         // key ranges per row tile; of a sequence's own keys
  int n_items;
  float scale_log2;               // scale * log2(e)
  float cap_in, cap_out;          // scale / cap, cap * log2(e)
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

__device__ __forceinline__ void tmem_ld_32x1(uint32_t taddr, uint32_t& v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
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

// One piece of work; the same in every thread of a warp.
struct Item {
  int n_rows;            // rows of the tile that are there (0: no such item)
  int r0;                // first of them among the packed rows of base_tok
  int base_tok;          // q row of packed row 0
  int kvh, trow, slot;   // kv head; row of the block table; slot of the partial sums
  int t0, t1;            // key tiles
  int lo_max, hi_min;    // keys in [lo_max, hi_min) are seen by every row
  int k_end;             // first key that no row sees
  int kv_end;            // keys of the sequence
  int own_lo, own_hi;    // span of rows that have no span of their own (one row per sequence)
  int delta;             // position of a token minus its q row (prompt rows)
  __device__ __forceinline__ bool dual() const { return n_rows <= BQ; }
  __device__ __forceinline__ int steps() const { return dual() ? t1 - t0 : 2 * (t1 - t0); }
};

template <bool SHARED>
__device__ __forceinline__ void span_of(const Params& p, const Item& it, int tok, int& lo, int& hi) {
  if (SHARED) {
    lo = it.own_lo;
    hi = min(it.own_hi, min(p.kv_len[tok], p.max_blocks * p.bs));
  } else {
    lo = p.lo ? max(0, p.lo[tok]) : 0;
    hi = min(p.hi ? p.hi[tok] : tok + it.delta + 1, it.kv_end);
  }
}

// Item `idx` of the list; false: there is nothing to do.  Called by whole warps.
template <bool SHARED>
__device__ __forceinline__ bool get_item(const Params& p, int idx, int lane, Item& it) {
  it.n_rows = 0;
  int split, splits;
  int rows_all;
  if (SHARED) {
    const int n_shared = p.row_tiles * p.Hkv * p.splits;
    if (idx < n_shared) {                                  // keys of a group
      split = idx % p.splits;
      splits = p.splits;
      it.kvh = idx / p.splits % p.Hkv;
      int tile = idx / (p.splits * p.Hkv), g = 0, b0 = 0, rows = 0;
      for (; g < p.n_groups; ++g) {
        b0 = max(0, min(p.batch, p.group_start[g]));
        rows = max(0, min(p.batch, p.group_start[g + 1]) - b0) * p.G;
        const int tiles = (rows + 2 * BQ - 1) / (2 * BQ);
        if (tile < tiles) break;
        tile -= tiles;
      }
      if (g == p.n_groups) return false;
      it.base_tok = it.trow = b0;
      it.r0 = tile * 2 * BQ;
      rows_all = rows;
      it.own_lo = 0;
      it.own_hi = p.shared_len[g];
      it.slot = split;
      if (it.own_hi <= 0) return false;                    // (the join does not look at its slots either)
    } else {                                               // a sequence's own keys
      idx -= n_shared;
      split = idx % p.own_splits;
      splits = p.own_splits;
      it.kvh = idx / p.own_splits % p.Hkv;
      const int b = idx / (p.own_splits * p.Hkv);
      it.base_tok = it.trow = b;
      it.r0 = 0;
      rows_all = p.G;
      it.own_lo = 0;
      for (int g = 0; g < p.n_groups; ++g)
        if (b >= p.group_start[g] && b < p.group_start[g + 1]) it.own_lo = max(0, p.shared_len[g]);
      it.own_hi = 0x7fffffff;
      it.slot = p.splits + split;
    }
    it.kv_end = p.max_blocks * p.bs;
    it.delta = 0;
  } else {
    split = idx % p.splits;
    splits = p.splits;
    int x = idx / p.splits;
    it.kvh = x % p.Hkv;
    x /= p.Hkv;
    const int b = x % p.batch, tile = p.row_tiles - 1 - x / p.batch;      // long contexts first
    const int q0 = p.q_start[b], n = p.q_len[b];
    const int len = q0 < 0 ? 0 : min(n, p.T - q0);
    rows_all = max(0, len) * p.G;
    it.r0 = tile * 2 * BQ;
    it.trow = b;
    it.base_tok = q0;
    it.kv_end = max(0, min(p.kv_len[b], p.max_blocks * p.bs));
    it.delta = p.kv_len[b] - n - q0;
    it.slot = split;
    it.own_lo = it.own_hi = 0;
  }
  it.n_rows = min(2 * BQ, rows_all - it.r0);
  if (it.n_rows <= 0) return false;
  const int tok0 = it.base_tok + it.r0 / p.G, tok1 = it.base_tok + (it.r0 + it.n_rows - 1) / p.G;
  int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = 0;
  for (int t = tok0 + lane; t <= tok1; t += 32) {
    int lo, hi;
    span_of<SHARED>(p, it, t, lo, hi);
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
  it.k_end = __reduce_max_sync(0xffffffffu, hi_max);
  it.t0 = it.t1 = 0;
  if (it.k_end > lo_min) {
    const int a = lo_min / BKV, n = (it.k_end + BKV - 1) / BKV - a, per = (n + splits - 1) / splits;
    it.t0 = a + min(n, split * per);
    it.t1 = a + min(n, (split + 1) * per);
  }
  return true;
}

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
};

template <bool SHARED, bool CAP>
__global__ void __launch_bounds__(NTHREADS, 1)
spans_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_base[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_base) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                       // [2 streams] tiles; scratch of the join of the streams
  uint8_t* sR = smem + 2 * TILE;                            // ring of key and value tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(sR + STAGES * TILE);
  uint64_t* r_full = bars;
  uint64_t* r_empty = bars + STAGES;
  uint64_t* v_ok = bars + 2 * STAGES;                       // values checked (tile by tile, not by place in the ring)
  uint64_t* q_full = bars + 3 * STAGES;                     // per stream: queries there, O zero
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = q_full + 4;
  uint64_t* o_full = q_full + 6;
  uint64_t* j_full = q_full + 8;                            // stream 1's part lies in the scratch
  uint64_t* j_empty = q_full + 9;                           // and has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 10);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(bars + 32); // [STAGES][4] keys with values that are not finite
  float* s_ml = reinterpret_cast<float*>(bars + 48);        // [2][128] maximum and sum of stream 1

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform: the issuer depends on it
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 1);
      mbar_init(&v_ok[i], 2);
    }
    for (int m = 0; m < 2; ++m) {
      mbar_init(&q_full[m], 4);
      mbar_init(&s_full[m], 1);
      mbar_init(&p_full[m], 4);
      mbar_init(&o_full[m], 1);
    }
    mbar_init(j_full, 4);
    mbar_init(j_empty, 4);
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
  pdl_launch_dependents();
  pdl_wait();

  Item it;
  // registers per thread at launch: 168 (3 x 168 = 2 x 216 + 72)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    Ring r = {0, 0}, c = {0, 0};                           // places of tiles in the ring; of value tiles among their checks
    bool ok = true;
    if (warp == 8) {
      const int rows = min(p.bs, BKV), per_tile = BKV / rows;              // pages (or parts of one) in a tile
      const uint32_t sub_bytes = rows * 128;                               // one 64-column half of one
      if (lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
      }
      r.ph = 1;
      for (int idx = blockIdx.x; ok && idx < p.n_items; idx += gridDim.x) {
        if (!get_item<SHARED>(p, idx, lane, it)) continue;
        const int* bt = p.block_table + (size_t)it.trow * p.max_blocks;
        const int last_page = (it.k_end - 1) / p.bs;
        auto page_row = [&](int tile) {                                    // cache row where this lane's part of a tile begins
          const int key = tile * BKV + lane * rows;
          const int page = min(key / p.bs, last_page);
          return tile < it.t1 && lane < per_tile ? (bt[page] * p.Hkv + it.kvh) * p.bs + key % p.bs : 0;
        };
        int row = page_row(it.t0);
        for (int t = it.t0; ok && t < it.t1; ++t) {
          const int n = min(per_tile, (it.k_end - t * BKV + rows - 1) / rows);
          const int next_row = page_row(t + 1);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok = __all_sync(0xffffffffu, mbar_wait(&r_empty[r.st], r.ph)) && !*abort_flag;
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(&r_full[r.st], n * 2 * sub_bytes);
            __syncwarp();
            if (lane < n) {
              uint8_t* dst = sR + r.st * TILE + lane * sub_bytes;
              tma_load_2d(dst, kv ? &tmV : &tmK, &r_full[r.st], 0, row);
              tma_load_2d(dst + ATOM, kv ? &tmV : &tmK, &r_full[r.st], 64, row);
            }
            r.next();
          }
          row = next_row;
        }
      }
      if (!ok && lane == 0) { atomicExch(p.status, ERR_WAIT_STAGE); *abort_flag = 1; }
    } else if (warp == 9) {
      // The whole warp walks the loop, so that addresses and descriptors stay warp-uniform, and one elected lane issues.
      const uint32_t on = elect_one();
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar, parity)) && !*abort_flag;
        return ok;
      };
      const uint64_t dq = umma_desc_sw128(sQ), dk = umma_desc_sw128(sR), dv = desc_mn_sw128(sR, ATOM, 1024);
      uint32_t ph_q[2] = {0, 0}, ph_p[2] = {0, 0};
      for (int idx = blockIdx.x; ok && idx < p.n_items; idx += gridDim.x) {
        if (!get_item<SHARED>(p, idx, lane, it)) continue;
        const int steps = it.steps();
        if (steps == 0) continue;
        const bool dual = it.dual();
        Ring k = r;                                        // keys of the tile whose scores come next
        auto issue_s = [&](int u) {
          const int m = u & 1;
          if (!wait(&r_full[k.st], k.ph)) return;
          tc_fence_after();
          const uint64_t a = dq + (dual ? 0 : m * (TILE >> 4)), b = dk + k.st * (TILE >> 4);
#pragma unroll
          for (int s = 0; s < 8; ++s)
            umma_bf16_ss_warp(on, tmem + m * 128, a + (s >> 2) * (ATOM >> 4) + 2 * (s & 3), b + (s >> 2) * (ATOM >> 4) + 2 * (s & 3), idesc_qk,
                              s ? 1u : 0u);
          if (dual || m) {
            umma_commit_warp(on, &r_empty[k.st]);
            k.skip(2);
          }
          umma_commit_warp(on, &s_full[m]);
        };
#pragma unroll
        for (int m = 0; m < 2; ++m)
          if (ok && m < steps && wait(&q_full[m], ph_q[m])) {
            ph_q[m] ^= 1;
            issue_s(m);
          }
        for (int u = 0; ok && u < steps; ++u) {
          const int m = u & 1;
          if (dual || m == 0) {
            if (u) r.next();
            r.next();                                      // r: values of this step's tile
          }
          if (!wait(&p_full[m], ph_p[m]) || !wait(&v_ok[c.st], c.ph)) break;
          ph_p[m] ^= 1;
          tc_fence_after();
          const uint64_t b = dv + r.st * (TILE >> 4);
#pragma unroll
          for (int s = 0; s < 8; ++s) umma_bf16_ts_warp(on, tmem + 256 + m * 128, tmem + m * 128 + s * 8, b + s * 128, idesc_pv, 1u);
          if (dual || m) {
            umma_commit_warp(on, &r_empty[r.st]);
            c.next();
          }
          if (u + 2 < steps) issue_s(u + 2);
          else umma_commit_warp(on, &o_full[m]);
        }
        r.next();
      }
      if (!ok && lane == 0) { atomicExch(p.status, ERR_WAIT_TMA); *abort_flag = 1; }
    } else {
      const int w = warp - 10;                             // keys 64 w .. 64 w + 63 of a tile, lane: two of them
      for (int idx = blockIdx.x; ok && idx < p.n_items; idx += gridDim.x) {
        if (!get_item<SHARED>(p, idx, lane, it)) continue;
        for (int t = it.t0; ok && t < it.t1; ++t) {
          r.next();
          ok = __all_sync(0xffffffffu, mbar_wait(&r_full[r.st], r.ph)) && !*abort_flag;
          if (!ok) break;
          const int key0 = t * BKV;
          if (key0 < it.lo_max || key0 + BKV > it.hi_min) {
            bool wrote = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int key = w * 64 + i * 32 + lane;
              uint8_t* row = sR + r.st * TILE + key * 128;
              const bool there = key0 + key < it.k_end;
              uint32_t acc = 0;
              if (there) {
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                  const uint4 x = *reinterpret_cast<const uint4*>(row + (d >> 3) * ATOM + (((d & 7) ^ (key & 7)) << 4));
                  // bit 15 / 31 where an exponent is all ones
                  acc |= ((x.x & 0x7F807F80u) + 0x00800080u) | ((x.y & 0x7F807F80u) + 0x00800080u) | ((x.z & 0x7F807F80u) + 0x00800080u) |
                         ((x.w & 0x7F807F80u) + 0x00800080u);
                }
              }
              const bool bad = (acc & 0x80008000u) != 0;
              const uint32_t mask = __ballot_sync(0xffffffffu, bad);
              if (lane == 0) s_bad[c.st * 4 + w * 2 + i] = mask;
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int m = warp >> 2;                               // stream
    const int lr = threadIdx.x & 127;                      // row of the stream == TMEM lane
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + m * 128 + lane_off, tO = tmem + 256 + m * 128 + lane_off;
    uint32_t ph_s = 0, ph_o = 0, ph_j = 0;
    Ring c = {0, 0};
    bool alive = true;
    for (int idx = blockIdx.x; alive && idx < p.n_items; idx += gridDim.x) {
      if (!get_item<SHARED>(p, idx, lane, it)) continue;
      const bool dual = it.dual();
      const int steps = it.steps();
      const int row = dual ? lr : threadIdx.x;             // of the item
      const bool row_ok = row < it.n_rows;
      const bool warp_on = __any_sync(0xffffffffu, row_ok);
      const int rr = it.r0 + min(row, it.n_rows - 1);
      const int tok = it.base_tok + rr / p.G, head = it.kvh * p.G + rr % p.G;
      const size_t at = (size_t)tok * p.Hq + head;         // row of q and out
      int lo, hi;
      span_of<SHARED>(p, it, tok, lo, hi);
      float m_run = -INFINITY, l_run = 0.f;
      const int my_steps = (steps - m + 1) / 2;
      if (my_steps > 0) {
        if (warp_on) {
          if (!(dual && m)) {
            uint8_t* dst = sQ + m * TILE + lr * 128;
            const uint4* src = reinterpret_cast<const uint4*>(p.q + at * D);
            uint4 x[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) x[c] = src[c];
#pragma unroll
            for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(dst + (c >> 3) * ATOM + (((c & 7) ^ (lr & 7)) << 4)) = x[c];
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
        bool ok = mbar_wait(&s_full[m], ph_s);
        ok = __all_sync(0xffffffffu, ok) && !*abort_flag;
        if (!ok) { alive = false; break; }
        ph_s ^= 1;
        if (warp_on) {
          tc_fence_after();
          uint32_t sv[4][32];                              // the row's 128 scores
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32(tS + c * 32, sv[c]);
          tmem_ld_wait();
          const int key0 = (it.t0 + t) * BKV;
          const bool edge = key0 < it.lo_max || key0 + BKV > it.hi_min;
          const float scale = CAP ? 1.f : p.scale_log2;
          if (CAP) {
            const float k = p.cap_in, c = p.cap_out;
#pragma unroll
            for (int i = 0; i < 128; ++i) {
              const float z = __uint_as_float(sv[i >> 5][i & 31]) * k;
              const float e = exp2f(z * 2.885390081777927f);
              sv[i >> 5][i & 31] = __float_as_uint(c - 2.f * c * __fdividef(1.f, 1.f + e));
            }
          }
          if (edge) {
            const int a = lo - key0, b = hi - key0;
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (i < a || i >= b) sv[i >> 5][i & 31] = 0xff800000u;      // -inf
          }
          float mx[8];                                     // independent chains
#pragma unroll
          for (int i = 0; i < 8; ++i) mx[i] = __uint_as_float(sv[0][i]);
#pragma unroll
          for (int i = 8; i < 128; ++i) mx[i & 7] = fmaxf(mx[i & 7], __uint_as_float(sv[i >> 5][i & 31]));
          const float m_tile = scale * fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
          const float m_new = fmaxf(m_run, m_tile);
          const bool grow = m_new > m_run + 8.f;           // (the first visible key: from -inf)
          const float m_next = grow ? m_new : m_run;
          if (__any_sync(0xffffffffu, grow && l_run != 0.f)) {
            // the product that last added to O has finished: it was issued before the scores that arrived
            const float alpha = grow ? exp2f(m_run - m_next) : 1.f;
            l_run *= alpha;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t v[32];
              tmem_ld_32x32(tO + c * 32, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
              tmem_st_32x32(tO + c * 32, v);
            }
          }
          m_run = m_next;
          const float m_use = m_run == -INFINITY ? 0.f : m_run;          // (nothing visible yet: every exponential is zero)
          const uint64_t sc2 = pack2(scale, scale), nm2 = pack2(-m_use, -m_use);
          uint64_t sum2[2] = {0, 0};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int kx = half * 64 + 2 * i;
              float e0, e1;
              unpack2(fma2(pack2(__uint_as_float(sv[kx >> 5][kx & 31]), __uint_as_float(sv[kx >> 5][(kx & 31) + 1])), sc2, nm2), e0, e1);
              e0 = exp2f(e0);
              e1 = exp2f(e1);
              sum2[i & 1] = add2(sum2[i & 1], pack2(e0, e1));
              __nv_bfloat162 x = __floats2bfloat162_rn(e0, e1);
              w[i] = *reinterpret_cast<uint32_t*>(&x);
            }
            // 64 keys = 32 columns of packed pairs over this tile's own scores, which are all in registers by now
            tmem_st_32x32(tS + half * 32, w);
          }
          tmem_st_wait();
          float l0, l1;
          unpack2(add2(sum2[0], sum2[1]), l0, l1);
          l_run += l0 + l1;
          if (edge) {
            Ring v = c;
            v.skip(t);
            bool ok2 = __all_sync(0xffffffffu, mbar_wait(&v_ok[v.st], v.ph));
            if (!ok2) { alive = false; break; }
            for (int part = 0; part < 4; ++part)
              for (uint32_t bad = *(volatile uint32_t*)(s_bad + v.st * 4 + part); bad; bad &= bad - 1) {
                // a key with values that are not finite: its row in shared memory is zero, the rows that see it add it here
                const int kx = part * 32 + __ffs(bad) - 1, key = key0 + kx;
                uint32_t w;
                tmem_ld_32x1(tS + (kx >> 1), w);
                tmem_ld_wait();
                const float pv = __uint_as_float(kx & 1 ? w & 0xFFFF0000u : w << 16);
                const bool seen = key >= lo && key < hi && pv != 0.f;
                const size_t vrow = ((size_t)p.block_table[(size_t)it.trow * p.max_blocks + key / p.bs] * p.Hkv + it.kvh) * p.bs + key % p.bs;
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
        if (lane == 0) mbar_arrive(&p_full[m]);
      }
      if (!alive) break;
      c.skip(it.t1 - it.t0);
      if (my_steps > 0) {
        const bool ok = mbar_wait(&o_full[m], ph_o);
        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        ph_o ^= 1;
        tc_fence_after();
      }
      // ---- results of the item: O / l, or O with (m, l) for the join of several items
      const bool joined = dual && steps > 1;               // both streams have a part of every row
      float w_own = 1.f, w_other = 0.f;
      float4* s_o = reinterpret_cast<float4*>(sQ);         // [32][128 rows]
      if (joined) {
        if (m == 1) {
          // (every score product of the item, which read the scratch as queries, was issued before the product this stream waited for)
          if (warp_on) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t u[32];
              tmem_ld_32x32(tO + c * 32, u);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i)
                s_o[(c * 8 + i) * 128 + lr] = make_float4(__uint_as_float(u[4 * i]), __uint_as_float(u[4 * i + 1]), __uint_as_float(u[4 * i + 2]), __uint_as_float(u[4 * i + 3]));
            }
          }
          s_ml[lr] = m_run;
          s_ml[128 + lr] = l_run;
          __syncwarp();
          if (lane == 0) mbar_arrive(j_full);
        } else {
          const bool ok = mbar_wait(j_full, ph_j);
          if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        }
        if (m == 0) {
          const float m1 = s_ml[lr], l1 = s_ml[128 + lr];
          const float mm = fmaxf(m_run, m1);
          w_own = m_run == -INFINITY ? 0.f : exp2f(m_run - mm);
          w_other = m1 == -INFINITY ? 0.f : exp2f(m1 - mm);
          l_run = (l_run == 0.f ? 0.f : l_run * w_own) + (l1 == 0.f ? 0.f : l1 * w_other);
          m_run = mm;
        }
      }
      if (warp_on && !(dual && m)) {
        if (p.part_o) {
          const size_t prow = (size_t)it.slot * p.T * p.Hq + at;
          if (row_ok) *reinterpret_cast<float2*>(p.part_ml + prow * 2) = make_float2(m_run, l_run);
          if (steps) {
            float4* dst = reinterpret_cast<float4*>(p.part_o + prow * D);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t u[32];
              tmem_ld_32x32(tO + c * 32, u);
              tmem_ld_wait();
              if (row_ok) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  float4 o = make_float4(__uint_as_float(u[4 * i]), __uint_as_float(u[4 * i + 1]), __uint_as_float(u[4 * i + 2]), __uint_as_float(u[4 * i + 3]));
                  if (joined) {
                    const float4 x = s_o[(c * 8 + i) * 128 + lr];
                    o.x = o.x * w_own + x.x * w_other;
                    o.y = o.y * w_own + x.y * w_other;
                    o.z = o.z * w_own + x.z * w_other;
                    o.w = o.w * w_own + x.w * w_other;
                  }
                  dst[c * 8 + i] = o;
                }
              }
            }
          }
        } else {
          const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
          w_own *= inv;
          w_other *= inv;
          __nv_bfloat16* dst = p.out + at * D;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t u[32];
            if (steps) {
              tmem_ld_32x32(tO + c * 32, u);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) u[i] = 0;
            }
            if (row_ok) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                float o[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) o[x] = __uint_as_float(u[i + x]) * w_own;
                if (joined) {
#pragma unroll
                  for (int x = 0; x < 2; ++x) {
                    const float4 y = s_o[(c * 8 + i / 4 + x) * 128 + lr];
                    o[4 * x] += y.x * w_other;
                    o[4 * x + 1] += y.y * w_other;
                    o[4 * x + 2] += y.z * w_other;
                    o[4 * x + 3] += y.w * w_other;
                  }
                }
                if (p.gate) {
                  const uint4 gu = *reinterpret_cast<const uint4*>(p.gate + at * D + c * 32 + i);
                  const __nv_bfloat162* gh = reinterpret_cast<const __nv_bfloat162*>(&gu);
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    const float2 gf = __bfloat1622float2(gh[x]);
                    o[2 * x] *= 1.f / (1.f + __expf(-gf.x));
                    o[2 * x + 1] *= 1.f / (1.f + __expf(-gf.y));
                  }
                }
                uint4 u4;
                __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&u4);
#pragma unroll
                for (int x = 0; x < 4; ++x) h2[x] = __floats2bfloat162_rn(o[2 * x], o[2 * x + 1]);
                *reinterpret_cast<uint4*>(dst + c * 32 + i) = u4;
              }
            }
          }
        }
      }
      tc_fence_before();
      if (joined) {                                        // the scratch is read before the next rows overwrite it
        __syncwarp();
        if (m == 0 && lane == 0) mbar_arrive(j_empty);
        const bool ok = mbar_wait(j_empty, ph_j);
        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        ph_j ^= 1;
      }
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

// Joins a row's partial sums; one warp per row of one head, lane: four columns.
template <bool SHARED>
__global__ void __launch_bounds__(256)
spans_join_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const size_t at = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (size_t)p.T * p.Hq;
  if (at >= rows) return;
  pdl_wait();
  const int tok = (int)(at / p.Hq);
  int s0 = 0;
  if (SHARED) {                                            // slots of the shared keys are there for rows of a group that shares some
    s0 = p.splits;
    for (int g = lane; g < p.n_groups; g += 32)
      if (tok >= p.group_start[g] && tok < p.group_start[g + 1] && p.shared_len[g] > 0) s0 = 0;
    s0 = __reduce_min_sync(0xffffffffu, s0);
  } else {                                                 // rows of no sequence stay as they are
    int mine = 0;
    for (int b = lane; b < p.batch; b += 32) mine |= p.q_start[b] >= 0 && tok >= p.q_start[b] && tok - p.q_start[b] < p.q_len[b];
    if (!__any_sync(0xffffffffu, mine)) return;
  }
  const int s1 = p.splits + p.own_splits;
  float M = -INFINITY;
  for (int s = s0 + lane; s < s1; s += 32) M = fmaxf(M, p.part_ml[(s * rows + at) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = s0; s < s1; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * rows + at) * 2);
    if (ml.y == 0.f) continue;                             // (nothing seen: the item may not have written its sums)
    const float w = exp2f(ml.x - M);
    const float4 x = *reinterpret_cast<const float4*>(p.part_o + (s * rows + at) * D + lane * 4);
    L += w * ml.y;
    o[0] += w * x.x; o[1] += w * x.y; o[2] += w * x.z; o[3] += w * x.w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] *= inv;
  if (p.gate) {
    const uint2 u = *reinterpret_cast<const uint2*>(p.gate + at * D + lane * 4);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
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

template <bool SHARED, bool CAP>
int launch_as(const CUtensorMap& tmK, const CUtensorMap& tmV, const Params& p, cudaStream_t stream) {
  static PerDeviceOnce once_;
  bool& configured = once_.slot();
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(spans_kernel<SHARED, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  cudaError_t e = launch_pdl(spans_kernel<SHARED, CAP>, dim3(min(p.n_items, sm_count())), dim3(NTHREADS), SMEM_BYTES, stream, tmK, tmV, p);
  if (e != cudaSuccess || !p.part_o) return (int)e;
  return (int)launch_pdl(spans_join_kernel<SHARED>, dim3((unsigned)(((size_t)p.T * p.Hq + 7) / 8)), dim3(256), 0, stream, p);
}

template <bool SHARED>
int launch(Params& p, const void* q, const void* k_cache, const void* v_cache, void* out, const void* gate, const int* block_table,
           const int* kv_len, int batch, int T, int max_blocks, int num_blocks, int block_size, int n_q_heads, int n_kv_heads, float scale,
           float cap, float* workspace, int slots, int* status, cudaStream_t stream) {
  const bool pow2 = block_size >= 16 && block_size <= 256 && !(block_size & (block_size - 1));
  if (!pow2 || n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads || batch < 1 || T < 1 || max_blocks < 1 || num_blocks < 1 ||
      !(scale > 0.f) || !(cap >= 0.f) || (long long)max_blocks * block_size > 0x7fffff00ll ||
      (long long)num_blocks * n_kv_heads * block_size > 0x7fffff00ll || (slots > 1 && !workspace))
    return -ERR_BAD_ARG;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.gate = reinterpret_cast<const __nv_bfloat16*>(gate);
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.v_cache = reinterpret_cast<const __nv_bfloat16*>(v_cache);
  p.block_table = block_table;
  p.kv_len = kv_len;
  p.batch = batch; p.T = T; p.max_blocks = max_blocks; p.bs = block_size;
  p.Hq = n_q_heads; p.Hkv = n_kv_heads; p.G = n_q_heads / n_kv_heads;
  const size_t rows = (size_t)T * n_q_heads;
  p.part_o = slots > 1 ? workspace : nullptr;
  p.part_ml = slots > 1 ? workspace + rows * slots * D : nullptr;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.cap_in = cap > 0.f ? scale / cap : 0.f;
  p.cap_out = cap * 1.4426950408889634f;
  p.status = status;
  CUtensorMap tmK, tmV;
  const uint64_t kv_rows = (uint64_t)num_blocks * n_kv_heads * block_size;
  const uint32_t box = block_size < BKV ? block_size : BKV;
  if (!make_tmap_2d(&tmK, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, k_cache, kv_rows, D, D * 2, box, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&tmV, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, v_cache, kv_rows, D, D * 2, box, 64, CU_TENSOR_MAP_SWIZZLE_128B))
    return -ERR_BAD_ARG;
  return cap > 0.f ? launch_as<SHARED, true>(tmK, tmV, p, stream) : launch_as<SHARED, false>(tmK, tmV, p, stream);
}

}  // namespace spans
}  // namespace b200

using namespace b200;

// Prompt rows.  q / out / gate [T, Hq, 128] bf16; caches [num_blocks, Hkv, block_size, 128] bf16, block_size a power of two from
// 16 to 256; sequence b: rows [q_start, q_start + q_len) and the first kv_len keys of table row b.  Row t sees the keys
// lo[t] <= j < min(hi[t], kv_len); without lo from 0, without hi up to its own position kv_len - q_len + i.  splits: items a
// row's keys are cut into; from 2 on workspace: fp32 [splits T Hq 130].  Rows of no sequence are left as they are.
extern "C" int b200_attn_spans(const void* q, const void* k_cache, const void* v_cache, void* out, const void* gate,
                               const int* block_table, const int* q_start, const int* q_len, const int* kv_len, const int* lo,
                               const int* hi, int batch, int max_q_len, int T, int max_blocks, int num_blocks, int block_size,
                               int n_q_heads, int n_kv_heads, float scale, float cap, int splits, float* workspace, int* status,
                               cudaStream_t stream) {
  if (max_q_len < 1 || max_q_len > T || splits < 1 || n_kv_heads < 1 || n_q_heads < n_kv_heads) return -ERR_BAD_ARG;
  spans::Params p = {};
  p.q_start = q_start; p.q_len = q_len; p.lo = lo; p.hi = hi;
  const long long tiles = ((long long)max_q_len * (n_q_heads / n_kv_heads) + 2 * spans::BQ - 1) / (2 * spans::BQ);
  if (tiles * batch * n_kv_heads * splits > 0x7fffffffll) return -ERR_BAD_ARG;
  p.row_tiles = (int)tiles;
  p.splits = splits;
  p.own_splits = 0;
  p.n_items = (int)(tiles * batch * n_kv_heads * splits);
  return spans::launch<false>(p, q, k_cache, v_cache, out, gate, block_table, kv_len, batch, T, max_blocks, num_blocks, block_size, n_q_heads,
                              n_kv_heads, scale, cap, workspace, splits, status, stream);
}

// One row per sequence.  q / out / gate [B, Hq, 128]; sequence b: the first kv_len[b] keys of table row b.  The sequences
// group_start[g] <= b < group_start[g + 1] hold the same first shared_len[g] keys in the same pages; sequences of no group
// share nothing.  splits / own_splits: items the shared keys and a sequence's own keys are cut into; workspace: fp32
// [(splits + own_splits) B Hq 130].
extern "C" int b200_attn_shared(const void* q, const void* k_cache, const void* v_cache, void* out, const void* gate,
                                const int* block_table, const int* kv_len, const int* group_start, const int* shared_len, int n_groups,
                                int batch, int max_blocks, int num_blocks, int block_size, int n_q_heads, int n_kv_heads, float scale,
                                float cap, int splits, int own_splits, float* workspace, int* status, cudaStream_t stream) {
  if (n_groups < 0 || splits < 1 || own_splits < 1 || n_kv_heads < 1 || n_q_heads < n_kv_heads || batch < 1) return -ERR_BAD_ARG;
  spans::Params p = {};
  p.group_start = group_start; p.shared_len = shared_len; p.n_groups = n_groups;
  const long long rows = (long long)batch * (n_q_heads / n_kv_heads), tiles = n_groups ? rows / (2 * spans::BQ) + n_groups : 0;
  if ((tiles * splits + (long long)batch * own_splits) * n_kv_heads > 0x7fffffffll) return -ERR_BAD_ARG;
  p.row_tiles = (int)tiles;
  p.splits = splits;
  p.own_splits = own_splits;
  p.n_items = (int)((tiles * splits + (long long)batch * own_splits) * n_kv_heads);
  return spans::launch<true>(p, q, k_cache, v_cache, out, gate, block_table, kv_len, batch, batch, max_blocks, num_blocks, block_size,
                             n_q_heads, n_kv_heads, scale, cap, workspace, splits + own_splits, status, stream);
}
