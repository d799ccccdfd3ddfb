// One query row per sequence over the keys that are the sequence's own, joined with what attn_spans.cu has summed over the keys it
// shares with others (paged bf16 cache, head width 128), sm_100a.
//
//   s_j = scale q . k_j (cap c: c tanh(s / c)), shared <= j < kv_len; o = (sum_j 2^(s_j - m) v_j + partial sums) / sum, out = o sigmoid(gate)
//
// Bound by memory: a key and its value are read once for the (up to 8 or 16) query heads of their kv head, straight into
// the fragments of the tensor core's warp-level products, 16 bytes a lane and whole lines a row:
//   scores^T [16 keys x 8 heads] = K [keys x dims] Q^T: the order of the 128 dims is free, so that a lane's 16 bytes of a row are
//     two of its fragments;
//   O^T [16 dims x 8 heads] = V^T [dims x keys] P^T: a lane holds the same 8 dims of its four keys and pairs them up;
//   P^T comes from the scores by an 8 x 8 transpose in registers.
// Heads as the narrow side of the products keep O of a kv head in 32 registers, so that a warp has 16 KB of keys and values on their way
// beside them.  64 sequences of 500 own keys, 8 kv heads (131 MB, 156 with the partial sums and what is read twice): 40 us behind the shared keys'
// kernel, 3.3 TB/s of the needed bytes and 3.8 of those moved (5.9 in the loop; the rest is the start of a block and the joins).  Weights are
// rounded to bf16 for the products (2^-8 of a weight at most), as they are for prompt rows; attn_gqa_decode.cu keeps them in 32 bits.
// Sums and statistics are 32 bits wide, and the sum adds the weights before they are rounded.  A warp takes 16 keys at a time (of one page: their
// page is looked up once), the warps of up to 8 blocks of a cluster share a sequence's keys, and the sums are joined in shared memory.
// The first products do not wait for the kernel before (it writes only the partial sums).
#include <cuda_bf16.h>
#include <stdint.h>
#include "launch.h"
#include "ops.h"
#include "score_cap.cuh"
#include "tma_host.h"

namespace {

constexpr int D = 128;
constexpr int LD = 132;              // floats of a row of O in shared memory: the fragments' stores then meet no bank twice

struct OwnParams {
  const __nv_bfloat16* q;            // [B, Hq, 128]
  const __nv_bfloat16* gate;         // optional
  __nv_bfloat16* out;
  const __nv_bfloat16* k_cache;      // [num_blocks, Hkv, bs, 128]
  const __nv_bfloat16* v_cache;
  const int* block_table;            // [B, max_blocks]
  const int* kv_len;                 // [B]
  const int* group_start;
  const int* shared_len;
  int n_groups;
  const float* part_o;               // [slots, B, Hq, 128]
  const float* part_ml;              // [slots, B, Hq, 2]
  int slots;
  int B, max_blocks, num_blocks, bs, bs_log2, Hq, Hkv, G, chunks, cluster;
  float scale_log2, cap_in, cap_out;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3, const uint32_t b0,
                                         const uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }
__device__ __forceinline__ uint4 lds128(const uint4* p) {          // (not to be kept in registers over a loop)
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"((uint32_t)__cvta_generic_to_shared(p)));
  return v;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_cluster4(const float* p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(r) : "memory");
  return v;
}

// NB: groups of 8 heads a block works on.  WARPS: 4, or 3 of which four blocks fit an SM instead of three.
template <int NB, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, NB == 2 ? 2 : 12 / WARPS)
own_rows_kernel(const __grid_constant__ OwnParams p) {
  constexpr int H = 8 * NB;
  __shared__ float s_m[WARPS][H], s_l[WARPS][H];
  __shared__ __align__(16) float s_o[WARPS][H][LD];
  __shared__ uint4 s_q[H][20];
  b200::pdl_grid_trigger();
  if (p.slots == 0) b200::pdl_grid_wait();               // (otherwise the kernel before has waited for what these products read)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % p.cluster;
  int x = blockIdx.x / p.cluster;
  const int h0 = (x % p.chunks) * H;                     // first head of the kv head's G
  x /= p.chunks;
  const int kvh = x % p.Hkv, b = x / p.Hkv;
  const int heads = min(H, p.G - h0);

  const int kv = max(0, min(p.kv_len[b], p.max_blocks * p.bs));
  int shared = 0, group_lo = -1, group_hi = -1;
  for (int i = lane; i < p.n_groups; i += 32) {
    const int lo = p.group_start[i], hi = p.group_start[i + 1], n = p.shared_len[i];     // (one trip to memory for the three)
    if (b >= lo && b < hi && n > 0) {
      shared = n;
      group_lo = lo;
      group_hi = hi;
    }
  }
  shared = __reduce_max_sync(0xffffffffu, shared);
  const int first = shared >> 4, n_blk = max(0, ((kv + 15) >> 4) - first);               // blocks of 16 keys
  const int* bt = p.block_table + (size_t)b * p.max_blocks;

  // The queries stay in shared memory (rows of 320 bytes: free of bank conflicts for the reads below): registers hold loads on their way.
  for (int i = threadIdx.x; i < H * 16; i += WARPS * 32) {
    const int h = i >> 4, d = i & 15;
    s_q[h][d] = h < heads ? reinterpret_cast<const uint4*>(p.q + ((size_t)b * p.Hq + kvh * p.G + h0 + h) * D)[d] : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  float o[NB][8][4];                                     // dims 8 g + i, 64 + 8 g + i of heads 2 c, 2 c + 1
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int y = 0; y < 4; ++y) o[i][d][y] = 0.f;
  float m[NB][2], l[NB][2];
#pragma unroll
  for (int i = 0; i < NB; ++i) m[i][0] = m[i][1] = -INFINITY, l[i][0] = l[i][1] = 0.f;

  // keys of block n: rows g and g + 8; values: keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9, dims 8 g and 64 + 8 g.  Rows that do not count are
  // zero: a product of zero with what they may hold would not be.  A page that is not there reads as zeros, as it does in attn_spans.cu.
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 k[2][4], v[4][2];
  auto row_of = [&](int blk) {
    const int key = (first + blk) << 4, page = bt[key >> p.bs_log2];
    return (unsigned)page < (unsigned)p.num_blocks ? ((size_t)page * p.Hkv + kvh) * p.bs + (key & (p.bs - 1)) : ~(size_t)0;
  };
  auto counts = [&](int blk, int i) {
    const int key = ((first + blk) << 4) + i;
    return blk < n_blk && key >= shared && key < kv;
  };
  auto there = [&](int blk, int i, size_t row) { return row != ~(size_t)0 && counts(blk, i); };
  auto load_k = [&](int blk, size_t row) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < 4; ++d)
        k[i][d] = there(blk, g + 8 * i, row) ? *reinterpret_cast<const uint4*>(p.k_cache + (row + g + 8 * i) * D + d * 32 + c * 8) : zero;
  };
  auto load_v = [&](int blk, size_t row) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 2 * c + (i & 1) + (i >> 1) * 8;
#pragma unroll
      for (int d = 0; d < 2; ++d)
        v[i][d] = there(blk, key, row) ? *reinterpret_cast<const uint4*>(p.v_cache + (row + key) * D + d * 64 + g * 8) : zero;
    }
  };
  const int step = WARPS * p.cluster;
  int blk = rank * WARPS + warp;
  size_t row = blk < n_blk ? row_of(blk) : ~(size_t)0;
  load_k(blk, row);
  load_v(blk, row);
  for (; blk < n_blk; blk += step) {
    const bool ok0 = counts(blk, g), ok1 = counts(blk, g + 8);
    float s[NB][4];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint4 q = lds128(&s_q[i * 8 + g][d * 4 + c]);                // head 8 i + g, dims 32 d + 8 c ..
        mma_bf16(s[i], k[0][d].x, k[1][d].x, k[0][d].y, k[1][d].y, q.x, q.y);
        mma_bf16(s[i], k[0][d].z, k[1][d].z, k[0][d].w, k[1][d].w, q.z, q.w);
      }
    }
    const int next = blk + step;
    const size_t next_row = next < n_blk ? row_of(next) : ~(size_t)0;
    load_k(next, next_row);
    uint32_t pt[NB][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (p.cap_out > 0.f) {
        const float big = fmaxf(fmaxf(fabsf(s[i][0]), fabsf(s[i][1])), fmaxf(fabsf(s[i][2]), fabsf(s[i][3])));
        if (__all_sync(0xffffffffu, big * p.cap_in <= 1.f)) {              // (NaN beside others: the polynomial keeps it)
#pragma unroll
          for (int y = 0; y < 4; ++y) s[i][y] = p.cap_out * b200::score_cap_small(s[i][y], p.cap_in);
        } else {
#pragma unroll
          for (int y = 0; y < 4; ++y) s[i][y] = p.cap_out * b200::score_cap(s[i][y], p.cap_in);
        }
      } else {
#pragma unroll
        for (int y = 0; y < 4; ++y) s[i][y] *= p.scale_log2;
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (!((y < 2) ? ok0 : ok1)) s[i][y] = -INFINITY;
      }
      float alpha[2];
      bool grown = false;
#pragma unroll
      for (int y = 0; y < 2; ++y) {                      // heads 2 c, 2 c + 1: their keys lie in the 8 lanes of the same c
        float mx = fmaxf(s[i][y], s[i][y + 2]);
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float mn = fmaxf(m[i][y], mx);
        const bool grow = mn > m[i][y] + 8.f;            // (the first key: from -inf)
        alpha[y] = grow ? exp2f(m[i][y] - mn) : 1.f;
        grown |= grow && m[i][y] != -INFINITY;
        if (grow) m[i][y] = mn;
        l[i][y] *= alpha[y];
        const float use = m[i][y] == -INFINITY ? 0.f : m[i][y];
        s[i][y] = exp2f(s[i][y] - use);
        s[i][y + 2] = exp2f(s[i][y + 2] - use);
        l[i][y] += s[i][y] + s[i][y + 2];
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          o[i][d][0] *= alpha[0];
          o[i][d][1] *= alpha[1];
          o[i][d][2] *= alpha[0];
          o[i][d][3] *= alpha[1];
        }
      }
      pt[i][0] = transpose8(pack(s[i][0], s[i][1]));
      pt[i][1] = transpose8(pack(s[i][2], s[i][3]));
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const uint32_t sel = d & 1 ? 0x7632 : 0x5410;      // the high or the low halves of two words
      const uint32_t a0 = __byte_perm(word(v[0][0], d >> 1), word(v[1][0], d >> 1), sel), a1 = __byte_perm(word(v[0][1], d >> 1), word(v[1][1], d >> 1), sel);
      const uint32_t a2 = __byte_perm(word(v[2][0], d >> 1), word(v[3][0], d >> 1), sel), a3 = __byte_perm(word(v[2][1], d >> 1), word(v[3][1], d >> 1), sel);
#pragma unroll
      for (int i = 0; i < NB; ++i) mma_bf16(o[i][d], a0, a1, a2, a3, pt[i][0], pt[i][1]);
    }
    row = next_row;
    load_v(next, row);
  }

  // ---- the warps' sums, then the blocks'
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[i][y] += __shfl_xor_sync(0xffffffffu, l[i][y], w);
      const int h = i * 8 + 2 * c + y;
      if (g == 0) {
        s_m[warp][h] = m[i][y];
        s_l[warp][h] = l[i][y];
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {                      // dim 64 y' + 8 g + d lies at 64 y' + 8 d + g
        s_o[warp][h][d * 8 + g] = o[i][d][y];
        s_o[warp][h][64 + d * 8 + g] = o[i][d][y + 2];
      }
    }
  __syncthreads();
  const bool many = p.cluster > 1;
  if (many) cluster_sync();
  if (p.slots) b200::pdl_grid_wait();
  const size_t rows = (size_t)p.B * p.Hq, at0 = (size_t)b * p.Hq + kvh * p.G + h0;
  // how often the keys of a head's row tile were cut: half as often for a rest of at most 128 (row, head) pairs
  group_lo = max(0, __reduce_max_sync(0xffffffffu, group_lo));
  group_hi = min(p.B, __reduce_max_sync(0xffffffffu, group_hi));
  auto slots_of = [&](int h) {
    const int r = (b - group_lo) * p.G + h0 + h, rest = (group_hi - group_lo) * p.G - r / 256 * 256;
    return shared <= 0 ? 0 : rest <= 128 ? (p.slots + 1) / 2 : p.slots;
  };
  const int slots = shared > 0 ? p.slots : 0, W = rank * WARPS + warp, n_warps = WARPS * p.cluster;
  // Every warp finds the maximum and the sum of every head over all warps and slots (a lane per warp and two slots); it then weighs
  // its own sums and every n_warps'th slot's, four dims a lane, into its rows of shared memory.
  float inv = 0.f;                                       // of head `lane`
#pragma unroll 1
  for (int i = 0; i < heads; i += 4) {                   // (four heads at a time: their slots' sums fit the registers)
    float2 ml[4][2];
    float mw[4], lw[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const bool ok = i + h < heads;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int sl = lane + 32 * y;
        ml[h][y] = ok && sl < slots_of(i + h) ? *reinterpret_cast<const float2*>(p.part_ml + (sl * rows + at0 + i + h) * 2) : make_float2(-INFINITY, 0.f);
      }
      mw[h] = -INFINITY;
      lw[h] = 0.f;
      if (lane < n_warps) {
        const int r = lane / WARPS, w = lane % WARPS;
        mw[h] = many ? ld_cluster(&s_m[w][i + h], r) : s_m[w][i + h];
        lw[h] = many ? ld_cluster(&s_l[w][i + h], r) : s_l[w][i + h];
      }
    }
    float f_own[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      float M = fmaxf(mw[h], fmaxf(ml[h][0].x, ml[h][1].x));
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
      // (-1 beside a sum of zero: nothing was seen, and what lies there may not have been written.  A weight that has become zero is
      // another thing: zero times a NaN that was seen is NaN.)
      const float fw = lw[h] == 0.f ? -1.f : exp2f(mw[h] - M);
      ml[h][0].x = ml[h][0].y == 0.f ? -1.f : exp2f(ml[h][0].x - M);
      ml[h][1].x = ml[h][1].y == 0.f ? -1.f : exp2f(ml[h][1].x - M);
      float L = fw * lw[h] + ml[h][0].x * ml[h][0].y + ml[h][1].x * ml[h][1].y;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
      if (lane == i + h) inv = L == 0.f ? 0.f : 1.f / L;
      f_own[h] = __shfl_sync(0xffffffffu, fw, W);
    }
    const int pos = (lane >> 4) * 64 + (lane & 1) * 32 + ((lane >> 1) & 7);            // of dims 4 lane ..: 64 y' + 8 d + g, d = 4 (lane & 1) ..
    float a[4][4];
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int y = 0; y < 4; ++y) a[h][y] = f_own[h] < 0.f ? 0.f : f_own[h] * s_o[warp][i + h][pos + 8 * y];
#pragma unroll 2
    for (int sl = W; sl < slots; sl += n_warps) {
      float4 x[4];
#pragma unroll
      for (int h = 0; h < 4; ++h)
        x[h] = i + h < heads ? *reinterpret_cast<const float4*>(p.part_o + (sl * rows + at0 + i + h) * D + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float f = __shfl_sync(0xffffffffu, sl < 32 ? ml[h][0].x : ml[h][1].x, sl & 31);
        if (f < 0.f) continue;                           // (nothing seen, or no such slot: what lies there is not looked at)
        a[h][0] += f * x[h].x; a[h][1] += f * x[h].y; a[h][2] += f * x[h].z; a[h][3] += f * x[h].w;
      }
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 4; ++h) *reinterpret_cast<float4*>(&s_o[warp][i + h][lane * 4]) = make_float4(a[h][0], a[h][1], a[h][2], a[h][3]);
  }
  __syncthreads();
  if (many) cluster_sync();
#pragma unroll 1
  for (int h = W; h < heads; h += n_warps) {             // a warp per head
    const size_t at = at0 + h;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    uint2 u = make_uint2(0, 0);
    if (p.gate) u = *reinterpret_cast<const uint2*>(p.gate + at * D + lane * 4);
    for (int r = 0; r < p.cluster; ++r)
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float4 x = many ? ld_cluster4(&s_o[w][h][lane * 4], r) : *reinterpret_cast<const float4*>(&s_o[w][h][lane * 4]);
        a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w;
      }
    const float f = __shfl_sync(0xffffffffu, inv, h);
#pragma unroll
    for (int y = 0; y < 4; ++y) a[y] *= f;
    if (p.gate) {
      const __nv_bfloat162* hp = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float2 z = __bfloat1622float2(hp[y]);
        a[2 * y] *= 1.f / (1.f + __expf(-z.x));
        a[2 * y + 1] *= 1.f / (1.f + __expf(-z.y));
      }
    }
    *reinterpret_cast<uint2*>(p.out + at * D + lane * 4) = make_uint2(pack(a[0], a[1]), pack(a[2], a[3]));
  }
  if (p.cluster > 1) cluster_sync();                     // the others may still read this block's sums
}

template <int NB, int WARPS>
cudaError_t launch(const OwnParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.B * p.Hkv * p.chunks * p.cluster));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, own_rows_kernel<NB, WARPS>, p);
}

}  // namespace

// Sequence b: the keys shared .. kv_len[b] - 1 of table row b, shared = shared_len[g] of the group with group_start[g] <= b <
// group_start[g + 1] (0 without one).  With groups: joined with the partial sums of b200_attn_shared, launched before this one with
// the same block.  cluster: thread blocks (1, 2, 4 or 8) that share a sequence's keys.
extern "C" int b200_attn_own_rows(const SpansCall* call) {
  const SpansCall& a = *call;
  const int bs = a.block_size;
  const bool pow2 = bs >= 16 && bs <= 256 && !(bs & (bs - 1));
  const int slots = a.n_groups > 0 ? a.splits : 0;
  if (a.bytes != (int)sizeof(a) || !pow2 || a.n_kv_heads < 1 || a.n_q_heads < 1 || a.n_q_heads % a.n_kv_heads || a.batch < 1 || a.max_blocks < 1 ||
      a.num_blocks < 1 || a.n_groups < 0 || !(a.scale > 0.f) || !(a.cap >= 0.f) || (long long)a.max_blocks * bs > 0x7fffff00ll || slots < 0 ||
      slots > 64 || (slots > 0 && !a.workspace) || (a.cluster != 1 && a.cluster != 2 && a.cluster != 4 && a.cluster != 8))
    return -6;
  OwnParams p = {};
  p.q = reinterpret_cast<const __nv_bfloat16*>(a.q);
  p.gate = reinterpret_cast<const __nv_bfloat16*>(a.gate);
  p.out = reinterpret_cast<__nv_bfloat16*>(a.out);
  p.k_cache = reinterpret_cast<const __nv_bfloat16*>(a.k_cache);
  p.v_cache = reinterpret_cast<const __nv_bfloat16*>(a.v_cache);
  p.block_table = a.block_table; p.kv_len = a.kv_len;
  p.group_start = a.group_start; p.shared_len = a.shared_len; p.n_groups = a.n_groups;
  p.part_o = a.workspace;
  p.part_ml = a.workspace ? a.workspace + (size_t)slots * a.batch * a.n_q_heads * D : nullptr;
  p.slots = slots;
  p.B = a.batch; p.max_blocks = a.max_blocks; p.num_blocks = a.num_blocks; p.bs = bs;
  while ((1 << p.bs_log2) < bs) ++p.bs_log2;
  p.Hq = a.n_q_heads; p.Hkv = a.n_kv_heads; p.G = a.n_q_heads / a.n_kv_heads;
  const int H = p.G <= 8 ? 8 : 16;
  p.chunks = (p.G + H - 1) / H;
  p.cluster = a.cluster;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.cap_in = a.cap > 0.f ? a.scale / a.cap : 0.f;
  p.cap_out = a.cap * 1.4426950408889634f;
  if ((long long)a.batch * a.n_kv_heads * p.chunks * a.cluster > 0x7fffffffll) return -6;
  if (H == 16) return (int)launch<2, 4>(p, a.stream);
  // A block of 3 warps takes a third longer, but four of them fit an SM: taken where that saves enough rounds of blocks, of which one in
  // twenty finds the kernel before still there.  Sequences of 500 own keys and 2048 shared ones, 8 kv heads, 4 / 3 warps: 32: 27.9 / 27.8 us,
  // 64: 67.6 / 48.3, 74: 69.2 / 73.9, 100: 76.1 / 78.2, 128: 89.4 / 81.9, 148: 91.4 / 95.9; 64 of 3000: 179.6 / 126.0.
  const long long blocks = (long long)a.batch * a.n_kv_heads * p.chunks * a.cluster, sms = b200::sm_count();
  auto rounds = [&](int per_sm) { return blocks * 20 / (per_sm * sms * 19) + 1; };
  const bool three = rounds(4) * 4 < rounds(3) * 3;
  return (int)(three ? launch<1, 3>(p, a.stream) : launch<1, 4>(p, a.stream));
}
