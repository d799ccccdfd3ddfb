// Attention prologue with rotary positions of several axes (time, height, width, ..): per-head RMSNorm of q and k ((1+gamma) or
// plain gamma), half-split RoPE over the first `rot` dims where pair i turns by positions[axis(i)] * inv_freq[i], split of the
// q||gate projection layout, and the write of K/V rows into the paged cache.
//
// Bound by memory: every row is read and written once.  A block takes a token, computes its cosines and sines once for all
// heads (angles in 64 bits: the product of a far position loses its fraction in 32) and then walks the rows of its heads,
// a warp per row, lane l dims [4l, 4l + 4), several rows of a warp on their way at a time.  8192 tokens of 40 + 2 x 8 heads with a
// gate (403 MB): 77.6 us, 5.2 TB/s.  2 / 8 rows on their way take 86.5 / 96.4; half a warp per row with loads of 16 bytes has half the
// instructions, but fewer warps: 79.5 at best.  1369 tokens of 28 + 2 x 4: 11.3 us, of which the two waves of blocks' latency is most.
//
// Reference behaviour: src/models/qwen4_exp/layers.py:288-326 (interleaved axes); norm, gate split and append as in rope_kv.cu.
#include <cuda_bf16.h>
#include <stdint.h>
#include "launch.h"
#include "ops.h"

namespace {

constexpr int D = 128;
constexpr int WARPS = 8;

struct AxesParams {
  const __nv_bfloat16* q_src; int ldq, q_off, q_head_stride, gate_in_q;      // head h at q_src[t * ldq + q_off + h * q_head_stride]
  const __nv_bfloat16* k_src; int ldk, k_off;
  const __nv_bfloat16* v_src; int ldv, v_off;
  const __nv_bfloat16* q_gamma; const __nv_bfloat16* k_gamma;                // optional [128]
  int unit_offset; float eps;
  const float* inv_freq; int rot; float mscale;
  const int* positions; int ld_pos;                                          // [axes, T]
  const int* slots;                                                          // [T]; slot = block * bs + offset, negative: not cached
  __nv_bfloat16* q_out; __nv_bfloat16* gate_out;                             // [T, Hq, 128]
  __nv_bfloat16* k_cache; __nv_bfloat16* v_cache; int bs; unsigned n_slots;  // [nb, Hkv, bs, 128]
  int T, Hq, Hkv;
  int block_rows;                                                            // of a block (grid.y blocks share a token's)
  unsigned char axis[D / 2];                                                 // of every pair
};

__device__ __forceinline__ void unpack4(const uint2 u, float (&f)[4]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const float2 a = __bfloat1622float2(h[0]), b = __bfloat1622float2(h[1]);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
__device__ __forceinline__ uint2 pack4(const float (&f)[4]) {
  uint2 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
  h[0] = __floats2bfloat162_rn(f[0], f[1]);
  h[1] = __floats2bfloat162_rn(f[2], f[3]);
  return u;
}

// U: rows of a warp that are on their way from memory together.
template <int U>
__global__ void __launch_bounds__(WARPS * 32)
qk_norm_rope_axes_append_kernel(const __grid_constant__ AxesParams p) {
  __shared__ __align__(16) float s_cos[D / 2], s_sin[D / 2];
  b200::pdl_grid_trigger();
  b200::pdl_grid_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x;
  const int half = p.rot >> 1, heads = p.Hq + 2 * p.Hkv;
  const int r0 = blockIdx.y * p.block_rows, r1 = min(heads, r0 + p.block_rows);
  auto source = [&](int hh) {
    return hh < p.Hq           ? p.q_src + (size_t)t * p.ldq + p.q_off + (size_t)hh * p.q_head_stride
           : hh < p.Hq + p.Hkv ? p.k_src + (size_t)t * p.ldk + p.k_off + (hh - p.Hq) * D
                               : p.v_src + (size_t)t * p.ldv + p.v_off + (hh - p.Hq - p.Hkv) * D;
  };
  uint2 u[U], gate[U];
  auto load = [&](int first) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int hh = first + j * WARPS;
      if (hh < r1) {
        const __nv_bfloat16* src = source(hh) + lane * 4;
        u[j] = *reinterpret_cast<const uint2*>(src);
        if (p.gate_in_q && hh < p.Hq) gate[j] = *reinterpret_cast<const uint2*>(src + D);
      }
    }
  };
  load(r0 + warp);                                          // on their way while the angles are computed
  const int slot = p.slots[t];
  uint2 gq = make_uint2(0, 0), gk = make_uint2(0, 0);
  if (p.q_gamma) gq = *reinterpret_cast<const uint2*>(p.q_gamma + lane * 4);
  if (p.k_gamma) gk = *reinterpret_cast<const uint2*>(p.k_gamma + lane * 4);
  if (threadIdx.x < half) {
    const int f = threadIdx.x;
    double a = (double)p.positions[(size_t)p.axis[f] * p.ld_pos + t] * (double)p.inv_freq[f];
    a -= 6.283185307179586 * rint(a * 0.15915494309189535);
    float sn, cs;
    __sincosf((float)a, &sn, &cs);
    s_cos[f] = cs * p.mscale;
    s_sin[f] = sn * p.mscale;
  }
  __syncthreads();
  // a lane's four dims: the first or the second of their pairs, or none of a pair
  const int d0 = lane * 4;
  const bool low = d0 < half, turns = d0 < p.rot;
  const int f = turns ? (low ? d0 : d0 - half) : 0, partner = low ? lane + (half >> 2) : lane - (half >> 2);
  const float4 cs = *reinterpret_cast<const float4*>(s_cos + f), sn = *reinterpret_cast<const float4*>(s_sin + f);
  const float c4[4] = {turns ? cs.x : 1.f, turns ? cs.y : 1.f, turns ? cs.z : 1.f, turns ? cs.w : 1.f};
  const float s4[4] = {turns ? (low ? -sn.x : sn.x) : 0.f, turns ? (low ? -sn.y : sn.y) : 0.f, turns ? (low ? -sn.z : sn.z) : 0.f,
                       turns ? (low ? -sn.w : sn.w) : 0.f};
  const size_t slot_row = (unsigned)slot < p.n_slots ? ((size_t)(slot / p.bs) * p.Hkv * p.bs + slot % p.bs) * D + d0 : ~(size_t)0;
  for (int first = r0 + warp; first < r1; first += WARPS * U) {
    if (first != r0 + warp) load(first);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int hh = first + j * WARPS;
      if (hh >= r1) break;
      const bool is_q = hh < p.Hq, is_k = !is_q && hh < p.Hq + p.Hkv;
      if (is_q || is_k) {
        float x[4];
        unpack4(u[j], x);
        if (is_q ? p.q_gamma != nullptr : p.k_gamma != nullptr) {
          float ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float inv = rsqrtf(ss * (1.f / D) + p.eps);
          float g[4];
          unpack4(is_q ? gq : gk, g);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = x[k] * inv * (p.unit_offset ? 1.f + g[k] : g[k]);
        }
        // partner of dim d < half: d + half, (half / 4) lanes on
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = __shfl_sync(0xffffffffu, x[k], partner);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = turns ? x[k] * c4[k] + y[k] * s4[k] : x[k];
        u[j] = pack4(x);
      }
      if (is_q) {
        const size_t at = ((size_t)t * p.Hq + hh) * D + d0;
        *reinterpret_cast<uint2*>(p.q_out + at) = u[j];
        if (p.gate_in_q) *reinterpret_cast<uint2*>(p.gate_out + at) = gate[j];
      } else if (slot_row != ~(size_t)0) {
        const int h = hh - p.Hq - (is_k ? 0 : p.Hkv);
        *reinterpret_cast<uint2*>((is_k ? p.k_cache : p.v_cache) + slot_row + (size_t)h * p.bs * D) = u[j];
      }
    }
  }
}

}  // namespace

// As b200_qk_norm_rope_append, with a row of positions for every axis and the axis of every rotary pair.  rot: a multiple of 8.
extern "C" int b200_qk_norm_rope_axes_append(const AxesAppendCall* call) {
  const AxesAppendCall& a = *call;
  if (a.bytes != (int)sizeof(a) || a.rot < 0 || a.rot > D || (a.rot & 7) || a.n_axes < 1 || a.T < 1 || a.Hq < 1 || a.Hkv < 1 || a.block_size < 1 ||
      a.num_blocks < 1 || (long long)a.num_blocks * a.block_size > 0x7fffffffll || (a.ldq & 3) || (a.q_off & 3) || (a.q_head_stride & 3) ||
      (a.ldk & 3) || (a.k_off & 3) || (a.ldv & 3) || (a.v_off & 3) || a.ld_pos < a.T || (a.gate_in_q && !a.gate_out) ||
      (a.rot && (!a.inv_freq || !a.positions)))
    return -6;
  AxesParams p = {};
  for (int i = 0; i < a.rot / 2; ++i) {
    if (a.axis[i] >= a.n_axes) return -6;
    p.axis[i] = a.axis[i];
  }
  p.q_src = reinterpret_cast<const __nv_bfloat16*>(a.q_src); p.ldq = a.ldq; p.q_off = a.q_off; p.q_head_stride = a.q_head_stride;
  p.gate_in_q = a.gate_in_q;
  p.k_src = reinterpret_cast<const __nv_bfloat16*>(a.k_src); p.ldk = a.ldk; p.k_off = a.k_off;
  p.v_src = reinterpret_cast<const __nv_bfloat16*>(a.v_src); p.ldv = a.ldv; p.v_off = a.v_off;
  p.q_gamma = reinterpret_cast<const __nv_bfloat16*>(a.q_gamma);
  p.k_gamma = reinterpret_cast<const __nv_bfloat16*>(a.k_gamma);
  p.unit_offset = a.unit_offset; p.eps = a.eps;
  p.inv_freq = a.inv_freq; p.rot = a.rot; p.mscale = a.mscale;
  p.positions = a.positions; p.ld_pos = a.ld_pos; p.slots = a.slots;
  p.q_out = reinterpret_cast<__nv_bfloat16*>(a.q_out);
  p.gate_out = reinterpret_cast<__nv_bfloat16*>(a.gate_out);
  p.k_cache = reinterpret_cast<__nv_bfloat16*>(a.k_cache);
  p.v_cache = reinterpret_cast<__nv_bfloat16*>(a.v_cache);
  p.bs = a.block_size; p.n_slots = (unsigned)a.num_blocks * a.block_size;
  p.T = a.T; p.Hq = a.Hq; p.Hkv = a.Hkv;
  const int heads = a.Hq + 2 * a.Hkv;
  // few tokens: a row per warp, so that the SMs share a token's heads (37 tokens of 64 rows: 2.2 us, with the other form 4.7; of 36 rows 2.7 / 3.5).
  // The two cross further out than the rule: 64 rows and 64 / 128 / 256 / 512 tokens 3.3 / 4.5 / 6.9 / 11.8 us, with the other form 4.8 / 6.4 /
  // 8.3 / 9.2; 36 rows and 128 / 256 / 512 tokens 3.3 / 4.8 / 7.8 and 4.4 / 6.0 / 6.6.
  const bool few = (long long)a.T * heads <= 148 * 2 * WARPS;
  p.block_rows = few ? WARPS : heads;
  const dim3 grid(a.T, (heads + p.block_rows - 1) / p.block_rows), block(WARPS * 32);
  return (int)(few ? b200::launch_pdl(qk_norm_rope_axes_append_kernel<1>, grid, block, 0, a.stream, p)
                   : b200::launch_pdl(qk_norm_rope_axes_append_kernel<4>, grid, block, 0, a.stream, p));
}
