// Attention prologue with rotary positions of several axes (time, height, width, ..): per-head RMSNorm of q and k ((1+gamma) or
// plain gamma), half-split RoPE over the first `rot` dims where pair i turns by positions[axis(i)] * inv_freq[i], split of the
// q||gate projection layout, and the write of K/V rows into the paged cache.
//
// Bound by memory: every row is read and written once.  A block takes a few tokens, computes their cosines and sines once for
// all heads (angles in 64 bits: the product of a far position loses its fraction in 32) and then walks the rows of
// their heads, a warp per row, lane l dims [4l, 4l + 4).
//
// Reference behaviour: src/models/qwen4_exp/layers.py:288-326 (interleaved axes); norm, gate split and append as in rope_kv.cu.
#include <cuda_bf16.h>
#include <stdint.h>
#include "launch.h"
#include "ops.h"

namespace {

constexpr int D = 128;
constexpr int WARPS = 8;
constexpr int MAX_TOKENS = 4;        // of a block

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
  int block_tokens, block_rows;                                              // of a block: tokens, rows of each (grid.y blocks share a token's)
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

__global__ void __launch_bounds__(WARPS * 32)
qk_norm_rope_axes_append_kernel(const __grid_constant__ AxesParams p) {
  __shared__ float s_cos[MAX_TOKENS][D / 2], s_sin[MAX_TOKENS][D / 2];
  b200::pdl_grid_trigger();
  b200::pdl_grid_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * p.block_tokens, n_tok = min(p.block_tokens, p.T - t0);
  const int half = p.rot >> 1, heads = p.Hq + 2 * p.Hkv;
  for (int i = threadIdx.x; i < n_tok * half; i += WARPS * 32) {
    const int t = i / half, f = i - t * half;
    double a = (double)p.positions[(size_t)p.axis[f] * p.ld_pos + t0 + t] * (double)p.inv_freq[f];
    a -= 6.283185307179586 * rint(a * 0.15915494309189535);
    float sn, cs;
    __sincosf((float)a, &sn, &cs);
    s_cos[t][f] = cs * p.mscale;
    s_sin[t][f] = sn * p.mscale;
  }
  __syncthreads();
  const int r0 = blockIdx.y * p.block_rows, rows = min(p.block_rows, heads - r0);
  for (int i = warp; i < n_tok * rows; i += WARPS) {
    const int tt = i / rows, hh = r0 + i - tt * rows, t = t0 + tt;
    const bool is_q = hh < p.Hq, is_k = !is_q && hh < p.Hq + p.Hkv;
    const int h = is_q ? hh : is_k ? hh - p.Hq : hh - p.Hq - p.Hkv;
    const __nv_bfloat16* src = is_q   ? p.q_src + (size_t)t * p.ldq + p.q_off + (size_t)h * p.q_head_stride
                               : is_k ? p.k_src + (size_t)t * p.ldk + p.k_off + h * D
                                      : p.v_src + (size_t)t * p.ldv + p.v_off + h * D;
    uint2 u = *reinterpret_cast<const uint2*>(src + lane * 4);
    if (is_q && p.gate_in_q)
      *reinterpret_cast<uint2*>(p.gate_out + ((size_t)t * p.Hq + h) * D + lane * 4) = *reinterpret_cast<const uint2*>(src + D + lane * 4);
    if (is_q || is_k) {
      float x[4];
      unpack4(u, x);
      const __nv_bfloat16* gamma = is_q ? p.q_gamma : p.k_gamma;
      if (gamma) {
        float ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss * (1.f / D) + p.eps);
        float g[4];
        unpack4(*reinterpret_cast<const uint2*>(gamma + lane * 4), g);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = x[k] * inv * (p.unit_offset ? 1.f + g[k] : g[k]);
      }
      // partner of dim d < half: d + half, (half / 4) lanes on
      const int d0 = lane * 4;
      const bool low = d0 < half;
      float y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = __shfl_sync(0xffffffffu, x[k], low ? lane + (half >> 2) : lane - (half >> 2));
      if (d0 < p.rot) {
        const int f = low ? d0 : d0 - half;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float cs = s_cos[tt][f + k], sn = s_sin[tt][f + k];
          x[k] = low ? x[k] * cs - y[k] * sn : x[k] * cs + y[k] * sn;
        }
      }
      u = pack4(x);
    }
    if (is_q) {
      *reinterpret_cast<uint2*>(p.q_out + ((size_t)t * p.Hq + h) * D + lane * 4) = u;
    } else {
      const int slot = p.slots[t];
      if ((unsigned)slot < p.n_slots)
        *reinterpret_cast<uint2*>((is_k ? p.k_cache : p.v_cache) + (((size_t)(slot / p.bs) * p.Hkv + h) * p.bs + slot % p.bs) * D + lane * 4) = u;
    }
  }
}

}  // namespace

// As b200_qk_norm_rope_append, with positions int32 [n_axes, T] (rows ld_pos apart) and `axes` (host, rot / 2 bytes): the axis of
// every rotary pair.  rot: a multiple of 8.
extern "C" int b200_qk_norm_rope_axes_append(
    const void* q_src, int ldq, int q_off, int q_head_stride, int gate_in_q, const void* k_src, int ldk, int k_off,
    const void* v_src, int ldv, int v_off, const void* q_gamma, const void* k_gamma, int unit_offset, float eps,
    const float* inv_freq, int rot, float mscale, const unsigned char* axes, int n_axes, const int* positions, int ld_pos,
    const int* slots, void* q_out, void* gate_out, void* k_cache, void* v_cache, int num_blocks, int block_size, int T, int Hq,
    int Hkv, cudaStream_t stream) {
  if (rot < 0 || rot > D || (rot & 7) || n_axes < 1 || T < 1 || Hq < 1 || Hkv < 1 || block_size < 1 || num_blocks < 1 ||
      (long long)num_blocks * block_size > 0x7fffffffll || (ldq & 3) || (q_off & 3) || (q_head_stride & 3) || (ldk & 3) || (k_off & 3) ||
      (ldv & 3) || (v_off & 3) || ld_pos < T || (gate_in_q && !gate_out) || (rot && (!axes || !inv_freq || !positions)))
    return -6;
  AxesParams p = {};
  for (int i = 0; i < rot / 2; ++i) {
    if (axes[i] >= n_axes) return -6;
    p.axis[i] = axes[i];
  }
  p.q_src = reinterpret_cast<const __nv_bfloat16*>(q_src); p.ldq = ldq; p.q_off = q_off; p.q_head_stride = q_head_stride;
  p.gate_in_q = gate_in_q;
  p.k_src = reinterpret_cast<const __nv_bfloat16*>(k_src); p.ldk = ldk; p.k_off = k_off;
  p.v_src = reinterpret_cast<const __nv_bfloat16*>(v_src); p.ldv = ldv; p.v_off = v_off;
  p.q_gamma = reinterpret_cast<const __nv_bfloat16*>(q_gamma);
  p.k_gamma = reinterpret_cast<const __nv_bfloat16*>(k_gamma);
  p.unit_offset = unit_offset; p.eps = eps;
  p.inv_freq = inv_freq; p.rot = rot; p.mscale = mscale;
  p.positions = positions; p.ld_pos = ld_pos; p.slots = slots;
  p.q_out = reinterpret_cast<__nv_bfloat16*>(q_out);
  p.gate_out = reinterpret_cast<__nv_bfloat16*>(gate_out);
  p.k_cache = reinterpret_cast<__nv_bfloat16*>(k_cache);
  p.v_cache = reinterpret_cast<__nv_bfloat16*>(v_cache);
  p.bs = block_size; p.n_slots = (unsigned)num_blocks * block_size;
  p.T = T; p.Hq = Hq; p.Hkv = Hkv;
  const int heads = Hq + 2 * Hkv;
  p.block_tokens = 1;
  p.block_rows = heads;
  const unsigned gy = (heads + p.block_rows - 1) / p.block_rows;
  return (int)b200::launch_pdl(qk_norm_rope_axes_append_kernel, dim3((T + p.block_tokens - 1) / p.block_tokens, gy), dim3(WARPS * 32), 0, stream, p);
}
