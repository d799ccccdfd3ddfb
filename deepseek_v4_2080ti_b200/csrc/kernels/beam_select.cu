// Beam search's selection over the beams of a request and the vocabulary, sm_100a.
//
//   total[w, v] = score[w] + x[w, v] - log sum_u exp x[w, u];  the n largest of a request, ties to the lowest (w, v)
//
// Candidates of different beams lie closer together than 32 bits tell apart (of 16 out of 8 beams a pair in 10^5 is nearer than 10^-6), and a
// swapped pair swaps two beams, so the sums are kept to 2^-30 and totals compared in 64 bits.  Within a beam the order is that of the logits.
//
// select_parts_kernel reads the logits once: a block takes `tiles` tiles of 8192 logits of one row, 32 a thread in registers, adds
// their exponentials and keeps its n largest logits, in order, beside the sum.  select_join_kernel, a block per request, adds up the sums of
// every beam and joins the lists.
//
// The exponentials: x = (32 k + j) ln 2 / 32 + r with |r| <= 0.011, exp x = 2^k 2^(j/32) (1 + p), p = r + r^2 / 2 + r^3 / 6 in fp32
// (off by 2^-30.7 at most), 2^(j/32) from a table as a double, whose exponent takes k; T and T p are summed in 64 bits.  exp from the
// exponential unit is off by 2^-22, and its error is much the same in every term.
//
// The n largest: the k largest thread maxima of each of 8 warps, k = n / 8 rounded up, are 8 k >= n logits, so the least of them
// bounds the n-th largest from below; what reaches it - little more than n of 8192 - goes to shared memory, where each counts those before it.
// Where more than CAP reach it (ties) the n-th largest is found bit by bit instead.  Further tiles add what exceeds the list's last.
#include <cuda_bf16.h>
#include "../ptx/sm100.cuh"
#include "launch.h"
#include "ops.h"

namespace b200 {
namespace select {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int PER = 32;                    // logits of a thread
constexpr int TILE = THREADS * PER;
constexpr int MAX_N = 128, MAX_BEAMS = 128;
constexpr int CAP = 1024;                  // candidates that are ordered by counting
constexpr float LOWEST = -80.f;            // exp of this beside 1 is below 2^-115: smaller ones count as this

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
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Unsigned numbers in the order of the floats (-0 as 0), and back; all below ORDER_NONE or equal are -inf (or nothing).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t ORDER_NONE = 0x007fffffu;
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}

// A sum of exponentials, sum * exp(ref).
struct Sum {
  double ref, sum;
  __device__ __forceinline__ void add(const Sum& o) {
    if (!(o.sum != 0.0)) return;                           // nothing (a NaN is something)
    if (!(sum != 0.0)) {
      *this = o;
      return;
    }
    const double top = ref > o.ref ? ref : o.ref;
    // (equal references, as those of infinities: no difference to take)
    sum = sum * (ref == top ? 1.0 : exp(ref - top)) + o.sum * (o.ref == top ? 1.0 : exp(o.ref - top));
    ref = top;
  }
  __device__ __forceinline__ Sum shuffled(int o) const { return {__shfl_xor_sync(0xffffffffu, ref, o), __shfl_xor_sync(0xffffffffu, sum, o)}; }
};

// The 32 powers of two as the halves of doubles.
struct Table {
  const uint32_t *hi, *lo;
};

// exp of pairs of numbers of at most 2^15 in size, over 2^N: adds to a (T) and b (T p).
__device__ __forceinline__ void add_exp2(uint64_t x, const Table& t, int N, double& a, double& b) {
  constexpr float BIG = 12582912.f, L = 46.16624130844683f;                // 1.5 2^23: the sum's low bits are the rounded integer; 32 / ln 2
  constexpr float C_HI = 0.02166085f, C_LO = (float)(0.021660849392498290 - (double)0.02166085f);
  const uint64_t n2 = fma2(x, pack2(L, L), pack2(BIG, BIG));
  const uint64_t m2 = add2(n2, pack2(-BIG, -BIG));
  const uint64_t r = fma2(m2, pack2(-C_LO, -C_LO), fma2(m2, pack2(-C_HI, -C_HI), x));
  const uint64_t p = fma2(mul2(r, r), fma2(r, pack2(1.f / 6.f, 1.f / 6.f), pack2(0.5f, 0.5f)), r);
  float nf[2], pf[2];
  unpack2(n2, nf[0], nf[1]);
  unpack2(p, pf[0], pf[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = __float_as_int(nf[i]);                   // 0x4b400000 + integer
    const int j = n & 31;
    const double T = __hiloint2double((int)t.hi[j] + ((n >> 5) << 20) - N, (int)t.lo[j]);
    a += T;
    b = fma(T, (double)pf[i], b);
  }
}

// Sum of a thread's numbers, of which m, finite, is the largest.
__device__ __forceinline__ Sum sum_exp(const float (&v)[PER], float m, const Table& t) {
  constexpr int BIG_BITS = 0x4b400000;
  double a[2] = {0, 0}, b[2] = {0, 0};
  Sum s;
  // Numbers beyond 2^15 relative to the largest: differences of such are exact where they count.
  const bool far = !(fabsf(m) <= 32768.f);
  const float top = far ? 0.f : m, low = m + LOWEST;
  const int k = __float2int_rn(top * 1.44269504f);
  const int N = ((BIG_BITS >> 5) << 20) + (k << 20);       // (wraps: bits of the exponent)
  if (!far) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      add_exp2(pack2(fmaxf(v[i], low), fmaxf(v[i + 1], low)), t, N, a[0], b[0]);
      add_exp2(pack2(fmaxf(v[i + 2], low), fmaxf(v[i + 3], low)), t, N, a[1], b[1]);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < PER; ++i) {
      float x = v[0];
#pragma unroll
      for (int j = 1; j < PER; ++j)
        if (i == j) x = v[j];
      const float d = x - m;
      double none = 0, more = 0;
      add_exp2(pack2(fmaxf(d, LOWEST), LOWEST), t, N, none, more);
      if (d >= LOWEST) {
        a[0] += none;
        b[0] += more;
      }
    }
  }
  s.sum = (a[0] + a[1]) + (b[0] + b[1]);
  s.ref = (double)k * 0.6931471805599453 + (far ? (double)m : 0.0);
  return s;
}

struct Shared {
  unsigned long long list[2][CAP];
  uint32_t hi[32], lo[32];
  double ref[WARPS], sum[WARPS];
  uint32_t least[WARPS];
  int count, votes[2][WARPS];
};

// Block-wide sum of a count per thread; `turn` alternates between calls.
__device__ __forceinline__ int block_count(Shared& s, int mine, int& turn) {
  const int w = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) s.votes[turn][threadIdx.x >> 5] = w;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) all += s.votes[turn][i];
  turn ^= 1;
  return all;
}

template <bool BF16, bool VEC>
__device__ __forceinline__ int place(int j) {              // of a thread's j-th logit in its tile
  if (!VEC) return j * THREADS + threadIdx.x;
  return BF16 ? (j >> 3) * (8 * THREADS) + threadIdx.x * 8 + (j & 7) : (j >> 2) * (4 * THREADS) + threadIdx.x * 4 + (j & 3);
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(THREADS, 3)
select_parts_kernel(const __grid_constant__ SelectCall p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = blockIdx.x;
  const size_t row = blockIdx.y;
  if (tid < 32) {
    const double T = exp2(tid / 32.0);
    s.hi[tid] = (uint32_t)__double2hiint(T);
    s.lo[tid] = (uint32_t)__double2loint(T);
  }
  if (tid == 0) s.count = 0;
  pdl_wait();
  pdl_launch_dependents();
  // beams that are at their end, or that have come to nothing, offer nothing of their row
  const float score = p.scores[row];
  if (p.finished && p.finished[row] || !(fabsf(score) < INFINITY)) return;
  __syncthreads();
  const Table table = {s.hi, s.lo};
  const int n = p.n, k = (n + WARPS - 1) / WARPS;
  Sum sum = {-INFINITY, 0.0};
  int have = 0, cur = 0, turn = 0;
  const char* base = reinterpret_cast<const char*>(p.logits) + row * (size_t)p.row_stride * (BF16 ? 2 : 4);
#pragma unroll 1
  for (int t = 0; t < p.tiles; ++t) {
    const int first = (part * p.tiles + t) * TILE;
    if (first >= p.vocab) break;
    const int left = p.vocab - first;
    float v[PER];
    if (VEC && BF16) {
#pragma unroll
      for (int i = 0; i < PER / 8; ++i) {
        const int at = i * (8 * THREADS) + tid * 8;
        uint4 x = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
        if (at < left) x = __ldcs(reinterpret_cast<const uint4*>(base + (size_t)(first + at) * 2));
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          v[i * 8 + 2 * c] = __uint_as_float(w[c] << 16);
          v[i * 8 + 2 * c + 1] = __uint_as_float(w[c] & 0xffff0000u);
        }
      }
    } else if (VEC) {
#pragma unroll
      for (int i = 0; i < PER / 4; ++i) {
        const int at = i * (4 * THREADS) + tid * 4;
        float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at < left) x = __ldcs(reinterpret_cast<const float4*>(base + (size_t)(first + at) * 4));
        v[i * 4] = x.x;
        v[i * 4 + 1] = x.y;
        v[i * 4 + 2] = x.z;
        v[i * 4 + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int at = i * THREADS + tid;
        v[i] = -INFINITY;
        if (at < left) {
          if (BF16) v[i] = __uint_as_float((uint32_t)__ldcs(reinterpret_cast<const unsigned short*>(base + (size_t)(first + at) * 2)) << 16);
          else v[i] = __ldcs(reinterpret_cast<const float*>(base + (size_t)(first + at) * 4));
        }
      }
    }
    float m = v[0];
#pragma unroll
    for (int i = 1; i + 1 < PER; i += 2) m = max3_nan(m, v[i], v[i + 1]);
    m = max3_nan(m, v[PER - 1], v[PER - 1]);

    if (fabsf(m) < INFINITY) sum.add(sum_exp(v, m, table));
    else if (!(m == -INFINITY)) sum = {INFINITY, __longlong_as_double(0x7ff8000000000000ll)};       // NaN or +inf: the row counts for nothing

    // ---- what exceeds the list's last, or reaches a bound of the n-th largest
    uint32_t bound;
    const uint32_t mine = order_of(m);
    if (have == n) {
      bound = (uint32_t)(s.list[cur][n - 1] >> 32) + 1;    // (of equals the earlier ones stay)
    } else {
      uint32_t x = mine, top = 0;
      for (int i = 0; i < k; ++i) {
        top = __reduce_max_sync(0xffffffffu, x);
        if (x == top) x = 0;
      }
      if (lane == 0) s.least[warp] = top;
      __syncthreads();
      bound = s.least[0];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) bound = min(bound, s.least[w]);
      bound = max(bound, ORDER_NONE + 1);
    }
    unsigned long long* list = s.list[cur];
    auto key = [&](uint32_t order, int j) {
      return (unsigned long long)order << 32 | (uint32_t)~(first + place<BF16, VEC>(j));
    };
    if (mine >= bound) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const uint32_t o = order_of(v[j]);
        if (o >= bound) {
          const int at = have + atomicAdd(&s.count, 1);
          if (at < CAP) list[at] = key(o, j);
        }
      }
    }
    __syncthreads();
    int count = have + s.count;
    if (count == have) continue;
    __syncthreads();
    if (tid == 0) s.count = 0;
    if (count > CAP) {
      // the tile's n-th largest bit by bit, and the last of its equals that counts
      uint32_t cut = 0;
#pragma unroll 1
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = cut | 1u << bit;
        int more = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) more += order_of(v[j]) >= c;
        if (block_count(s, more, turn) >= n) cut = c;
      }
      cut = max(cut, ORDER_NONE + 1);
      int above = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) above += order_of(v[j]) > cut;
      const int wanted = n - block_count(s, above, turn);  // of those equal to the cut
      int end = 0;                                         // places below this hold fewer than `wanted` of them
#pragma unroll 1
      for (int bit = TILE / 2; bit > 0; bit >>= 1) {
        const int c = end + bit;
        int before = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) before += order_of(v[j]) == cut && place<BF16, VEC>(j) < c;
        if (block_count(s, before, turn) < wanted) end = c;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const uint32_t o = order_of(v[j]);
        if (o > cut || o == cut && place<BF16, VEC>(j) <= end) {
          const int at = have + atomicAdd(&s.count, 1);
          if (at < CAP) list[at] = key(o, j);
        }
      }
      __syncthreads();
      count = min(CAP, have + s.count);
      __syncthreads();
      if (tid == 0) s.count = 0;
    }
    for (int i = tid; i < count; i += THREADS) {
      const unsigned long long x = list[i];
      int before = 0;
      for (int j = 0; j < count; ++j) before += list[j] > x;
      if (before < n) s.list[cur ^ 1][before] = x;
    }
    have = min(n, count);
    cur ^= 1;
    __syncthreads();
  }
  unsigned long long* out = reinterpret_cast<unsigned long long*>(p.lists) + (row * p.parts + part) * n;
  for (int i = tid; i < n; i += THREADS) out[i] = i < have ? s.list[cur][i] : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum.add(sum.shuffled(o));
  if (lane == 0) {
    s.ref[warp] = sum.ref;
    s.sum[warp] = sum.sum;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) sum.add({s.ref[w], s.sum[w]});
    reinterpret_cast<double2*>(p.sums)[row * p.parts + part] = make_double2(sum.ref, sum.sum);
  }
}

struct Candidate {
  double total;
  long long flat;                          // beam * vocabulary + token
};
__device__ __forceinline__ bool before(double a, long long fa, double b, long long fb) { return a > b || a == b && fa < fb; }

__global__ void __launch_bounds__(THREADS)
select_join_kernel(const __grid_constant__ SelectCall p) {
  // total = (x - ref) + base, so that large logits lose nothing; base: score - log of the sum, -inf where the beam offers nothing of its row
  __shared__ double s_ref[MAX_BEAMS], s_base[MAX_BEAMS];
  __shared__ int s_active[MAX_BEAMS];        // beams that offer
  __shared__ Candidate s_cand[CAP];
  __shared__ unsigned long long s_least[WARPS];
  __shared__ int s_count, s_n_active;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x, W = p.beams, n = p.n;
  pdl_wait();
  pdl_launch_dependents();
  const size_t row0 = (size_t)b * W;
  for (int w = warp; w < W; w += WARPS) {                  // a warp per beam
    const float score = p.scores[row0 + w];
    double base = -INFINITY, ref = 0.0;
    if (!(p.finished && p.finished[row0 + w]) && fabsf(score) < INFINITY) {
      Sum sum = {-INFINITY, 0.0};
      for (int i = lane; i < p.parts; i += 32) {
        const double2 x = reinterpret_cast<const double2*>(p.sums)[(row0 + w) * p.parts + i];
        sum.add({x.x, x.y});
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum.add(sum.shuffled(o));
      base = (double)score - log(sum.sum);
      ref = sum.ref;
      if (!(base > -INFINITY && base < INFINITY && ref < INFINITY)) base = -INFINITY;        // a row with NaN or +inf, or of nothing but -inf
    }
    if (lane == 0) {
      s_base[w] = base;
      s_ref[w] = ref;
    }
  }
  if (tid == 0) s_count = 0;
  __syncthreads();
  if (warp == 0) {
    int active = 0;
    for (int w0 = 0; w0 < W; w0 += 32) {
      const bool on = w0 + lane < W && s_base[w0 + lane] > -INFINITY;
      const uint32_t go = __ballot_sync(0xffffffffu, on);
      if (on) s_active[active + __popc(go & ((1u << lane) - 1))] = w0 + lane;
      active += __popc(go);
    }
    if (lane == 0) s_n_active = active;
  }
  __syncthreads();
  const int lists = s_n_active * p.parts;
  auto entry = [&](int list, int i, long long& flat) {     // total of the i-th of a list, -inf where there is none
    const int w = s_active[list / p.parts];
    const unsigned long long x = reinterpret_cast<const unsigned long long*>(p.lists)[((row0 + w) * p.parts + list % p.parts) * n + i];
    flat = (long long)w * p.vocab + (uint32_t)~(uint32_t)x;
    return x == 0 ? -INFINITY : ((double)from_order((uint32_t)(x >> 32)) - s_ref[w]) + s_base[w];
  };
  // a bound from below of the n-th largest, as in the rows: from the first d entries of the lists
  const int k = (n + WARPS - 1) / WARPS;
  unsigned long long bound = 0;
  if (lists > 0) {
    const int d = min(n, (WARPS * k + lists - 1) / lists);
    double top = -INFINITY;
    for (int q = warp + WARPS * lane; q < lists * d; q += THREADS) {
      long long flat;
      const double x = entry(q / d, q % d, flat);
      top = x > top ? x : top;
    }
    unsigned long long x = order_of(top), most = 0;
    for (int i = 0; i < k; ++i) {
      const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32));
      const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u);
      most = (unsigned long long)hi << 32 | lo;
      if (x == most) x = 0;
    }
    if (lane == 0) s_least[warp] = most;
    __syncthreads();
    bound = s_least[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) bound = min(bound, s_least[w]);
  }
  auto finished = [&](int w) { return p.finished && p.finished[row0 + w] && fabsf(p.scores[row0 + w]) < INFINITY; };
  auto push = [&](double total, long long flat) {
    const int at = atomicAdd(&s_count, 1);
    if (at < CAP) s_cand[at] = {total, flat};
  };
  for (int list = warp; list < lists; list += WARPS)       // a warp per list, as far as it reaches the bound
    for (int i = 0; i < n; i += 32) {
      long long flat = 0;
      const double x = i + lane < n ? entry(list, i + lane, flat) : -INFINITY;
      const bool in = x > -INFINITY && order_of(x) >= bound;
      if (in) push(x, flat);
      if (!__all_sync(0xffffffffu, in)) break;
    }
  if (p.finished)
    for (int w = tid; w < W; w += THREADS)
      if (finished(w)) push((double)p.scores[row0 + w], (long long)w * p.vocab + p.pad_token);
  __syncthreads();
  int count = s_count;
  auto put = [&](int rank, double total, long long flat) {
    const size_t at = (size_t)b * n + rank;
    p.out_scores[at] = (float)total;
    p.out_parents[at] = (int)(flat / p.vocab);
    p.out_tokens[at] = (int)(flat % p.vocab);
  };
  if (count <= CAP) {
    for (int i = tid; i < count; i += THREADS) {
      const Candidate x = s_cand[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += before(s_cand[j].total, s_cand[j].flat, x.total, x.flat);
      if (rank < n) put(rank, x.total, x.flat);
    }
  } else {
    // more candidates tie with the n-th than are ordered by counting: the best head of all lists, n times
    __shared__ Candidate s_best[WARPS];
    __shared__ int s_from[WARPS];
    // a thread's lists are its own, so that their places need no other: list l belongs to thread l % THREADS; 16 bits for each in s_cand's room
    unsigned short* at = reinterpret_cast<unsigned short*>(s_cand);
    const int all = lists + W;                             // (behind the lists: beams at their end)
    __syncthreads();
    for (int l = tid; l < all; l += THREADS) at[l] = l < lists || finished(l - lists) ? 0 : 1;
    count = 0;
    for (int r = 0; r < n; ++r) {
      double best = -INFINITY;
      long long where = 0x7fffffffffffffffll;
      int from = -1;
      for (int l = tid; l < all; l += THREADS) {
        double x = -INFINITY;
        long long flat = 0;
        if (l < lists) {
          if (at[l] < n) x = entry(l, at[l], flat);
        } else if (at[l] == 0) {
          x = (double)p.scores[row0 + l - lists];
          flat = (long long)(l - lists) * p.vocab + p.pad_token;
        }
        if (x > -INFINITY && before(x, flat, best, where)) {
          best = x;
          where = flat;
          from = l;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double x = __shfl_xor_sync(0xffffffffu, best, o);
        const long long f = __shfl_xor_sync(0xffffffffu, where, o);
        const int l = __shfl_xor_sync(0xffffffffu, from, o);
        if (before(x, f, best, where)) {
          best = x;
          where = f;
          from = l;
        }
      }
      __syncthreads();
      if (lane == 0) {
        s_best[warp] = {best, where};
        s_from[warp] = from;
      }
      __syncthreads();
      for (int w = 0; w < WARPS; ++w)
        if (before(s_best[w].total, s_best[w].flat, best, where)) {
          best = s_best[w].total;
          where = s_best[w].flat;
          from = s_from[w];
        }
      if (from < 0) break;
      if (from % THREADS == tid) ++at[from];
      if (tid == 0) put(r, best, where);
      ++count;
    }
  }
  for (int r = count + tid; r < n; r += THREADS) {
    const size_t at = (size_t)b * n + r;
    p.out_scores[at] = -INFINITY;
    p.out_parents[at] = p.out_tokens[at] = -1;
  }
}

}  // namespace select
}  // namespace b200

using namespace b200;

extern "C" int b200_beam_select(const SelectCall* call) {
  const SelectCall& a = *call;
  if (a.bytes != (int)sizeof(a) || a.requests < 1 || a.beams < 1 || a.beams > select::MAX_BEAMS || a.vocab < 1 || a.n < 1 || a.n > select::MAX_N ||
      a.tiles < 1 || a.parts < 1 || (long long)a.parts * a.beams + a.beams > select::CAP * 8 || a.vocab > 0x7fff0000 ||
      ((long long)a.vocab + select::TILE - 1) / select::TILE > (long long)a.parts * a.tiles || (long long)a.requests * a.beams > 65535 ||
      a.pad_token < 0 || a.pad_token >= a.vocab)
    return -ERR_BAD_ARG;
  const dim3 grid(a.parts, a.requests * a.beams), block(select::THREADS);
  cudaError_t e = a.bf16 ? (a.vectors ? launch_pdl(select::select_parts_kernel<true, true>, grid, block, 0, a.stream, a)
                                      : launch_pdl(select::select_parts_kernel<true, false>, grid, block, 0, a.stream, a))
                         : (a.vectors ? launch_pdl(select::select_parts_kernel<false, true>, grid, block, 0, a.stream, a)
                                      : launch_pdl(select::select_parts_kernel<false, false>, grid, block, 0, a.stream, a));
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(select::select_join_kernel, dim3(a.requests), block, 0, a.stream, a);
}
