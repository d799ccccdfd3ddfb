// Beam search's selection over the beams of a request and the vocabulary, sm_100a.
//
//   total[w, v] = score[w] + x[w, v] - log sum_u exp x[w, u];  the n largest of a request, ties to the lowest w, the largest x, the lowest v
//
// select_parts_kernel reads the logits once: a block takes `tiles` tiles of 8192 logits of one row, 32 a thread in registers, adds
// their exponentials and keeps its n largest logits, in order, beside the sum.  select_join_kernel, a block per request, adds up the sums of
// every beam and joins the lists.
//
// Candidates of different beams may lie closer together than sums in 32 bits tell apart (of the 16 best of 8 beams a neighbouring pair in
// 10^5 is nearer than 10^-6), and a swapped pair swaps two beams.  So the sums carry a bound (off_of), and where two neighbours of different
// beams are nearer than their bounds the beams' rows are read again and summed to 2^-30 before their order is taken as certain; totals are
// compared in 64 bits.  Within a beam the order is that of the logits.
//
// The sums of the second pass: x = (32 k + j) ln 2 / 32 + r with |r| <= 0.011, exp x = 2^k 2^(j/32) (1 + p), p = r + r^2 / 2 + r^3 / 6 in fp32 (off by 2^-30.7), 2^(j/32) from a table as a double, whose
// exponent takes k; T and T p are summed in 64 bits.
//
// The n largest: every warp keeps a list of its own, in no order until it is full, and needs no other warp for it.  What is below a bound of
// the block's n-th largest does not get into it: the least of the warps' k-th largest, k = n / 8 rounded up, is one (8 k >= n logits reach
// it), first by lane maxima, then by what a warp found when it put its list in order.  So little more than n of 8192 get in, and a warp
// whose largest logit is below the bound is done with one look.  Where more get in than a list takes (ties) a warp finds its n-th largest bit
// by bit.
//
// What it takes: 64 requests of 8 beams (a fifth of them at their end) over 248320 tokens, 16 candidates, 86 us, 76 of them the first kernel
// at 5.4 TB/s: reading and maxima alone take 65 (at the rate of a copy 62), lists and what lets them in 10; the join is a chain of 10.
// With sums to 2^-30 in the first pass it was 150 us.  One request of 4 beams is 12 us: two dependent kernels' latency, 6 each.  Which entries of the
// parts' lists the join orders: see raise_bound and look_further.
#include <cuda_bf16.h>
#include <limits.h>
#include "../ptx/sm100.cuh"
#include "launch.h"
#include "ops.h"

namespace b200 {
namespace select {

constexpr int THREADS = 256, WARPS = THREADS / 32;
static_assert(THREADS == 256, "a thread's number in eight bits");
constexpr int PER = 32;                    // logits of a thread
constexpr int TILE = THREADS * PER;
constexpr int MAX_N = 128, MAX_BEAMS = 128;
constexpr int WARP_TILE = 32 * PER;
constexpr int AHEAD = 2;                   // tiles on their way to L2
constexpr int LIST = 256;                  // candidates of a warp: n and as many new ones
constexpr int CAP = 1024;                  // candidates that are ordered by counting
constexpr int FEW = 128;                   // candidates that are ordered with no look first at which may be among the best (64: 8.7 us, 9.5 with it; 256: 14.0, 10.9 with it)
constexpr float LOWEST = -80.f;            // exp of this beside 1 is below 2^-115: smaller ones count as this
constexpr float LOG2E = 1.44269504f;

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

// A sum of exponentials, sum * exp(k ln 2 + far); far is 0 for logits of at most 2^15 in size.  Those of the first pass count in powers of
// e^(1 / LOG2E), so that what LOG2E is off by counts for the distance from the largest logit and not for the logits themselves.
template <bool EXACT>
struct Sum {
  double sum;
  int k;
  float far;
  __device__ __forceinline__ double ref() const { return (double)k * (EXACT ? 0.6931471805599453 : 1.0 / (double)LOG2E) + (double)far; }
  __device__ __forceinline__ void add(const Sum& o) {
    if (!(o.sum != 0.0)) return;                           // nothing (a NaN is something)
    if (!(sum != 0.0)) {
      *this = o;
    } else if (far == o.far) {                             // powers of two, no rounding
      const int top = max(k, o.k);
      sum = sum * power(k - top) + o.sum * power(o.k - top);
      k = top;
    } else {
      const double a = ref(), b = o.ref();
      const Sum& top = a > b ? *this : o;
      const double t = a > b ? a : b;
      sum = sum * (a == t ? 1.0 : exp(a - t)) + o.sum * (b == t ? 1.0 : exp(b - t));
      k = top.k;
      far = top.far;
    }
  }
  static __device__ __forceinline__ double power(int e) { return __hiloint2double((1023 + max(e, -1022)) << 20, 0); }
};
// The sum of a warp's lanes, in every lane.
template <bool EXACT>
__device__ __forceinline__ void warp_sum(Sum<EXACT>& s) {
  if (!__any_sync(0xffffffffu, s.sum != 0.0 && s.far != 0.f)) {            // as almost always
    const int top = __reduce_max_sync(0xffffffffu, s.sum != 0.0 ? s.k : INT_MIN);
    if (s.sum != 0.0) s.sum *= s.power(s.k - top);
    s.k = top;
    s.far = 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, o);
  } else {
    for (int o = 16; o > 0; o >>= 1)
      s.add({__shfl_xor_sync(0xffffffffu, s.sum, o), __shfl_xor_sync(0xffffffffu, s.k, o), __shfl_xor_sync(0xffffffffu, s.far, o)});
  }
}
// The sum of a block's threads, in warp 0.
template <bool EXACT>
__device__ __forceinline__ void block_sum(Sum<EXACT>& s, Sum<EXACT>* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  warp_sum(s);
  if (lane == 0) sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    if (lane < WARPS) s = sums[lane];
    else s.sum = 0.0;
    warp_sum(s);
  }
}

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

// Numbers beyond 2^15 are taken relative to the largest: differences of such are exact where they count.
struct Scale {
  float far, low;                          // what is subtracted first; the least number that counts
  int k;                                   // the largest is about k ln 2 + far
  __device__ __forceinline__ explicit Scale(float m) {
    const bool is_far = !(fabsf(m) <= 32768.f);
    far = is_far ? m : 0.f;
    low = is_far ? LOWEST : m + LOWEST;
    k = is_far ? 0 : __float2int_rn(m * 1.44269504f);
  }
};

// Sum of a thread's numbers, of which m, finite, is the largest, to 2^-30.
__device__ __forceinline__ Sum<true> sum_exactly(const float (&v)[PER], float m, const Table& t) {
  constexpr int BIG_BITS = 0x4b400000;
  double a[2] = {0, 0}, b[2] = {0, 0};
  const Scale s(m);
  const int N = ((BIG_BITS >> 5) << 20) + (s.k << 20);     // (wraps: bits of the exponent)
#pragma unroll
  for (int i = 0; i < PER; i += 4) {
    add_exp2(pack2(fmaxf(v[i] - s.far, s.low), fmaxf(v[i + 1] - s.far, s.low)), t, N, a[0], b[0]);
    add_exp2(pack2(fmaxf(v[i + 2] - s.far, s.low), fmaxf(v[i + 3] - s.far, s.low)), t, N, a[1], b[1]);
  }
  return {(a[0] + a[1]) + (b[0] + b[1]), s.k, s.far};
}

// The same of one number.
__device__ __forceinline__ Sum<true> sum_of_one(float m, const Table& t) {
  double a = 0, b = 0;
  const Scale s(m);
  add_exp2(pack2(m - s.far, s.low), t, ((0x4b400000 >> 5) << 20) + (s.k << 20), a, b);     // (the other one, 2^-115 of it, is lost in the rounding)
  return {a + b, s.k, s.far};
}

// The same for the first pass, in two operations and an exponential a logit: 2^t with t = x log2 e - k.
__device__ __forceinline__ Sum<false> sum_quickly(const float (&v)[PER], float m) {
  const Scale s(m);
  const float far = s.far;
  const uint64_t far2 = pack2(-far, -far), k2 = pack2(-(float)s.k, -(float)s.k), log2e = pack2(LOG2E, LOG2E);
  uint64_t a[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < PER; i += 2) {
    uint64_t x = pack2(v[i], v[i + 1]);
    if (far != 0.f) x = add2(x, far2);
    float e[2];
    unpack2(fma2(x, log2e, k2), e[0], e[1]);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[0]));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[1]));
    a[i / 2 & 3] = add2(a[i / 2 & 3], pack2(e[0], e[1]));
  }
  double sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x, y;
    unpack2(a[i], x, y);
    sum += (double)x + (double)y;
  }
  return {sum, s.k, far};
}
// How far a logarithm of such a sum over v logits may be off.  t is off by 2^-24 of itself and by what LOG2E is (2^-26); weighted with the
// exponentials |t| is log2 v + 1 at most (their entropy).  The exponentials are off by 2^-22, four terms added in 32 bits by 3 2^-24.
__device__ __forceinline__ double off_of(int v) { return 5.1e-8 * (33 - __clz(v)) + 4.5e-7; }

struct Shared {
  unsigned long long list[WARPS][2][LIST]; // in turn
  Sum<false> sum[WARPS];
  uint32_t least[WARPS];
  unsigned long long joined[WARPS * MAX_N];
  int n_list[WARPS], count;
};

// Place of a lane's j-th logit in its warp's tile.
template <bool BF16, bool VEC>
__device__ __forceinline__ int place(int j) {
  const int lane = threadIdx.x & 31;
  if (!VEC) return j * 32 + lane;
  return BF16 ? (j >> 3) * 256 + lane * 8 + (j & 7) : (j >> 2) * 128 + lane * 4 + (j & 3);
}

template <bool BF16, bool VEC, bool FULL>
__device__ __forceinline__ void load_logits(const char* base, int left, float (&v)[PER]) {
  if (VEC && BF16) {
#pragma unroll
    for (int i = 0; i < PER / 8; ++i) {
      const int at = place<BF16, VEC>(i * 8);
      uint4 x = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
      if (FULL || at < left) x = __ldcs(reinterpret_cast<const uint4*>(base + (size_t)at * 2));
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
      const int at = place<BF16, VEC>(i * 4);
      float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (FULL || at < left) x = __ldcs(reinterpret_cast<const float4*>(base + (size_t)at * 4));
      v[i * 4] = x.x;
      v[i * 4 + 1] = x.y;
      v[i * 4 + 2] = x.z;
      v[i * 4 + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = place<BF16, VEC>(i);
      v[i] = -INFINITY;
      if (FULL || at < left) {
        if (BF16) v[i] = __uint_as_float((uint32_t)__ldcs(reinterpret_cast<const unsigned short*>(base + (size_t)at * 2)) << 16);
        else v[i] = __ldcs(reinterpret_cast<const float*>(base + (size_t)at * 4));
      }
    }
  }
}
// A lane's logits of the warp's tile that begins at `first`, of which `left` are there; -inf behind them.
template <bool BF16, bool VEC>
__device__ __forceinline__ void load_tile(const char* base, int first, int left, float (&v)[PER]) {
  const char* tile = base + (size_t)first * (BF16 ? 2 : 4);
  if (left >= WARP_TILE) load_logits<BF16, VEC, true>(tile, left, v);
  else load_logits<BF16, VEC, false>(tile, left, v);
}
__device__ __forceinline__ float largest(const float (&v)[PER]) {          // NaN if there is one
  float m = v[0];
#pragma unroll
  for (int i = 1; i + 1 < PER; i += 2) m = max3_nan(m, v[i], v[i + 1]);
  return max3_nan(m, v[PER - 1], v[PER - 1]);
}

// The warp's tile's n largest, when more than a list takes reach the bound: all above `cut`, and of its equals those at places up to `end`.
template <bool BF16, bool VEC>
__device__ __forceinline__ void cut_tile(const float (&v)[PER], int n, uint32_t& cut, int& end) {
  cut = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = cut | 1u << bit;
    int more = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) more += order_of(v[j]) >= c;
    if (__reduce_add_sync(0xffffffffu, more) >= n) cut = c;
  }
  cut = max(cut, ORDER_NONE + 1);
  int above = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) above += order_of(v[j]) > cut;
  const int wanted = n - __reduce_add_sync(0xffffffffu, above);
  end = 0;                                                 // places below this hold fewer than `wanted` of the cut's equals
#pragma unroll 1
  for (int bit = WARP_TILE / 2; bit > 0; bit >>= 1) {
    const int c = end + bit;
    int earlier = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) earlier += order_of(v[j]) == cut && place<BF16, VEC>(j) < c;
    if (__reduce_add_sync(0xffffffffu, earlier) < wanted) end = c;
  }
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(THREADS, 3)
select_parts_kernel(const __grid_constant__ SelectCall p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = blockIdx.x;
  const size_t row = blockIdx.y;
  if (tid == 0) s.count = 0;
  pdl_wait();
  pdl_launch_dependents();
  // beams that are at their end, or that have come to nothing, offer nothing of their row
  const float score = p.scores[row];
  if (p.finished && p.finished[row] || !(fabsf(score) < INFINITY)) return;
  const int n = p.n, k = (n + WARPS - 1) / WARPS;
  const char* base = reinterpret_cast<const char*>(p.logits) + row * (size_t)p.row_stride * (BF16 ? 2 : 4);
  Sum<false> sum = {0.0, 0, 0.f};
  unsigned long long* list = s.list[warp][0];
  unsigned long long* other = s.list[warp][1];
  int count = 0;                                           // of the list
  uint32_t own = ORDER_NONE + 1;                           // what a logit has to reach for this warp's list
  volatile uint32_t* least = s.least;
  // The list in order, n of it at most; the warp's share in the bound.
  auto put_in_order = [&]() {
    __syncwarp();
    for (int i = lane; i < count; i += 32) {
      const unsigned long long x = list[i];
      int before = 0;
      for (int j = 0; j < count; ++j) before += list[j] > x;
      if (before < n) other[before] = x;
    }
    __syncwarp();
    unsigned long long* t = list;
    list = other;
    other = t;
    count = min(count, n);
    if (count == n) own = max(own, (uint32_t)(list[n - 1] >> 32) + 1);     // (of equals the earlier ones stay, and this warp's earlier ones come first)
    if (count >= k && lane == 0) least[warp] = (uint32_t)(list[k - 1] >> 32);
  };
#pragma unroll 1
  for (int t = 0; t < p.tiles; ++t) {
    const int first = (part * p.tiles + t) * TILE + warp * WARP_TILE, left = p.vocab - first;
    if (t > 0 && left <= 0) break;
    if (t + AHEAD < p.tiles && lane < WARP_TILE * (BF16 ? 2 : 4) / 128 && left > AHEAD * TILE + lane * (128 / (BF16 ? 2 : 4)))
      asm volatile("prefetch.global.L2 [%0];" ::"l"(base + ((size_t)first + AHEAD * TILE) * (BF16 ? 2 : 4) + lane * 128));
    float v[PER];
    load_tile<BF16, VEC>(base, first, left, v);
    const float m = largest(v);
    const uint32_t mine = order_of(m);
    if (t == 0) {
      // the k-th largest of the lane maxima; where warps have nothing (short rows), for this warp alone the n-th, if there are as many lanes
      const bool alone = n <= 32 && p.vocab - part * p.tiles * TILE < TILE;
      uint32_t x = mine, top = 0, share = 0;
      for (int i = 0; i < (alone ? n : k); ++i) {
        top = __reduce_max_sync(0xffffffffu, x);
        if (x == top) x = 0;
        if (i == k - 1) share = top;
      }
      if (alone) own = max(own, top);
      if (lane == 0) least[warp] = share;
      __syncthreads();
    }
    if (fabsf(m) < INFINITY) sum.add(sum_quickly(v, m));
    else if (!(m == -INFINITY)) sum = {__longlong_as_double(0x7ff8000000000000ll), 0, 0.f};          // NaN or +inf: the row counts for nothing
    uint32_t bound = least[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) bound = min(bound, least[w]);
    bound = max(bound, own);
    if (!__any_sync(0xffffffffu, mine >= bound)) continue;
    auto key = [&](int j) { return (unsigned long long)order_of(v[j]) << 32 | (uint32_t)~(first + place<BF16, VEC>(j)); };
    int all = count;
    auto collect = [&]() {                                 // what reaches the bound behind the list; how many there are then
      if (lane == 0) s.n_list[warp] = count;
      __syncwarp();
      if (mine >= bound) {
        const float least_of_all = from_order(bound);
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (v[j] >= least_of_all) {
            const int at = atomicAdd(&s.n_list[warp], 1);
            if (at < LIST) list[at] = key(j);
          }
      }
      __syncwarp();
      all = *(volatile int*)&s.n_list[warp];
    };
    collect();
    if (all > LIST) {                                      // more than there is room for: first only the n best of those before, then of these
      put_in_order();
      bound = max(bound, own);
      collect();
      if (all > LIST) {
        uint32_t cut;
        int end;
        cut_tile<BF16, VEC>(v, n, cut, end);
        if (lane == 0) s.n_list[warp] = count;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const uint32_t o = order_of(v[j]);
          if (o > cut || o == cut && place<BF16, VEC>(j) <= end) list[atomicAdd(&s.n_list[warp], 1)] = key(j);           // (n at most; LIST >= 2 n)
        }
        __syncwarp();
        all = *(volatile int*)&s.n_list[warp];
      }
    }
    count = all;
    if (count > n + (n > 32 ? n / 2 : 0)) put_in_order();  // (at once where that is one look of every lane: a bound that is behind lets more in)
  }
  if (count > n) put_in_order();
  __syncthreads();
  uint32_t bound = s.least[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) bound = min(bound, s.least[w]);
  unsigned long long* found = s.joined;
  for (int i = lane; i < count; i += 32) {
    const unsigned long long x = list[i];
    if ((uint32_t)(x >> 32) >= bound) found[atomicAdd(&s.count, 1)] = x;
  }
  __syncthreads();
  const int have = s.count;
  unsigned long long* out = reinterpret_cast<unsigned long long*>(p.lists) + (row * p.parts + part) * n;
  for (int i = tid; i < have; i += THREADS) {
    const unsigned long long x = found[i];
    int before = 0;
    for (int j = 0; j < have; ++j) before += found[j] > x;
    if (before < n) out[before] = x;
  }
  for (int i = have + tid; i < n; i += THREADS) out[i] = 0ull;
  block_sum(sum, s.sum);
  if (tid == 0) reinterpret_cast<Sum<false>*>(p.sums)[row * p.parts + part] = sum;
}

// total = (x - ref) + base, so that large logits lose nothing; base: score - log of the sum, -inf where the beam offers nothing of its row.
struct Beam {
  double ref, base, off;                   // off: how far totals may be off
};
// Of one beam the larger logit is first, also where 64 bits do not tell the totals apart (logits of 1e-30 beside 0, scores of -1e30), so that fewer
// candidates are the first of more.
struct Candidate {
  double total;
  long long place;                         // beam << 32 | token
  float x;                                 // logit; score of a beam at its end
  __device__ __forceinline__ int beam() const { return (int)(place >> 32); }
  __device__ __forceinline__ bool before(const Candidate& o) const {
    return total > o.total || total == o.total && (x == o.x || beam() != o.beam() ? place < o.place : x > o.x);
  }
};

struct Join {
  Beam beam[MAX_BEAMS];
  unsigned char again[MAX_BEAMS];            // beams whose order is not certain
  unsigned char has_lists[MAX_BEAMS];        // beams that offer tokens,
  unsigned char live[MAX_BEAMS];             // and which they are
  Candidate cand[CAP];                       // any order
  ulonglong2 key[CAP];                       // their totals as numbers, and places
  unsigned short order[CAP];                 // best first
  alignas(16) uint32_t sample[THREADS];
  float bound;
  Sum<true> sum[WARPS], share;
  uint32_t hi[32], lo[32];
  Candidate best[WARPS];
  int from[WARPS], list[MAX_BEAMS];
  int count, n_again, n_live;
  int mixed;                                 // equal totals of one beam whose logits are not
};

__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ Sum<true> of_rank(const Sum<true>* p, uint32_t rank) {
  uint32_t a;
  Sum<true> s;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(s.sum) : "r"(a) : "memory");
  asm volatile("ld.shared::cluster.b32 %0, [%1 + 8];" : "=r"(s.k) : "r"(a) : "memory");
  asm volatile("ld.shared::cluster.f32 %0, [%1 + 12];" : "=f"(s.far) : "r"(a) : "memory");
  return s;
}

// The i-th of a list of a beam that offers tokens, a total of -inf where there is none; lists in those beams' order.
__device__ __forceinline__ Candidate entry_of(const Join& s, const SelectCall& p, size_t row0, int list, int i) {
  const uint32_t at = (uint32_t)list / (uint32_t)p.parts;
  const int w = s.live[at];
  const unsigned long long y = reinterpret_cast<const unsigned long long*>(p.lists)[((row0 + w) * p.parts + ((uint32_t)list - at * p.parts)) * p.n + i];
  const float x = from_order((uint32_t)(y >> 32));
  return {y == 0 ? -INFINITY : ((double)x - s.beam[w].ref) + s.beam[w].base, (long long)w << 32 | (uint32_t)~(uint32_t)y, x};
}
// A sample's total as a number of 32 bits, rounded down, the last eight the thread's, so that no two are equal; lower by how far two totals may be off.
// Of all threads' samples the r-th largest becomes the bound, if it is nearer.
__device__ __forceinline__ void raise_bound(Join& s, double total, double off, int r) {
  const uint32_t key = order_of(__double2float_rd(total - 2 * off)) & ~255u | (uint32_t)(255 - threadIdx.x);
  s.sample[threadIdx.x] = key;
  __syncthreads();
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < THREADS / 4; ++i) {
    const uint4 x = reinterpret_cast<const uint4*>(s.sample)[i];
    above += (int)(x.x > key) + (int)(x.y > key) + (int)(x.z > key) + (int)(x.w > key);
  }
  if (above == r - 1 && key > (ORDER_NONE | 255u)) s.bound = fmaxf(s.bound, from_order(key & ~255u));
  __syncthreads();
}
__device__ __forceinline__ void push(Join& s, const Candidate& c) {
  const int at = atomicAdd(&s.count, 1);
  if (at < CAP) s.cand[at] = c;
}
// Beams at their end offer their score, which is what it is.
__device__ __forceinline__ void push_ended(Join& s, const SelectCall& p, size_t row0) {
  for (int w = threadIdx.x; w < p.beams; w += THREADS) {
    const float score = p.scores[row0 + w];
    if (p.finished && p.finished[row0 + w] && fabsf(score) < INFINITY) {
      s.beam[w] = {0.0, 0.0, 0.0};
      push(s, {(double)score, (long long)w << 32 | p.pad_token, score});
    }
  }
}
// More have come in than are ordered by counting, as the first entries of the lists hold too few of a beam's that is far ahead of the others: a second
// bound, from entries further back.  One at place step - 1 stands for `step` that reach it, so that the n / step-th largest of such is a bound;
// lists of n let in more than CAP only where CAP / n lists or more reach far enough, of which n / step are asked for.  One of 8 beams ahead, 64
// candidates over 248320 tokens: 53 us, and 192 where all were taken for ties.  (Not in line: small calls, which do without it, take 0.3 to 0.4 us of 10 more.)
__device__ __noinline__ void look_further(Join& s, const SelectCall& p, size_t row0, int lists, double off) {
  const int step = max(2, (p.n * p.n + CAP - 1) / CAP);
  const float bound = s.bound;
  double best = -INFINITY;
  for (int list = threadIdx.x; list < lists && step <= p.n; list += THREADS) best = fmax(best, entry_of(s, p, row0, list, step - 1).total);
  raise_bound(s, best, off, (p.n + step - 1) / step);
  const float nearer = s.bound;
  if (!(nearer > bound)) return;                           // ties
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  for (int list = threadIdx.x; list < lists; list += THREADS)
    for (int i = 0; i < p.n; ++i) {
      const Candidate c = entry_of(s, p, row0, list, i);
      if (!(c.total > -INFINITY && c.total >= nearer)) break;
      push(s, c);
    }
  push_ended(s, p, row0);
  __syncthreads();
}

__device__ __forceinline__ void put(const SelectCall& p, int b, int r, const Candidate& c) {
  const size_t at = (size_t)b * p.n + r;
  p.out_scores[at] = (float)c.total;
  p.out_parents[at] = c.beam();
  p.out_tokens[at] = (int)(uint32_t)c.place;
}
// Where counting does not give the order - more candidates about the n-th than it takes, or equal totals of one beam whose logits are not -: the best
// head of all lists, n times.  A thread's lists are its own, list l thread l % THREADS's, their places 16 bits each in s.cand's room.  How many
// there were.  (With the logits in every comparison of the counting, selections took 4 to 40 % longer.)
__device__ __noinline__ int pick_in_turn(Join& s, const SelectCall& p, size_t row0, int b, int rank, int lists) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.n;
  unsigned short* at = reinterpret_cast<unsigned short*>(s.cand);
  const int all = lists + p.beams;                         // (behind the lists: beams at their end)
  for (int l = tid; l < all; l += THREADS) at[l] = l < lists || p.finished && p.finished[row0 + l - lists] && fabsf(p.scores[row0 + l - lists]) < INFINITY ? 0 : 1;
  for (int r = 0; r < n; ++r) {
    Candidate best = {-INFINITY, 0x7fffffffffffffffll, 0.f};
    int from = -1;
    for (int l = tid; l < all; l += THREADS) {
      Candidate c = {-INFINITY, 0, 0.f};
      if (l < lists) {
        if (at[l] < n) c = entry_of(s, p, row0, l, at[l]);
      } else if (at[l] == 0) {
        const float score = p.scores[row0 + l - lists];
        c = {(double)score, (long long)(l - lists) << 32 | p.pad_token, score};
      }
      if (c.total > -INFINITY && c.before(best)) {
        best = c;
        from = l;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Candidate c = {__shfl_xor_sync(0xffffffffu, best.total, o), __shfl_xor_sync(0xffffffffu, best.place, o), __shfl_xor_sync(0xffffffffu, best.x, o)};
      const int l = __shfl_xor_sync(0xffffffffu, from, o);
      if (c.before(best)) {
        best = c;
        from = l;
      }
    }
    __syncthreads();
    if (lane == 0) {
      s.best[warp] = best;
      s.from[warp] = from;
    }
    __syncthreads();
    for (int w = 0; w < WARPS; ++w)
      if (s.best[w].before(best)) {
        best = s.best[w];
        from = s.from[w];
      }
    if (from < 0) return r;
    if (from % THREADS == tid) ++at[from];
    if (tid == 0 && rank == 0) put(p, b, r, best);
  }
  return n;
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(THREADS)
select_join_kernel(const __grid_constant__ SelectCall p) {
  __shared__ Join s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the blocks of a cluster do the same work, apart from the rows that are summed again; the first writes the results
  const int b = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster, W = p.beams, n = p.n;
  pdl_wait();
  pdl_launch_dependents();
  const size_t row0 = (size_t)b * W;
  auto offers = [&](int w) { return fabsf(p.scores[row0 + w]) < INFINITY; };
  auto finished = [&](int w) { return p.finished && p.finished[row0 + w]; };
  const double off = off_of(p.vocab);
  auto settle = [&](int w, double ref, double base, double off) {
    const bool ok = base > -INFINITY && base < INFINITY && ref < INFINITY;             // (not a row with NaN or +inf, or of nothing but -inf)
    s.beam[w] = {ok ? ref : 0.0, ok ? base : -INFINITY, off};
    s.has_lists[w] = ok;
  };
  for (int w = warp; w < W; w += WARPS) {                  // a warp per beam
    const float score = p.scores[row0 + w];
    const bool ended = finished(w);
    Sum<false> sum = {0.0, 0, 0.f};                        // (of a beam that offers nothing: what lies there, and does not count)
    for (int i = lane; i < p.parts; i += 32) sum.add(reinterpret_cast<const Sum<false>*>(p.sums)[(row0 + w) * p.parts + i]);
    warp_sum(sum);
    if (lane == 0) settle(w, sum.ref(), (double)score - log(ended || !(fabsf(score) < INFINITY) ? 0.0 : sum.sum), off);
  }
  for (int w = tid; w < W; w += THREADS) s.again[w] = 0;
  if (tid == 0) s.count = s.n_again = s.mixed = 0;
  __syncthreads();
  // Lists of the beams that offer tokens alone: of the others nothing has been written, and samples of theirs would stand for nothing below (a
  // search's first step, one beam of 8 and 64 candidates over 248320 tokens: 29 us, and 108 with them, as 1984 entries came in and were taken for ties).
  if (warp == 0) {
    int found = 0;
    for (int w0 = 0; w0 < W; w0 += 32) {
      const bool on = w0 + lane < W && s.has_lists[w0 + lane];
      const uint32_t go = __ballot_sync(0xffffffffu, on);
      if (on) s.live[found + __popc(go & ((1u << lane) - 1))] = (unsigned char)(w0 + lane);
      found += __popc(go);
    }
    if (lane == 0) s.n_live = found;
  }
  __syncthreads();
  const int lists = s.n_live * p.parts;
  auto of_beam = [&](int w, float x) { return ((double)x - s.beam[w].ref) + s.beam[w].base; };
  auto entry = [&](int list, int i) { return entry_of(s, p, row0, list, i); };
  // A bound from below of the n-th largest: that of THREADS of them, the first d of every list or the best of several lists' first.
  const int d = lists < THREADS ? min(n, THREADS / max(1, lists)) : 1;
  Candidate mine = {-INFINITY, 0, 0.f};
  if (lists <= THREADS) {
    if (tid < lists * d) mine = entry((uint32_t)tid / (uint32_t)d, (uint32_t)tid % (uint32_t)d);
  } else {
    for (int list = tid; list < lists; list += THREADS) mine.total = fmax(mine.total, entry(list, 0).total);
  }
  if (tid == 0) s.bound = -INFINITY;
  const bool all = lists * n <= THREADS;                   // every thread holds one, and there are no others
  if (lists * n > FEW) raise_bound(s, mine.total, off, n);
  else __syncthreads();
  const double bound = s.bound;
  auto reaches = [&](const Candidate& c) { return c.total > -INFINITY && c.total >= bound; };
  if (all) {
    if (reaches(mine)) push(s, mine);
  } else {
    for (int list = tid; list < lists; list += THREADS)    // a thread per list, whose entries are in order, four on their way at a time
      for (int i = 0; i < n; i += 4) {
        Candidate c[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) c[x] = i + x < n ? entry(list, i + x) : Candidate{-INFINITY, 0, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (reaches(c[x])) push(s, c[x]);
        if (!reaches(c[3])) break;
      }
  }
  push_ended(s, p, row0);
  __syncthreads();
  if (s.count > CAP) look_further(s, p, row0, lists, off);
  const int count = s.count;
  const bool ties = count > CAP;                           // more candidates about the n-th than are ordered by counting
  for (;;) {
    if (ties) {
      for (int w = tid; w < W; w += THREADS) s.again[w] = W > 1 && s.beam[w].base > -INFINITY && s.beam[w].off > 0.0;
    } else {
      for (int i = tid; i < count; i += THREADS) s.key[i] = make_ulonglong2(order_of(s.cand[i].total), (unsigned long long)s.cand[i].place);
      __syncthreads();
      for (int i = tid; i < count; i += THREADS) {
        const ulonglong2 x = s.key[i];
        int better = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) {
          const ulonglong2 y = s.key[j];
          better += (int)(y.x > x.x) | ((int)(y.x == x.x) & (int)(y.y < x.y));         // (no branches)
        }
        s.order[better] = (unsigned short)i;
      }
      __syncthreads();
      // Neighbours among the n best and as many behind them as may belong before the last.  (That is enough: where two of
      // different beams are nearer than their bounds and others lie between them, so are two neighbours of different beams on the way.)
      for (int r = tid; r + 1 < count; r += THREADS) {
        const Candidate &x = s.cand[s.order[r]], &y = s.cand[s.order[r + 1]];
        if (r >= n && s.cand[s.order[n - 1]].total - y.total > 2 * off) break;
        const int v = x.beam(), w = y.beam();
        if (v != w && x.total - y.total <= s.beam[v].off + s.beam[w].off) s.again[v] = s.again[w] = 1;
        if (x.total == y.total && v == w && x.x < y.x) s.mixed = 1;
      }
    }
    __syncthreads();
    if (warp == 0) {
      int found = 0;
      for (int w0 = 0; w0 < W; w0 += 32) {
        const bool on = w0 + lane < W && s.again[w0 + lane] && s.beam[w0 + lane].off > 0.0;
        const uint32_t go = __ballot_sync(0xffffffffu, on);
        if (on) s.list[found + __popc(go & ((1u << lane) - 1))] = w0 + lane;
        found += __popc(go);
      }
      if (lane == 0) s.n_again = found;
      if (found) {
        const double T = exp2(lane / 32.0);
        s.hi[lane] = (uint32_t)__double2hiint(T);
        s.lo[lane] = (uint32_t)__double2loint(T);
      }
    }
    __syncthreads();
    if (s.n_again == 0) break;
    const Table table = {s.hi, s.lo};
    for (int a = 0; a < s.n_again; ++a) {                  // (every beam once at most: its `off` is 0 afterwards)
      const int w = s.list[a];
      const char* base = reinterpret_cast<const char*>(p.logits) + (row0 + w) * (size_t)p.row_stride * (BF16 ? 2 : 4);
      Sum<true> sum = {0.0, 0, 0.f};
#pragma unroll 1
      for (int first = (rank * WARPS + warp) * WARP_TILE; first < p.vocab; first += p.cluster * TILE) {
        float v[PER];
        load_tile<BF16, VEC>(base, first, p.vocab - first, v);
        const float m = largest(v);
        if (fabsf(m) < INFINITY) sum.add(sum_exactly(v, m, table));        // (others than -inf are not among a beam's that offers)
      }
      block_sum(sum, s.sum);
      if (p.cluster > 1) {                                 // (all blocks of a cluster come here for the same beams)
        if (tid == 0) s.share = sum;
        cluster_sync();
        if (warp == 0) {
          sum = of_rank(&s.share, lane < p.cluster ? lane : 0);
          if (lane >= p.cluster) sum.sum = 0.0;
          warp_sum(sum);
        }
        cluster_sync();                                    // read before the next beam's, or the block's end
      }
      // The logarithm relative to the row's largest logit m, which is taken out of the sum as it went in: log sum = m + log1p(the others / exp m),
      // so that the total of a token that is the only one is the score itself and beams that are equal by that stay equal.
      if (warp == 0) {
        uint32_t top = 0;
        for (int i = lane; i < p.parts; i += 32)
          top = max(top, (uint32_t)(reinterpret_cast<const unsigned long long*>(p.lists)[((row0 + w) * p.parts + i) * n] >> 32));
        const float m = from_order(__reduce_max_sync(0xffffffffu, top));
        if (lane == 0) {
          const Sum<true> own = sum_of_one(m, table);
          const double all = sum.k == own.k && sum.far == own.far ? sum.sum : sum.sum * exp(sum.ref() - own.ref());
          settle(w, (double)m, (double)p.scores[row0 + w] - log1p(fmax(all - own.sum, 0.0) / exp((double)m - own.ref())), 0.0);
        }
      }
      __syncthreads();
    }
    if (!ties)
      for (int i = tid; i < count; i += THREADS) {
        Candidate& c = s.cand[i];
        c.total = of_beam(c.beam(), c.x);
      }
    __syncthreads();
  }
  int done = min(count, n);
  if (!ties && !s.mixed) {
    for (int r = tid; r < done && rank == 0; r += THREADS) put(p, b, r, s.cand[s.order[r]]);
  } else {
    done = pick_in_turn(s, p, row0, b, rank, lists);
  }
  for (int r = done + tid; r < n && rank == 0; r += THREADS) {
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
      a.tiles < 1 || a.parts < 1 || (long long)a.parts * a.beams + a.beams > select::CAP * 8 || a.vocab > 1 << 29 ||
      ((long long)a.vocab + select::TILE - 1) / select::TILE > (long long)a.parts * a.tiles || (long long)a.requests * a.beams > 65535 ||
      a.pad_token < 0 || a.pad_token >= a.vocab)
    return -ERR_BAD_ARG;
  const dim3 grid(a.parts, a.requests * a.beams), block(select::THREADS);
  SelectCall c = a;
  c.cluster = 8;
  while (c.cluster > 1 && c.cluster * c.requests > 148 * 3) c.cluster /= 2;
  auto both = [&](auto parts, auto joined) {
    cudaError_t e = launch_pdl(parts, grid, block, 0, c.stream, c);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c.requests * c.cluster);
    cfg.blockDim = block;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = c.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = c.cluster > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, joined, c);
  };
  using namespace select;
  if (a.bf16) return a.vectors ? both(select_parts_kernel<true, true>, select_join_kernel<true, true>) : both(select_parts_kernel<true, false>, select_join_kernel<true, false>);
  return a.vectors ? both(select_parts_kernel<false, true>, select_join_kernel<false, true>) : both(select_parts_kernel<false, false>, select_join_kernel<false, false>);
}
