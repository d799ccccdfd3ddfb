// Trees of drafted tokens, sm_100a: positions and masks of their rows, and the path that the target agrees with.
//
// Row q_start + i of a sequence is node i of its tree; parent[i] < i is the node that it continues, -1 the context (node 0 always: the
// token that the target has chosen already).  b200_attn_tree (attn_spans.cu) attends with what tree_layout_kernel gives; tree_accept_kernel
// walks from node 0 to the lowest child that holds the token predicted at its parent, for as long as there is one, and moves the
// path's rows of every layer's caches up behind the context.
//
// What bounds them: a small launch's latency (one tree of 7 nodes 2.3 us, and 2.6 with its rows in 16 layers); 64 trees of 61 nodes, whose
// walks are nine steps through L1, 4.5 us; their accepted rows, 25 MB in and out in pieces of 256 bytes, 13 to 17 us, of which the walk, the
// pages and the first reads are a chain of 5 (16.5 instead of 13 with the nodes, the predictions and the pages in four waits and not two).
#include "../ptx/sm100.cuh"
#include "launch.h"
#include "ops.h"

namespace b200 {
namespace tree {

constexpr int MAX_NODES = 1024, MAX_PATH = 256;
constexpr int PAGES = 64;
constexpr int THREADS = 128;
constexpr int RESIDENT = 148 * 16;         // blocks of THREADS threads that run at once

// A warp per row: all lanes walk to the context together, lane w keeps word w of the mask.
__global__ void __launch_bounds__(256)
tree_layout_kernel(const int* __restrict__ parents, const int* __restrict__ q_start, const int* __restrict__ q_len, const int* __restrict__ kv_len,
                   int batch, int T, int words, int* __restrict__ positions, uint32_t* __restrict__ mask) {
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= T) return;
  int first = -1, context = 0;
  for (int base = 0; base < batch && first < 0; base += 32) {            // a sequence per lane
    int q0 = 0, n = 0;
    if (base + lane < batch) {
      q0 = q_start[base + lane];
      n = q_len[base + lane];
    }
    const uint32_t here = __ballot_sync(0xffffffffu, q0 >= 0 && row >= q0 && row - q0 < n);
    if (here) {
      const int src = __ffs(here) - 1;
      first = __shfl_sync(0xffffffffu, q0, src);
      context = kv_len[base + src] - __shfl_sync(0xffffffffu, n, src);
    }
  }
  uint32_t mine = 0;
  int depth = 0;
  if (first >= 0) {
    int node = row - first;
    mine = lane == node >> 5 ? 1u << (node & 31) : 0u;
    for (int up = parents[row]; up >= 0 && up < node; up = parents[first + node]) {      // (a parent behind its child ends the walk)
      node = up;
      if (lane == node >> 5) mine |= 1u << (node & 31);
      ++depth;
    }
  }
  if (lane < words) mask[(size_t)row * words + lane] = mine;
  if (lane == 0) positions[row] = first >= 0 ? context + depth : 0;      // (rows of no sequence: 0, and no node)
}

// Rows of the path move to lower places of their own sequence only, row i to place i: path[j] > i for every j > i, so that what is read
// later has not been written, and a thread that takes the same bytes of every row in turn needs no other.
template <typename V>
__device__ __forceinline__ void move_rows(char* at, const long long* src, const long long* dst, int moves, int row_bytes) {
  constexpr int AHEAD = 8;
  for (int i = 0; i < moves; i += AHEAD) {
    V x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i + k < moves) x[k] = *reinterpret_cast<const V*>(at + src[i + k] * row_bytes);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i + k < moves) *reinterpret_cast<V*>(at + dst[i + k] * row_bytes) = x[k];
  }
}

// Block (x, b): every block of a sequence walks its path, the first writes it down, each moves a share of the rows' bytes.
__global__ void __launch_bounds__(THREADS)
tree_accept_kernel(const __grid_constant__ AcceptCall p) {
  __shared__ int s_child[MAX_NODES], s_predicted[MAX_NODES];
  __shared__ int s_pages[PAGES];                           // of the tree's first keys
  __shared__ int s_path[MAX_PATH];
  __shared__ long long s_src[MAX_PATH], s_dst[MAX_PATH];
  __shared__ int s_count, s_moves;
  const int b = blockIdx.y, tid = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int q0 = p.q_start[b], len = p.q_len[b];
  const int n = q0 < 0 ? 0 : max(0, min(min(len, p.T - q0), MAX_NODES));
  // What has to be read before the rows comes in two waits, the pages of the keys with the nodes.
  const int first = p.n_caches ? p.kv_len[b] - len : 0, page0 = p.n_caches ? max(0, first) / p.block_size : 0;
  const int* pages = p.block_table + (size_t)b * p.max_blocks;
  for (int i = tid; i < PAGES && page0 + i < p.max_blocks; i += THREADS) s_pages[i] = pages[page0 + i];
  int up[MAX_NODES / THREADS], token[MAX_NODES / THREADS];
#pragma unroll
  for (int x = 0; x < MAX_NODES / THREADS; ++x) {
    const int i = x * THREADS + tid;
    if (i < n) {
      up[x] = p.parents[q0 + i];
      token[x] = p.tokens[q0 + i];
      s_predicted[i] = p.predicted[q0 + i];
      s_child[i] = MAX_NODES;
    }
  }
  if (tid == 0) s_moves = 0;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < MAX_NODES / THREADS; ++x) {
    const int i = x * THREADS + tid;
    if (i < n && up[x] >= 0 && up[x] < i && token[x] >= 0 && token[x] == s_predicted[up[x]]) atomicMin(&s_child[up[x]], i);
  }
  __syncthreads();
  if (tid == 0) {
    int c = 0, count = 0;
    while (c < n && count < p.max_path) {                                // (a child lies behind its parent, so that this ends)
      s_path[count++] = c;
      c = s_child[c];
    }
    s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  if (blockIdx.x == 0) {
    for (int i = tid; i < p.max_path; i += THREADS) {
      const int node = i < count ? s_path[i] : -1;
      p.path[(size_t)b * p.max_path + i] = node;
      p.emitted[(size_t)b * p.max_path + i] = node < 0 ? -1 : s_predicted[node];
    }
    if (tid == 0) p.count[b] = count;
  }
  if (p.n_caches == 0 || count <= 1) return;
  // Places of the rows that move, in the path's order, as (page, row of it).
  const auto page_of = [&](int key) {
    const int page = key / p.block_size;
    return page - page0 < PAGES ? s_pages[page - page0] : pages[page];
  };
  if (tid < 32) {
    int moves = 0;
    for (int base = 0; base < count; base += 32) {
      const int i = base + tid, from = i < count ? s_path[i] : i;
      long long src = 0, dst = 0;
      bool ok = from != i && first >= 0 && (long long)first + from < (long long)p.max_blocks * p.block_size;
      if (ok) {
        const int ps = page_of(first + from), pd = page_of(first + i);
        ok = (unsigned)ps < (unsigned)p.num_blocks && (unsigned)pd < (unsigned)p.num_blocks;
        src = (long long)ps << 32 | (first + from) % p.block_size;
        dst = (long long)pd << 32 | (first + i) % p.block_size;
      }
      const uint32_t go = __ballot_sync(0xffffffffu, ok);
      if (ok) {
        const int to = moves + __popc(go & ((1u << tid) - 1));
        s_src[to] = src;
        s_dst[to] = dst;
      }
      moves += __popc(go);
    }
    if (tid == 0) s_moves = moves;
  }
  __syncthreads();
  const int moves = s_moves;
  if (moves == 0) return;
  uint32_t base = 0;                                                     // columns of the caches before this one
  const uint32_t step = gridDim.x * THREADS, mine = blockIdx.x * THREADS + tid;
  int heads = 0;
  for (int c = 0; c < p.n_caches; ++c) {
    const AcceptCache& k = p.caches[c];
    if (k.heads != heads) {                                              // places as rows of this cache's first head
      __syncthreads();
      for (int i = tid; i < moves; i += THREADS) {
        const auto row = [&](long long x) {
          return heads == 0 ? (x >> 32) * k.heads * p.block_size + (x & 0xffffffffll)
                            : x / ((long long)heads * p.block_size) * k.heads * p.block_size + x % p.block_size;
        };
        s_src[i] = row(s_src[i]);
        s_dst[i] = row(s_dst[i]);
      }
      heads = k.heads;
      __syncthreads();
    }
    const uint32_t per_row = k.row_bytes / k.vec, columns = (uint32_t)k.layers * k.heads * per_row, skip = base % step;
    for (uint32_t col = mine >= skip ? mine - skip : mine + step - skip; col < columns; col += step) {
      const uint32_t y = col / per_row, layer = y / k.heads, head = y - layer * k.heads;
      char* to = reinterpret_cast<char*>(k.base) + layer * k.layer_bytes + (long long)head * p.block_size * k.row_bytes + (col - y * per_row) * k.vec;
      if (k.vec == 16) move_rows<uint4>(to, s_src, s_dst, moves, k.row_bytes);
      else move_rows<uint32_t>(to, s_src, s_dst, moves, k.row_bytes);
    }
    base += columns;
  }
}

}  // namespace tree
}  // namespace b200

using namespace b200;

extern "C" int b200_tree_layout(const TreeLayoutCall* call) {
  const TreeLayoutCall& a = *call;
  if (a.bytes != (int)sizeof(a) || a.T < 1 || a.batch < 0 || a.words < 1 || a.words > tree::MAX_NODES / 32) return -ERR_BAD_ARG;
  return (int)launch_pdl(tree::tree_layout_kernel, dim3((a.T + 7) / 8), dim3(256), 0, a.stream, a.parents, a.q_start, a.q_len, a.kv_len, a.batch, a.T,
                         a.words, a.positions, a.mask);
}

extern "C" int b200_tree_accept(const AcceptCall* call) {
  const AcceptCall& a = *call;
  if (a.bytes != (int)sizeof(a) || a.batch < 1 || a.batch > 65535 || a.T < 0 || a.max_path < 1 || a.max_path > tree::MAX_PATH || a.n_caches < 0 ||
      a.n_caches > ACCEPT_CACHES || (a.n_caches && (a.block_size < 1 || a.max_blocks < 1 || a.num_blocks < 1)))
    return -ERR_BAD_ARG;
  long long columns = 0;
  for (int c = 0; c < a.n_caches; ++c) {
    const AcceptCache& k = a.caches[c];
    if (k.layers < 1 || k.heads < 1 || k.row_bytes < 4 || (k.vec != 16 && k.vec != 4) || k.row_bytes % k.vec) return -ERR_BAD_ARG;
    columns += (long long)k.layers * k.heads * (k.row_bytes / k.vec);
  }
  if (columns > 0x7fffffffll) return -ERR_BAD_ARG;
  // a column of bytes per thread, as long as all blocks run at once
  const long long want = (columns + tree::THREADS - 1) / tree::THREADS, most = tree::RESIDENT / a.batch;
  const int slices = (int)(want < 1 || most < 1 ? 1 : want < most ? want : most);
  return (int)launch_pdl(tree::tree_accept_kernel, dim3(slices, a.batch), dim3(tree::THREADS), 0, a.stream, a);
}
