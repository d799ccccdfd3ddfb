// States that follow the beams, in place, sm_100a: state[slot of beam w] <- state[slot of beam parent[w]] for all beams of a request at
// once, in several tensors.
//
// A share of the state's bytes - the same columns of every beam of one request - is one item: all wanted parents' columns come into shared
// memory, each once, then go to the beams that continue them.  Nothing else touches those columns, so no beam is overwritten before
// it has been read, whatever cycles the parents make, and there is no copy of the state anywhere else.  Beams that continue themselves move
// nothing.
//
// What bounds it is memory (16 beams of 13 to 103 MB, copies in and out: 6.0 to 6.5 TB/s where 14 or 16 of them move, 5.2 to 5.5 where 10 of 16 do,
// whose items are less full): warp 0 keeps bulk copies of items on their way
// both in and out, STAGES items in shared memory; it only issues them.  Warps 1 to 3 do the tensors whose rows are no multiples of 16 bytes (tables, tails) by plain loads, at the same time.
#include "../ptx/sm100.cuh"
#include "launch.h"
#include "ops.h"
#include "per_device.h"

namespace b200 {
namespace reorder {

constexpr int MAX_BEAMS = 128;
constexpr int STAGES = 3, AHEAD = 2;       // an item is loaded AHEAD items before it is stored
constexpr int STAGE_BYTES = 65536;
constexpr int PLAIN_BYTES = 16384;
constexpr int THREADS = 128;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + PLAIN_BYTES + 128;
static_assert(SMEM_BYTES + 4096 <= 232448, "shared memory of a block");

struct Params {
  ReorderCall c;
  int chunk, plain_chunk;                  // bytes of a state that an item takes of every beam
  int bulk_items, plain_items;             // of all tensors
  int items[REORDER_STATES];               // of each
  uint32_t chunks[REORDER_STATES];         // items that a state of each is cut into
};

struct Item {
  char* base;                              // column 0 of slot 0
  long long slot_bytes;
  int bytes;
  int request;
};

// Item `at` of the bulk tensors, or of the others.
__device__ __forceinline__ Item item_of(const Params& p, int at, int bulk, int chunk) {
  int i = 0;
  while (p.c.states[i].bulk != bulk || at >= p.items[i]) {
    if (p.c.states[i].bulk == bulk) at -= p.items[i];
    ++i;
  }
  const ReorderState& s = p.c.states[i];
  const uint32_t chunks = p.chunks[i];
  const uint32_t x = (uint32_t)at / chunks, col = (uint32_t)at - x * chunks, outer = x / (uint32_t)p.c.requests;
  Item it;
  it.request = (int)(x - outer * p.c.requests);
  it.base = reinterpret_cast<char*>(s.base) + outer * s.outer_bytes + (long long)col * chunk;
  it.slot_bytes = s.slot_bytes;
  it.bytes = (int)min((long long)chunk, s.inner_bytes - (long long)col * chunk);
  return it;
}
// Parent of a beam, and where the two are; false: the beam stays as it is (its own parent, none, or a slot that is not there).
__device__ __forceinline__ bool move_of(const ReorderCall& c, int request, int w, int& parent, int& from, int& to) {
  const int* parents = c.parents + (size_t)request * c.beams;
  parent = parents[w];
  if ((unsigned)parent >= (unsigned)c.beams || parent == w) return false;
  const int* slots = c.slots + (size_t)request * c.beams;
  from = c.slots ? slots[parent] : request * c.beams + parent;
  to = c.slots ? slots[w] : request * c.beams + w;
  return (unsigned)from < (unsigned)c.n_slots && (unsigned)to < (unsigned)c.n_slots && from != to;
}

__device__ __forceinline__ void bulk_store(void* dst, const void* smem, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(smem)), "r"(bytes) : "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

template <typename V>
__device__ __forceinline__ void plain_item(const ReorderCall& c, const Item& it, uint8_t* room, int chunk, int tid, int threads) {
  const int n = it.bytes / (int)sizeof(V);
  for (int w = 0; w < c.beams; ++w) {                      // (a parent that several beams continue comes in once for each: into the same place)
    int parent, from, to;
    if (!move_of(c, it.request, w, parent, from, to)) continue;
    V* in = reinterpret_cast<V*>(room + parent * chunk);
    const V* src = reinterpret_cast<const V*>(it.base + from * it.slot_bytes);
    for (int i = tid; i < n; i += threads) in[i] = src[i];
  }
  asm volatile("bar.sync 1, 96;" ::: "memory");
  for (int w = 0; w < c.beams; ++w) {
    int parent, from, to;
    if (!move_of(c, it.request, w, parent, from, to)) continue;
    const V* in = reinterpret_cast<const V*>(room + parent * chunk);
    V* dst = reinterpret_cast<V*>(it.base + to * it.slot_bytes);
    for (int i = tid; i < n; i += threads) dst[i] = in[i];
  }
  asm volatile("bar.sync 1, 96;" ::: "memory");
}

__global__ void __launch_bounds__(THREADS, 1)
reorder_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[STAGES];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const ReorderCall& c = p.c;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  if (warp == 0) {
    const int step = gridDim.x, mine = p.bulk_items <= (int)blockIdx.x ? 0 : (p.bulk_items - (int)blockIdx.x + step - 1) / step;
    // Beams of a request in turn, 32 at a time: with (w, its slot, its parent, whether it moves) of a lane.
    const auto beams = [&](int request, auto with) {
      const int* parents = c.parents + (size_t)request * c.beams;
      const int* slots = c.slots + (size_t)request * c.beams;
      for (int w = lane; w - lane < c.beams; w += 32) {
        int parent = -1, slot = -1;
        if (w < c.beams) {
          parent = parents[w];
          slot = c.slots ? slots[w] : request * c.beams + w;
        }
        bool moves = (unsigned)parent < (unsigned)c.beams && parent != w && (unsigned)slot < (unsigned)c.n_slots;
        if (moves) {
          const int from = c.slots ? slots[parent] : request * c.beams + parent;
          moves = (unsigned)from < (unsigned)c.n_slots && from != slot;
        }
        with(w, slot, parent, moves);
      }
    };
    uint32_t loaded = 0, phases = 0;                       // a bit per stage: its item moves something; parity of its next load
    auto load = [&](int i) {                               // of this block
      const Item it = item_of(p, blockIdx.x + i * step, 1, p.chunk);
      const int st = i % STAGES;
      uint8_t* stage = smem + st * STAGE_BYTES;
      // parents that are wanted: a bit each, 32 to a lane's word
      uint32_t want[MAX_BEAMS / 32] = {};
      beams(it.request, [&](int, int, int parent, bool moves) {
#pragma unroll
        for (int x = 0; x < MAX_BEAMS / 32; ++x)
          if (32 * x < c.beams) want[x] |= __reduce_or_sync(0xffffffffu, moves && parent >> 5 == x ? 1u << (parent & 31) : 0u);
      });
      int n = 0;
#pragma unroll
      for (int x = 0; x < MAX_BEAMS / 32; ++x) n += __popc(want[x]);
      loaded = loaded & ~(1u << st) | (n > 0 ? 1u << st : 0u);
      if (n == 0) return;
      if (lane == 0) mbar_expect_tx(&full[st], n * it.bytes);
      __syncwarp();
#pragma unroll
      for (int x = 0; x < MAX_BEAMS / 32; ++x)
        if (want[x] >> lane & 1) {
          const int w = 32 * x + lane, from = c.slots ? c.slots[(size_t)it.request * c.beams + w] : it.request * c.beams + w;
          bulk_load(stage + w * p.chunk, it.base + from * it.slot_bytes, it.bytes, &full[st]);
        }
      __syncwarp();
    };
    bool ok = true;
    for (int i = -AHEAD; i < mine && ok; ++i) {
      if (i + AHEAD < mine) {
        bulk_wait_read<STAGES - AHEAD - 1>();              // what was stored from that stage, STAGES items before, has been read
        __syncwarp();
        load(i + AHEAD);
      }
      const int st = i % STAGES;
      if (i >= 0 && loaded >> st & 1) {
        const Item it = item_of(p, blockIdx.x + i * step, 1, p.chunk);
        ok = __all_sync(0xffffffffu, mbar_wait(&full[st], phases >> st & 1));
        if (!ok) break;
        phases ^= 1u << st;
        beams(it.request, [&](int, int slot, int parent, bool moves) {
          if (moves) bulk_store(it.base + slot * it.slot_bytes, smem + st * STAGE_BYTES + parent * p.chunk, it.bytes);
        });
        __syncwarp();
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");            // (one per item, also of items that store nothing)
    }
    if (!ok) {
      // loads that are still on their way would come into another block's shared memory: wait for them, again with a limit
      if (lane == 0) atomicExch(c.status, ERR_WAIT_TMA);
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else {
    uint8_t* room = smem + STAGES * STAGE_BYTES;
    const int tid = threadIdx.x - 32;
    for (int i = blockIdx.x; i < p.plain_items; i += gridDim.x) {
      const Item it = item_of(p, i, 0, p.plain_chunk);
      const uint32_t low = (uint32_t)(uintptr_t)it.base | (uint32_t)it.slot_bytes | (uint32_t)it.bytes;
      if (low % 4 == 0) plain_item<uint32_t>(c, it, room, p.plain_chunk, tid, 96);
      else if (low % 2 == 0) plain_item<uint16_t>(c, it, room, p.plain_chunk, tid, 96);
      else plain_item<uint8_t>(c, it, room, p.plain_chunk, tid, 96);
    }
  }
}

}  // namespace reorder
}  // namespace b200

using namespace b200;

extern "C" int b200_beam_reorder(const ReorderCall* call) {
  using namespace reorder;
  Params p = {};
  p.c = *call;
  const ReorderCall& a = p.c;
  if (a.bytes != (int)sizeof(a) || a.requests < 1 || a.beams < 1 || a.beams > MAX_BEAMS || a.n_slots < 1 || a.n_states < 1 || a.n_states > REORDER_STATES)
    return -ERR_BAD_ARG;
  long long bulk = 0, all[2] = {0, 0};
  for (int i = 0; i < a.n_states; ++i) {
    const ReorderState& s = a.states[i];
    if (s.outer < 1 || s.inner_bytes < 1 || (s.bulk && ((uintptr_t)s.base | s.outer_bytes | s.slot_bytes | s.inner_bytes) % 16)) return -ERR_BAD_ARG;
    if (s.bulk) bulk += s.inner_bytes * s.outer * a.requests;
  }
  // Items as large as a stage holds: with stages of 32 / 48 / 64 KB 16 beams of 49 MB of one request, all of which move and 11 are wanted (1.33 GB in
  // and out), take 340 / 246 / 206 us, of 4 requests (14 and 12, 1.28 GB) 276 / 216 / 211.  Smaller ones, of 1 KB a beam at least, where every SM
  // would not have two otherwise (8 / 4 / 2 a SM: 15.0 / 9.6 / 6.6 us for the last pages of 4 beams in 16 layers, 25 MB).
  const long long most = STAGE_BYTES / a.beams / 128 * 128, even = bulk / (148 * 2) / 128 * 128;
  p.chunk = (int)(even < 1024 ? (most < 1024 ? most : 1024) : even < most ? even : most);
  p.plain_chunk = PLAIN_BYTES / a.beams / 16 * 16;
  for (int i = 0; i < a.n_states; ++i) {
    const ReorderState& s = a.states[i];
    const int chunk = s.bulk ? p.chunk : p.plain_chunk;
    const long long n = (s.inner_bytes + chunk - 1) / chunk * s.outer * a.requests;
    all[s.bulk != 0] += n;
    if (all[s.bulk != 0] > 0x7fffffffll) return -ERR_BAD_ARG;
    p.c.states[i].bulk = s.bulk != 0;
    p.chunks[i] = (uint32_t)((s.inner_bytes + chunk - 1) / chunk);
    p.items[i] = (int)n;
  }
  p.bulk_items = (int)all[1];
  p.plain_items = (int)all[0];
  static PerDeviceOnce once_;
  bool& configured = once_.slot();
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  const long long n = all[0] > all[1] ? all[0] : all[1];
  return (int)launch_pdl(reorder_kernel, dim3((unsigned)(n < 148 ? n : 148)), dim3(THREADS), SMEM_BYTES, a.stream, p);
}
