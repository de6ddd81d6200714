// The care of a paged cache's blocks, for every (layer, K / V) plane at once: block prefixes copied, sequences forked,
// live blocks moved together. A block is opaque bytes: block_size slots of `slot_bytes` and, in a 4-bit cache, behind
// them block_size slots of `scale_bytes` (fp4_common.h), so the first n slots of a block are one or two runs. The planes
// lie one behind the other, kv[plane][block].
//
// Everything is a copy, bound by HBM (each byte read and written once) once it is more than a launch: a workgroup moves
// 16 KB, each lane four 16-byte pieces whose loads are issued before the first store, without a branch where the chunk is
// whole. 12 layers of 2 kv heads in bf16, 604 MB moved by a compaction: 126-131 us with its plan (6), 4.9-5.0 TB/s, the
// rate of a large copy; 156 us with branches around each piece and stores that stay in the caches. 28 layers, 32 children of 24
// parents, 252 MB: 43.5 us (a parent's block is read from memory once for all its children), 59 us so. Two pieces a lane 45.0
// us, eight 42.3; 4096 workgroups for the moves in place of 2048: the same. The same in 4 bits: 174 MB 42.8 us, 67 MB 16.2.
#include "vox_common.h"
#include "vox_kernels.h"

namespace vox {

namespace {

constexpr int kThreadsPages = 256;
constexpr int kPerLanePages = 4;
constexpr int kChunkBytes = kThreadsPages * kPerLanePages * 16;

__device__ __forceinline__ int64_t block_bytes(const PagesArgs& a) {
  return (int64_t)a.block_size * (a.slot_bytes + a.scale_bytes);
}

// Bytes [base, base + kChunkBytes) of the first `bytes` bytes of a run. Non-temporal stores: they need not displace what
// is in the caches (ONCE: nor do the loads, of blocks that nothing reads again).
template <bool ONCE>
__device__ __forceinline__ void copy_chunk(uint8_t* dst, const uint8_t* src, int64_t bytes, int64_t base) {
  const auto load = [](const uint8_t* x) {
    return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x)) : ld_g16(x);
  };
  const auto store = [](uint8_t* x, u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(x)); };
  const int at = (int)threadIdx.x * 16;
  if (base + kChunkBytes <= bytes) {  // workgroup-uniform
    u32x4 v[kPerLanePages];
#pragma unroll
    for (int i = 0; i < kPerLanePages; ++i) v[i] = load(src + base + i * kThreadsPages * 16 + at);
#pragma unroll
    for (int i = 0; i < kPerLanePages; ++i) store(dst + base + i * kThreadsPages * 16 + at, v[i]);
    return;
  }
  for (int64_t off = base + at; off < bytes; off += kThreadsPages * 16) {
    if (off + 16 <= bytes)
      store(dst + off, load(src + off));
    else
      for (int64_t k = off; k < bytes; ++k) dst[k] = src[k];  // a run's last bytes: one lane's
  }
}

// Chunk `chunk` of the first n slots of block src, to block dst: the slots' chunks first, then the scales'.
template <bool ONCE>
__device__ __forceinline__ void copy_slots(const PagesArgs& a, int64_t plane, int src, int dst, int n, int chunk) {
  const int64_t bb = block_bytes(a);
  const uint8_t* s = a.kv + (plane * a.num_blocks + src) * bb;
  uint8_t* d = a.kv + (plane * a.num_blocks + dst) * bb;
  const int slot_chunks = (int)(((int64_t)a.block_size * a.slot_bytes + kChunkBytes - 1) / kChunkBytes);
  if (chunk < slot_chunks) {
    copy_chunk<ONCE>(d, s, (int64_t)n * a.slot_bytes, (int64_t)chunk * kChunkBytes);
  } else {
    const int64_t at = (int64_t)a.block_size * a.slot_bytes;
    copy_chunk<ONCE>(d + at, s + at, (int64_t)n * a.scale_bytes, (int64_t)(chunk - slot_chunks) * kChunkBytes);
  }
}

// Chunks of a whole block, as copy_slots numbers them.
__host__ __device__ inline int64_t chunks_of(int block_size, int64_t slot_bytes, int64_t scale_bytes) {
  return ((int64_t)block_size * slot_bytes + kChunkBytes - 1) / kChunkBytes +
         ((int64_t)block_size * scale_bytes + kChunkBytes - 1) / kChunkBytes;
}

// Workgroup (entry, plane, chunk): entries (src block, dst block, n slots); those with a block outside the cache or
// n <= 0 do nothing, n is clipped to block_size.
__global__ __launch_bounds__(kThreadsPages) void copy_entries_kernel(PagesArgs a, const int32_t* entries) {
  const int e = blockIdx.x;
  const int src = entries[3 * e], dst = entries[3 * e + 1], n = min(entries[3 * e + 2], a.block_size);
  if (n <= 0 || src < 0 || src >= a.num_blocks || dst < 0 || dst >= a.num_blocks) return;
  copy_slots<false>(a, blockIdx.y, src, dst, n, (int)blockIdx.z);
}

// Fork i: the child of row parents[i] shares its full blocks and has the copy new_blocks[i] of its last, partly filled
// one. Workgroup (fork, plane, chunk); the first of a fork also writes the child's table row and length.
__global__ __launch_bounds__(kThreadsPages) void fork_kernel(PagesArgs a, ForkArgs f) {
  const int i = blockIdx.x;
  const int p = f.parents[i], fresh = f.new_blocks[i];
  const bool known = p >= 0 && p < f.batch;
  const int len = known ? max(0, min(f.context_lens[p], f.max_blocks * a.block_size)) : 0;
  const int full = len / a.block_size, tail = len % a.block_size;
  const int32_t* row = f.block_tables + (int64_t)(known ? p : 0) * f.bt_stride;
  const int src = tail > 0 ? row[full] : -1;
  const bool copies = src >= 0 && src < a.num_blocks && fresh >= 0 && fresh < a.num_blocks;
  if (blockIdx.y == 0 && blockIdx.z == 0) {
    for (int c = threadIdx.x; c < f.max_blocks; c += kThreadsPages)
      f.child_tables[(int64_t)i * f.max_blocks + c] = c < full ? row[c] : (c == full && copies ? fresh : -1);
    if (threadIdx.x == 0) f.child_lens[i] = len;
  }
  if (copies && fresh != src) copy_slots<false>(a, blockIdx.y, src, fresh, tail, (int)blockIdx.z);
}

// ---- compaction

constexpr int kPlanThreads = 1024;

// Sum over the workgroup's threads, and this thread's exclusive prefix (scratch: 16 ints of LDS).
__device__ __forceinline__ int block_scan(int x, int* total, int* scratch) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int incl = wave_incl_scan(x, lane);
  if (lane == 63) scratch[w] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    before += i < w ? scratch[i] : 0;
    all += scratch[i];
  }
  __syncthreads();
  *total = all;
  return before + incl - x;
}

// The plan, by one workgroup: a bitmap of the live blocks (those a table names within its context) in LDS; with L of
// them, the live blocks from L on (movers) go to the dead ones below L (holes), the r-th to the r-th: as many of the one
// as of the other, and no mover's place is another's source, so the copies need no order.
//   moves  int32 [2 num_blocks + 1]: the count, then (from, to) of each
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PagesArgs a, CompactArgs c) {
  extern __shared__ uint32_t bits[];
  __shared__ int scratch[kPlanThreads / 64];
  const int tid = threadIdx.x;
  const int n = (int)a.num_blocks;
  const int words = (n + 31) / 32;
  for (int w = tid; w < words; w += kPlanThreads) bits[w] = 0;
  __syncthreads();
  const int64_t cells = (int64_t)c.batch * c.max_blocks;
  auto cell = [&](int64_t x, int& id) {  // whether table cell x lies within its context
    const int b = (int)(x / c.max_blocks), col = (int)(x - (int64_t)b * c.max_blocks);
    id = c.block_tables[(int64_t)b * c.bt_stride + col];
    return (int64_t)col * a.block_size < c.context_lens[b];
  };
  for (int64_t x = tid; x < cells; x += kPlanThreads) {
    int id;
    if (cell(x, id) && id >= 0 && id < n) atomicOr(&bits[id >> 5], 1u << (id & 31));
  }
  __syncthreads();
  // a thread's words: `per` consecutive ones
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  const int w0 = min(words, tid * per), w1 = min(words, w0 + per);
  int mine = 0, live = 0;
  for (int w = w0; w < w1; ++w) mine += __builtin_popcount(bits[w]);
  block_scan(mine, &live, scratch);
  // the bits of word w that are live at or past `live`, and dead below it
  auto below = [&](int w) { return live >= (w + 1) * 32 ? ~0u : live <= w * 32 ? 0u : (1u << (live - w * 32)) - 1u; };
  int holes = 0, movers = 0, total = 0;
  for (int w = w0; w < w1; ++w) {
    const uint32_t lo = below(w);
    holes += __builtin_popcount(~bits[w] & lo);
    movers += __builtin_popcount(bits[w] & ~lo);
  }
  int rh = block_scan(holes, &total, scratch);
  int rm = block_scan(movers, &total, scratch);
  for (int w = w0; w < w1; ++w) {
    const uint32_t lo = below(w), v = bits[w];
    for (uint32_t x = ~v & lo; x; x &= x - 1) c.moves[2 + 2 * rh++] = w * 32 + __builtin_ctz(x);
    for (uint32_t x = v & ~lo; x; x &= x - 1) c.moves[1 + 2 * rm++] = w * 32 + __builtin_ctz(x);
  }
  for (int i = tid; i < n; i += kPlanThreads)
    c.remap[i] = (bits[i >> 5] >> (i & 31)) & 1u ? i : -1;
  if (tid == 0) {
    c.moves[0] = total;
    c.live[0] = live;
  }
  __syncthreads();  // (orders the workgroup's global stores for its own loads, too)
  for (int r = tid; r < total; r += kPlanThreads) c.remap[c.moves[1 + 2 * r]] = c.moves[2 + 2 * r];
  __syncthreads();
  for (int64_t x = tid; x < cells; x += kPlanThreads) {
    int id;
    const bool in = cell(x, id);
    c.new_tables[x] = !in ? -1 : id >= 0 && id < n ? c.remap[id] : id;  // (an entry that names no block stays)
  }
}

// The moves, by a fixed grid over (move, plane, chunk): how many there are is known on the device only.
__global__ __launch_bounds__(kThreadsPages) void compact_copy_kernel(PagesArgs a, CompactArgs c) {
  const int64_t chunks = chunks_of(a.block_size, a.slot_bytes, a.scale_bytes);
  const int64_t per = chunks * a.num_planes;
  const int64_t items = c.moves[0] * per;
  for (int64_t x = blockIdx.x; x < items; x += gridDim.x) {
    const int64_t r = x / per, rest = x - r * per;
    const int64_t plane = rest / chunks;
    copy_slots<true>(a, plane, c.moves[1 + 2 * r], c.moves[2 + 2 * r], a.block_size, (int)(rest - plane * chunks));
  }
}

}  // namespace

hipError_t launch_copy_entries(const PagesArgs& a, const int32_t* entries, int num_entries, hipStream_t stream) {
  const dim3 grid((unsigned)num_entries, (unsigned)a.num_planes,
                  (unsigned)chunks_of(a.block_size, a.slot_bytes, a.scale_bytes));
  copy_entries_kernel<<<grid, dim3(kThreadsPages), 0, stream>>>(a, entries);
  return hipGetLastError();
}

hipError_t launch_fork(const PagesArgs& a, const ForkArgs& f, hipStream_t stream) {
  const dim3 grid((unsigned)f.num_forks, (unsigned)a.num_planes,
                  (unsigned)chunks_of(a.block_size, a.slot_bytes, a.scale_bytes));
  fork_kernel<<<grid, dim3(kThreadsPages), 0, stream>>>(a, f);
  return hipGetLastError();
}

hipError_t launch_compact(const PagesArgs& a, const CompactArgs& c, hipStream_t stream) {
  const size_t lds = (size_t)((a.num_blocks + 31) / 32) * 4;
  compact_plan_kernel<<<dim3(1), dim3(kPlanThreads), lds, stream>>>(a, c);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  compact_copy_kernel<<<dim3(2048), dim3(kThreadsPages), 0, stream>>>(a, c);
  return hipGetLastError();
}

}  // namespace vox
