// Tokens dropped from a paged cache by what they have received of the attention, in every layer and kv head at once, in two
// launches: which tokens stay (select_kernel), and their rows moved to the front of the sequence (move_kernel).
//
// select: a workgroup per (kv head, sequence, layer). Of the tokens [sinks, n - recent) the `want` heaviest stay, of equal
// ones the earliest: the want-th largest weight T is found digit by digit, 8 bits a pass over the weights as ordered
// integers (a histogram in LDS, the digit whose count reaches what is still wanted), then tokens above T stay, and the
// first ones equal to T up to the number still wanted. One more pass in token order gives each kept token its place (the
// count of kept ones before it), moves its weight there and leaves the slot it comes from for move_kernel.
//
// Both passes that move work in place: place j takes token i_j >= j, a tile's reads are done before its writes, and a later
// tile reads only behind them. So a sequence's tokens of one kv head are one workgroup's, tile after tile.
#include "vox_common.h"
#include "vox_kernels.h"

namespace vox {

namespace {

constexpr int kSelThreads = 256;
constexpr int kMoveThreads = 256;
constexpr int kMovePieces = 8;  // 16-byte pieces a lane keeps in flight

// Weights as integers of the same order: NaN above everything, the two zeros the same.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u << 1) > 0xff000000u) return 0xffffffffu;
  if ((u << 1) == 0u) return 0x80000000u;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// This thread's exclusive prefix of two counts over the workgroup, and their totals (scratch: 2 ints a wave).
__device__ __forceinline__ void scan2(int a, int b, int (*scratch)[2], int& pa, int& pb, int& ta, int& tb) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int ia = wave_incl_scan_dpp(a), ib = wave_incl_scan_dpp(b);
  if (lane == 63) {
    scratch[w][0] = ia;
    scratch[w][1] = ib;
  }
  __syncthreads();
  pa = ia - a;
  pb = ib - b;
  ta = tb = 0;
#pragma unroll
  for (int x = 0; x < kSelThreads / kWave; ++x) {
    const int va = scratch[x][0], vb = scratch[x][1];
    pa += x < w ? va : 0;
    pb += x < w ? vb : 0;
    ta += va;
    tb += vb;
  }
  __syncthreads();
}

__global__ __launch_bounds__(kSelThreads) void select_kernel(EvictArgs p) {
  __shared__ int hist[256];
  __shared__ int scratch[kSelThreads / kWave][2];
  __shared__ int s_digit, s_want;
  const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
  const int reach = p.max_blocks * p.block_size;
  const int n = max(0, min(p.context_lens[b], reach));
  const int64_t row = p.rows ? (int64_t)p.rows[b] : b;
  const bool drops = n > p.budget && row >= 0 && row < p.row_count;  // workgroup-uniform
  const int left = drops ? p.budget : n;
  const int32_t* table = p.block_tables + (int64_t)b * p.bt_stride;
  const int32_t* into = p.into ? p.into + (int64_t)b * p.into_stride : nullptr;
  if (g == 0 && layer == 0) {
    const int used = (left + p.block_size - 1) / p.block_size;
    for (int c = tid; c < p.max_blocks; c += kSelThreads) {
      int blk = c < used ? table[c] : -1;
      if (drops && into && c < used && into[c] >= 0) blk = into[c];
      p.new_tables[(int64_t)b * p.max_blocks + c] = blk;
    }
    if (tid == 0) p.new_lens[b] = left;
  }
  int32_t* moves = p.moves + (((int64_t)layer * p.batch + b) * p.num_heads + g) * p.kept;
  if (!drops) {
    for (int j = tid; j < left && j < p.kept; j += kSelThreads) moves[j] = -1;
    return;
  }
  float* w = p.weights + (((int64_t)layer * p.row_count + row) * p.num_heads + g) * p.width;
  const int lo = p.sinks, hi = n - p.recent;  // (n > budget >= sinks + recent)
  int want = p.budget - p.sinks - p.recent;
  uint32_t top = 0;  // T's digits so far
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      hist[tid] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t key = ordered(w[i]);
        if (shift == 24 || (key >> (shift + 8)) == (top >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      // digit d holds the want-th largest when fewer than `want` lie in the digits above it and at least as many with it
      const int d = 255 - tid, mine = hist[d];
      int before, unused, total, total2;
      scan2(mine, 0, scratch, before, unused, total, total2);
      if (before < want && before + mine >= want) {
        s_digit = d;
        s_want = want - before;
      }
      __syncthreads();
      top |= (uint32_t)s_digit << shift;
      want = s_want;
      __syncthreads();
    }
  }
  // want: how many of those equal to T stay
  int done = 0, ties = 0;  // kept, and equal ones met, before this tile
  for (int base = 0; base < n; base += kSelThreads) {
    const int i = base + tid;
    const float x = i < n ? w[i] : 0.f;
    const uint32_t key = ordered(x);
    const bool mid = i >= lo && i < hi;
    const bool tie = mid && p.budget > p.sinks + p.recent && key == top;
    bool keep = i < n && (!mid || (p.budget > p.sinks + p.recent && key > top));
    int before, ties_before, kept, met;
    scan2(0, tie, scratch, before, ties_before, kept, met);
    keep = keep || (tie && ties + ties_before < want);
    ties += met;
    scan2(keep, 0, scratch, before, ties_before, kept, met);  // (every read of the tile lies before its barriers)
    if (keep) {
      const int j = done + before;
      w[j] = x;
      const int src = table[i / p.block_size];
      int dst = table[j / p.block_size];
      if (into && into[j / p.block_size] >= 0) dst = into[j / p.block_size];
      const bool there = src >= 0 && src < p.num_blocks && dst >= 0 && dst < p.num_blocks;
      const int64_t from = (int64_t)src * p.block_size + i % p.block_size;
      moves[j] = there && from != (int64_t)dst * p.block_size + j % p.block_size ? (int)from : -1;
    }
    done += kept;
    __syncthreads();
  }
}

// Workgroup (sequence, plane = layer and K / V, kv head): rows of PIECES units of type V, `head_run` bytes a head, `slot_run`
// a slot, from `at` bytes into the block on.
template <typename V>
__device__ __forceinline__ void move_rows(const EvictArgs& p, const int32_t* moves, int left, uint8_t* plane,
                                          int64_t block_bytes, int64_t at, int64_t slot_run, int pieces,
                                          const int32_t* table, const int32_t* into) {
  const int rows = kMoveThreads * kMovePieces / pieces;  // a tile's
  for (int base = 0; base < left; base += rows) {
    V v[kMovePieces];
    uint8_t* dst[kMovePieces];
#pragma unroll
    for (int u = 0; u < kMovePieces; ++u) {
      const int idx = u * kMoveThreads + (int)threadIdx.x;
      const int j = base + idx / pieces, piece = idx % pieces;
      const int from = idx / pieces < rows && j < left ? moves[j] : -1;
      dst[u] = nullptr;
      if (from >= 0) {
        int blk = table[j / p.block_size];
        if (into && into[j / p.block_size] >= 0) blk = into[j / p.block_size];
        const int64_t src = (int64_t)(from / p.block_size) * block_bytes + at + (from % p.block_size) * slot_run;
        dst[u] = plane + (int64_t)blk * block_bytes + at + (j % p.block_size) * slot_run + piece * (int)sizeof(V);
        v[u] = *reinterpret_cast<const V*>(plane + src + piece * (int)sizeof(V));
      }
    }
    wait_vmem_all();  // every read of the tile before its first write
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMovePieces; ++u)
      if (dst[u]) *reinterpret_cast<V*>(dst[u]) = v[u];
  }
}

__global__ __launch_bounds__(kMoveThreads) void move_kernel(EvictArgs p) {
  const int b = blockIdx.x, plane = blockIdx.y, g = blockIdx.z;
  const int n = max(0, min(p.context_lens[b], p.max_blocks * p.block_size));
  const int64_t row = p.rows ? (int64_t)p.rows[b] : b;
  if (n <= p.budget || row < 0 || row >= p.row_count) return;
  const int32_t* moves = p.moves + (((int64_t)(plane >> 1) * p.batch + b) * p.num_heads + g) * p.kept;
  const int32_t* table = p.block_tables + (int64_t)b * p.bt_stride;
  const int32_t* into = p.into ? p.into + (int64_t)b * p.into_stride : nullptr;
  const int64_t block_bytes = (int64_t)p.block_size * p.num_heads * (p.head_bytes + p.scale_bytes);
  uint8_t* base = p.kv + (int64_t)plane * p.num_blocks * block_bytes;
  move_rows<u32x4>(p, moves, p.budget, base, block_bytes, (int64_t)g * p.head_bytes, (int64_t)p.num_heads * p.head_bytes,
                   p.head_bytes / 16, table, into);
  if (p.scale_bytes)
    move_rows<uint32_t>(p, moves, p.budget, base, block_bytes,
                        (int64_t)p.block_size * p.num_heads * p.head_bytes + (int64_t)g * p.scale_bytes,
                        (int64_t)p.num_heads * p.scale_bytes, p.scale_bytes / 4, table, into);
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
  if (a.batch <= 0 || a.layers <= 0 || a.num_heads <= 0) return hipSuccess;
  select_kernel<<<dim3((unsigned)a.num_heads, (unsigned)a.batch, (unsigned)a.layers), dim3(kSelThreads), 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  move_kernel<<<dim3((unsigned)a.batch, (unsigned)(2 * a.layers), (unsigned)a.num_heads), dim3(kMoveThreads), 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace vox
