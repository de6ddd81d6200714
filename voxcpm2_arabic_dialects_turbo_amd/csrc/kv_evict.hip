// Tokens dropped from a paged cache by what they have received of the attention, in every layer and kv head at once, in two
// launches: which tokens stay (select_kernel), and their rows moved to the front of the sequence (move_kernel).
//
// select: a workgroup per (kv head, sequence, layer). Of the tokens [sinks, n - recent) the `want` heaviest stay, of equal
// ones the earliest. The want-th largest weight T is found digit by digit over the weights as ordered integers (ordered), 11,
// 11 and 10 bits, each digit from a histogram in LDS of the weights that share the ones before it. Tokens above T stay, and of
// those equal to T the first ones that are still wanted. Place j of a kept token at i is how many kept ones lie before it:
// (those above T or protected before i) + min(those equal to T before i, still wanted), from ballots and one scan. Its weight
// moves there, and move_kernel gets the pair of slots. Weights are held in registers (lane-contiguous rounds of the
// workgroup); rows longer than those are read again. Bound by the chain of three histograms and scans (8 us for one sequence
// of 28 layers), for long rows by a workgroup's instructions (39 us for 8 sequences of 20000-32768 tokens, 12 layers; eight
// histograms side by side, against lanes that meet in a bin: 38.5).
//
// Both kernels work in place: place j takes token i_j >= j, a round's reads are done before its writes, and a later round
// reads only behind them. So a sequence's tokens of one kv head (and of one slice of a row's bytes) are one workgroup's.
// move is bound by HBM where there are workgroups enough: 48 sequences, 0.98 GB read and written in 382 us, 5.1 TB/s.
#include "vox_common.h"
#include "vox_kernels.h"

namespace vox {

namespace {

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 8;  // rows a lane keeps in flight, twice (a round's, and the next one's)
constexpr int kBins = 2048;
constexpr int kTable = 512;  // blocks of a sequence that a workgroup holds in LDS

// Weights as integers of the same order: NaN above everything, the two zeros the same.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u << 1) > 0xff000000u) return 0xffffffffu;
  if ((u << 1) == 0u) return 0x80000000u;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// This thread's exclusive prefixes of two counts over the workgroup of NW waves, and their totals.
template <int NW>
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
  for (int x = 0; x < NW; ++x) {
    const int va = scratch[x][0], vb = scratch[x][1];
    pa += x < w ? va : 0;
    pb += x < w ? vb : 0;
    ta += va;
    tb += vb;
  }
  __syncthreads();
}

// NT threads, E weights each in registers.
template <int NT, int E>
__global__ __launch_bounds__(NT) void select_kernel(EvictArgs p) {
  constexpr int NW = NT / kWave, CHUNK = NT * E, PER = kBins / NT;
  static_assert(E * NW <= NT && kBins % NT == 0, "a thread scans a count and its bins");
  __shared__ int hist[kBins];
  __shared__ int scratch[NW][2];
  __shared__ int counts[E * NW][2];  // [round][wave]: tokens that stay for sure, and those equal to T
  __shared__ int s_bin, s_want, s_first;
  __shared__ int s_from[kTable], s_to[kTable];  // the blocks of the sequence, and those that take what it keeps
  const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 63, wv = tid >> 6;
  const int bs = p.block_size;
  const int n = max(0, min(p.context_lens[b], p.max_blocks * bs));
  const int64_t row = p.rows ? (int64_t)p.rows[b] : b;
  const bool drops = n > p.budget && row >= 0 && row < p.row_count;  // workgroup-uniform
  const int32_t* table = p.block_tables + (int64_t)b * p.bt_stride;
  const int32_t* into = p.into ? p.into + (int64_t)b * p.into_stride : nullptr;
  if (g == 0 && layer == 0) {
    const int left = drops ? p.budget : n, used = (left + bs - 1) / bs;
    for (int c = tid; c < p.max_blocks; c += NT) {
      int blk = c < used ? table[c] : -1;
      if (drops && into && c < used && into[c] >= 0) blk = into[c];
      p.new_tables[(int64_t)b * p.max_blocks + c] = blk;
    }
    if (tid == 0) p.new_lens[b] = left;
  }
  if (!drops) return;
  float* w = p.weights + (((int64_t)layer * p.row_count + row) * p.num_heads + g) * p.width;
  int2* moves = p.moves + (((int64_t)layer * p.batch + b) * p.num_heads + g) * (p.kept + 1);
  if (tid == 0) s_first = p.budget;  // (before the barriers below)
  const int lo = p.sinks, hi = n - p.recent;  // (n > budget >= sinks + recent)
  int want = p.budget - p.sinks - p.recent;
  const int chunks = (n + CHUNK - 1) / CHUNK;

  const bool held = p.max_blocks <= kTable;
  for (int c = tid; held && c < p.max_blocks; c += NT) {
    const int blk = table[c];
    s_from[c] = blk;
    s_to[c] = into && into[c] >= 0 ? into[c] : blk;
  }
  const int* const from_block = held ? s_from : table;  // (read behind the barriers below)
  const int* const to_block = held ? s_to : table;

  // a lane's weights, and as ordered integers; 0, which none has, for the tokens that are not among the `mid` ones
  float x[E];
  uint32_t key[E];
  auto load = [&](int c) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = c * CHUNK + e * NT + tid;
      x[e] = w[min(i, n - 1)];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = c * CHUNK + e * NT + tid;
      key[e] = i >= lo && i < hi ? ordered(x[e]) : 0u;
    }
  };
  load(0);
  uint32_t top = 0xffffffffu;  // T; where none of the mid ones stays, none is above it, and of those equal to it none is wanted
  if (want > 0) {
    top = 0;
    // T's digits of 11, 11 and 10 bits, each from a histogram of the weights that have the digits before it
#pragma unroll
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const uint32_t span = level == 0 ? 0xffffffffu : level == 1 ? 0x1fffffu : 0x3ffu;
      for (int i = tid; i < kBins; i += NT) hist[i] = 0;
      __syncthreads();
      for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) load(c);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t at = key[e] - top;
          if (level == 0 ? key[e] != 0 : at <= span) atomicAdd(&hist[at >> shift], 1);
        }
      }
      __syncthreads();
      // the bin that holds the want-th: fewer than `want` lie in the bins above it, and not fewer with it. Thread t has
      // bins kBins - 1 - (PER t + [0, PER))
      int mine = 0, cnt[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        cnt[i] = hist[kBins - 1 - (tid * PER + i)];
        mine += cnt[i];
      }
      int before, none, total, none2;
      scan2<NW>(mine, 0, scratch, before, none, total, none2);
      if (before < want && before + mine >= want) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (before < want && before + cnt[i] >= want) {
            s_bin = kBins - 1 - (tid * PER + i);
            s_want = want - before;
          }
          before += cnt[i];
        }
      }
      __syncthreads();
      top += (uint32_t)s_bin << shift;
      want = s_want;
    }
    if (chunks > 1) load(0);
  }
  // `want`: how many of those equal to T stay
  int sure0 = 0, ties0 = 0;  // of the chunks before
  int first = p.budget;      // the first place of this lane's whose row moves
  for (int c = 0; c < chunks; ++c) {
    if (c > 0) load(c);
    auto kind = [&](int e, bool& sure, bool& tie) {
      const int i = c * CHUNK + e * NT + tid;
      sure = key[e] > top || (key[e] == 0 && i < n);
      tie = key[e] == top;
    };
#pragma unroll
    for (int e = 0; e < E; ++e) {
      bool sure, tie;
      kind(e, sure, tie);
      const int a = __builtin_popcountll(__builtin_amdgcn_ballot_w64(sure)), z = __builtin_popcountll(__builtin_amdgcn_ballot_w64(tie));
      if (lane == 0) {
        counts[e * NW + wv][0] = a;
        counts[e * NW + wv][1] = z;
      }
    }
    __syncthreads();
    int pa, pb, ta, tb;
    const bool in = tid < E * NW;
    scan2<NW>(in ? counts[tid][0] : 0, in ? counts[tid][1] : 0, scratch, pa, pb, ta, tb);
    if (in) {
      counts[tid][0] = sure0 + pa;
      counts[tid][1] = ties0 + pb;
    }
    __syncthreads();  // (and every read of the chunk lies before this)
    sure0 += ta;
    ties0 += tb;
    auto put = [&](auto block_of) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        bool sure, tie;
        kind(e, sure, tie);
        const uint64_t a = __builtin_amdgcn_ballot_w64(sure), z = __builtin_amdgcn_ballot_w64(tie);
        const int before = counts[e * NW + wv][0] +
                           __builtin_amdgcn_mbcnt_hi((uint32_t)(a >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)a, 0));
        const int ties = counts[e * NW + wv][1] +
                         __builtin_amdgcn_mbcnt_hi((uint32_t)(z >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)z, 0));
        if (sure || (tie && ties < want)) {
          const int i = c * CHUNK + e * NT + tid, j = before + min(ties, want);
          w[j] = x[e];
          const int ci = block_of(i), cj = block_of(j), src = from_block[ci];
          int dst = to_block[cj];
          if (!held && into && into[cj] >= 0) dst = into[cj];
          const bool there = src >= 0 && src < p.num_blocks && dst >= 0 && dst < p.num_blocks;
          const int from = there ? src * bs + i - ci * bs : -1, to = there ? dst * bs + j - cj * bs : -1;
          moves[j] = make_int2(from == to ? -1 : from, to);
          if (from != to) first = min(first, j);
        }
      }
    };
    if ((bs & (bs - 1)) == 0) {  // (a division is some twenty instructions)
      const int sh = __builtin_ctz(bs);
      put([&](int i) { return i >> sh; });
    } else {
      put([&](int i) { return i / bs; });
    }
    __syncthreads();
  }
  first = p.budget - wave_max_dpp(p.budget - first);
  if (lane == 0 && first < p.budget) atomicMin(&s_first, first);
  __syncthreads();
  if (tid == 0) moves[p.kept] = make_int2(s_first, 0);
}

// The rows of one (plane, sequence, kv head) moved: units of V, `pieces` a row, from byte `at` of a block on, a slot's
// `slot_run` bytes apart, from place `first` on; idle: a slot of the sequence's. LINEAR: the cache's slots are evenly spaced (no
// scales behind a block's slots); else a place takes a division (30 x 700-1500 tokens of a 4-bit cache: 4.0 TB/s).
template <typename V, bool LINEAR>
__device__ __forceinline__ void move_rows(const EvictArgs& p, const int2* moves, uint8_t* plane, int64_t block_bytes, int64_t at,
                                          int64_t slot_run, int pieces, int idle, int first) {
  const int per = kMoveThreads / pieces;  // rows a step of the workgroup moves
  const int r = (int)threadIdx.x / pieces, piece = (int)threadIdx.x % pieces;
  const bool on = r < per;
  uint8_t* const base = plane + at + piece * (int)sizeof(V);
  auto place = [&](int slot) -> V* {
    if constexpr (LINEAR) return reinterpret_cast<V*>(base + (int64_t)slot * slot_run);
    const int blk = slot / p.block_size;
    return reinterpret_cast<V*>(base + blk * block_bytes + (int64_t)(slot - blk * p.block_size) * slot_run);
  };
  const int left = p.budget, round = per * kMoveRows;
  auto pairs = [&](int j0, int2 (&m)[kMoveRows]) {
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      const int j = first + j0 + u * per + r;
      m[u] = moves[min(j, left - 1)];
      if (!on || j >= left) m[u].x = -1;
    }
  };
  // (rows that stay read the sequence's first slot, a line for them all, and store nothing: loads behind branches would have
  // every wait for an earlier round wait for all)
  auto rows = [&](const int2 (&m)[kMoveRows], V (&v)[kMoveRows]) {
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) v[u] = __builtin_nontemporal_load(place(m[u].x >= 0 ? m[u].x : idle));
  };
  auto write = [&](const int2 (&m)[kMoveRows], V (&v)[kMoveRows]) {
    // every wave's reads of the round before its first write; the next round's, already on their way, lie behind them
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) asm volatile("" : "+v"(v[u]));
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
      if (m[u].x >= 0) __builtin_nontemporal_store(v[u], place(m[u].y));
  };
  int2 ma[kMoveRows], mb[kMoveRows];
  V va[kMoveRows], vb[kMoveRows];
  const int rounds = (left - first + round - 1) / round;
  pairs(0, ma);
  rows(ma, va);
  pairs(round, mb);
  int t = 0;
  for (; t + 2 < rounds; t += 2) {  // two rounds a turn, without copies of the registers
    rows(mb, vb);
    write(ma, va);
    pairs((t + 2) * round, ma);
    rows(ma, va);
    write(mb, vb);
    pairs((t + 3) * round, mb);
  }
  if (t + 1 < rounds) {
    rows(mb, vb);
    write(ma, va);
    write(mb, vb);
  } else {
    write(ma, va);
  }
}

// Workgroup (sequence, plane = layer and K / V, kv head x part): part x of p.parts slices of a row's bytes, or the scales.
__global__ __launch_bounds__(kMoveThreads) void move_kernel(EvictArgs p) {
  const int b = blockIdx.x, plane = blockIdx.y, parts = p.parts + (p.scale_bytes ? 1 : 0);
  const int g = blockIdx.z / parts, x = blockIdx.z % parts;
  const int n = max(0, min(p.context_lens[b], p.max_blocks * p.block_size));
  const int64_t row = p.rows ? (int64_t)p.rows[b] : b;
  if (n <= p.budget || row < 0 || row >= p.row_count) return;
  const int2* moves = p.moves + (((int64_t)(plane >> 1) * p.batch + b) * p.num_heads + g) * (p.kept + 1);
  const int first = moves[p.kept].x;  // (the rows before the first dropped token are where they belong)
  if (first >= p.budget) return;
  const int64_t block_bytes = (int64_t)p.block_size * p.num_heads * (p.head_bytes + p.scale_bytes);
  const int64_t run = (int64_t)p.num_heads * p.head_bytes;
  uint8_t* base = p.kv + (int64_t)plane * p.num_blocks * block_bytes;
  const int blk0 = p.block_tables[(int64_t)b * p.bt_stride], idle = blk0 >= 0 && blk0 < p.num_blocks ? blk0 * p.block_size : 0;
  const int bytes = p.head_bytes / p.parts;
  const int64_t at = (int64_t)g * p.head_bytes + x * bytes;
  if (!p.scale_bytes)
    move_rows<u32x4, true>(p, moves, base, block_bytes, at, run, bytes / 16, idle, first);
  else if (x < p.parts)
    move_rows<u32x4, false>(p, moves, base, block_bytes, at, run, bytes / 16, idle, first);
  else
    move_rows<uint32_t, false>(p, moves, base, block_bytes, (int64_t)p.block_size * run + (int64_t)g * p.scale_bytes,
                               (int64_t)p.num_heads * p.scale_bytes, p.scale_bytes / 4, idle, first);
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a0, hipStream_t stream) {
  EvictArgs a = a0;
  if (a.batch <= 0 || a.layers <= 0 || a.num_heads <= 0) return hipSuccess;
  const dim3 grid((unsigned)a.num_heads, (unsigned)a.batch, (unsigned)a.layers);
  // sequences that the tables let grow past 2048 tokens: 16 waves with 32 weights a lane (32768 tokens)
  if ((int64_t)a.max_blocks * a.block_size <= 2048)
    select_kernel<256, 8><<<grid, dim3(256), 0, stream>>>(a);
  else
    select_kernel<1024, 32><<<grid, dim3(1024), 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // slices of a row of 64 bytes or more, until there are two workgroups a CU
  a.parts = 1;
  while (a.parts < 4 && a.head_bytes % (a.parts * 128) == 0 &&
         (int64_t)a.batch * 2 * a.layers * a.num_heads * a.parts < 512)
    a.parts *= 2;
  move_kernel<<<dim3((unsigned)a.batch, (unsigned)(2 * a.layers), (unsigned)(a.num_heads * (a.parts + (a.scale_bytes ? 1 : 0)))),
                dim3(kMoveThreads), 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace vox
