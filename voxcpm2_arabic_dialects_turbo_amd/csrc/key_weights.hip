// What every key of a causal varlen call receives: for sequence b, kv head g and key j
//   got[g, j] = sum over b's queries i that see j and the query heads h of g of exp2(c q_ih . k_j - lse_ih),
// c the log2-scaled softmax scale, lse_ih = log2 sum_j exp2(c q_ih . k_j): the column sums of the attention's probabilities.
// The attention (prefill_tile32.h) leaves every row's lse behind, and key_weights_kernel makes the scores again: sums down
// the columns inside the attention would be a cross-workgroup sum for every (row tile, key), this one's are registers. It has
// neither atomics nor an order that changes: an item is (128 keys, a part of the query rows, kv head, sequence), one
// workgroup's; key_weights_sum_kernel adds the parts where a sequence has several. fp32 throughout but for the scores' bf16
// inputs. A new key's weight is set, a cached one's grows.
//
// A workgroup is KW x QW = 2 x 2 waves: wave (kw, qw) holds its 64 keys' K rows in registers (the A operand of the score MFMA)
// and takes the 64-row query tiles qw, qw + 2, ... from the first that sees its keys, out of LDS (two buffers, filled by
// loads straight into LDS while the other is read). Rows are (token, query head of g), so S^T[32 keys x 32 rows] has a row's
// scores in one lane column and its lse in one register: fma, exp2, add, beside the next half tile's MFMAs in a fixed order.
// The lanes' sums meet in LDS at the end.
//
// Bound by those fma, exp2 (quarter rate) and adds, about as many cycles as the MFMAs: 6 chunks of 1000-2000 tokens over
// 1500-2500 (16 heads of 2, 107 GFLOP of scores) 143-160 us, beside 223-245 for the attention; small calls by latency
// (44 chunks of 33-59 over 50: 9.8 us).
#include <cfloat>
#include <type_traits>

#include "fp4_common.h"
#include "prefill_tile32.h"
#include "vox_common.h"
#include "vox_kernels.h"

namespace vox {

namespace {

constexpr int kKwD = 128;

// Items numbered sequence by sequence: the first of each of `batch` <= kMaxSeqPerLaunch sequences, with items_of(b) of them,
// into starts[0, batch] (LDS, with wtot[4]) by 256 threads; returns how many there are.
template <typename F>
__device__ __forceinline__ int number_items(int batch, int* starts, int* wtot, F&& items_of) {
  const int tid = threadIdx.x, w = tid >> 6;
  int total = 0;
  for (int base = 0; base < batch; base += 256) {
    const int b = base + tid;
    const int items = b < batch ? items_of(b) : 0;
    const int incl = wave_incl_scan_dpp(items);
    if ((tid & 63) == 63) wtot[w] = incl;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) before += x < w ? wtot[x] : 0;
    if (b < batch) starts[b] = total + before + incl - items;
    total += wtot[0] + wtot[1] + wtot[2] + wtot[3];
    __syncthreads();
  }
  if (tid == 0) starts[batch] = total;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(total);
}
// The sequence of an item: the last that starts at or before it (an empty one shares its start with the next).
__device__ __forceinline__ int sequence_of(int item, int batch, const int* starts) {
  int b = -1;
  for (int c = 0; c < batch; c += kWave) {
    const int lane = threadIdx.x & 63;
    const int at = c + lane < batch ? starts[c + lane] : INT32_MAX;
    b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(at <= item));
  }
  return __builtin_amdgcn_readfirstlane(b);
}

// Heavy q tiles, which see most keys, first: one that starts late is the launch's end. WALK: a workgroup for each of the q tiles
// that there are, sequence by sequence, where the (q tile, sequence) grid would be mostly empty, or so large that its empty
// ones cost more than the items' layout.
template <int SRC, int RG, int KS, bool WALK>
__global__ __launch_bounds__(64 * RG * KS, 2) void prefill32_lse_kernel(PrefillArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t kt0[pf32::kTB];
  __shared__ __attribute__((aligned(1024))) uint8_t kt1[pf32::kTB];
  __shared__ __attribute__((aligned(1024))) uint8_t vt0[pf32::kTB];
  __shared__ __attribute__((aligned(1024))) uint8_t vt1[pf32::kTB];
  __shared__ float red[KS == 2 ? 256 : 1];
  const pf32::Bufs bufs{kt0, kt1, vt0, vt1, red};
  if constexpr (WALK) {
    __shared__ int starts[kMaxSeqPerLaunch + 1];
    __shared__ int wtot[4];
    const int BQ = 32 * RG / p.group, HK = p.num_kv_heads;
    const int total = number_items(p.batch, starts, wtot, [&](int b) {
      const int nq = p.cu_q[b + 1] - p.cu_q[b];
      return nq <= 0 || (p.skip_single && nq == 1) ? 0 : (nq + BQ - 1) / BQ * HK;
    });
    const int item = blockIdx.x;
    if (item >= total) return;
    const int b = sequence_of(item, p.batch, starts);
    const int from = __builtin_amdgcn_readfirstlane(starts[b]), n = __builtin_amdgcn_readfirstlane(starts[b + 1]) - from;
    pf32::tile<SRC, RG, KS, true>(p, (n - 1 - (item - from)) / HK, b, (item - from) % HK, bufs);
  } else {
    pf32::tile<SRC, RG, KS, true>(p, (int)(gridDim.x - 1 - blockIdx.x), (int)blockIdx.y, (int)blockIdx.z, bufs);
  }
}

constexpr int kKwKeys = 128;  // keys of an item (DIRECT grids may halve it)
constexpr int kKwRows = 64;   // query rows of a tile

// A sequence's items: query rows [0, n) in parts of k.part_rows, the cached keys `old` before its own, key blocks.
struct KwSeq {
  int q0, nq, k0, nk, old, n, parts;
  int64_t row;
  // key blocks that see a row of part x: those that start at or before the part's last token
  __device__ __forceinline__ int blocks(const KeyWeightsArgs& k, int x, int gsh) const {
    const int last = (min(n, (x + 1) * k.part_rows) - 1) >> gsh;
    const int64_t end = min((int64_t)min(nk, old + last + 1), k.width);
    return end <= 0 ? 0 : (int)((end + (1 << k.item_shift) - 1) >> k.item_shift);
  }
  // the place of its first part among the partials, where it has several: with r the call's rows before it over part_rows, two
  // sequences' floor(r) are apart by at least the parts of the first less one, so twice that by at least its parts
  __device__ __forceinline__ int64_t first_part(const KeyWeightsArgs& k, int gsh) const {
    return (((int64_t)q0 << gsh) / k.part_rows) * 2;
  }
};
__device__ __forceinline__ KwSeq kw_seq(const KeyWeightsArgs& k, int b, int gsh) {
  const PrefillArgs& p = k.a;
  KwSeq s;
  s.q0 = p.cu_q[b];
  s.nq = p.cu_q[b + 1] - s.q0;
  s.k0 = p.cu_k[b];
  s.nk = p.cu_k[b + 1] - s.k0;
  if (p.block_tables) s.nk = min(s.nk, p.max_blocks * p.block_size);  // (the attention ends, and aligns the queries, there)
  s.old = s.nk - s.nq;
  s.row = k.rows ? (int64_t)k.rows[b] : b + k.row0;
  const bool mine = s.nq > 0 && s.nk > 0 && s.row >= 0 && s.row < k.row_count && !(p.skip_single && s.nq == 1);
  // (the rows that the attention took, and the keys that those may see)
  s.nq = (int)max((int64_t)0, min((int64_t)min(s.nq, k.max_q), p.row_limit - s.q0));
  s.nk = min(min(s.nk, s.old + s.nq), k.max_k);
  s.n = mine ? s.nq << gsh : 0;
  s.parts = (s.n + k.part_rows - 1) / k.part_rows;
  return s;
}

// Persistent: the items (128 keys, a part of the query rows, kv head, sequence), the key blocks of a part side by side, are
// dealt to the XCDs in contiguous ranges, whose workgroups read the part's rows from that XCD's L2. DIRECT, where the grid of
// all there may be is small: a workgroup for each, without the items' layout. FP4: the keys come from a 4-bit cache, as bf16,
// which holds their values exactly; where 32 keys have a scale past which it does not, a quarter of them all, at four times the
// softmax scale.
template <bool DIRECT, int KT, bool FP4>
__global__ __launch_bounds__(256, 2) void key_weights_kernel(KeyWeightsArgs k) {
  constexpr int KW = 2, QW = 2;
  constexpr int KEYS = 32 * KT;               // keys of a wave
  constexpr int TILE = kKwRows * 256;
  constexpr int BUF = QW * TILE + 4 * 256;    // a tile for each query wave, and each wave's copy of its rows' lse
  const PrefillArgs& p = k.a;
  // (distinct arrays, so the compiler can tell a tile's reads from the loads in flight)
  __shared__ __attribute__((aligned(1024))) uint8_t buf0[BUF];
  __shared__ __attribute__((aligned(1024))) uint8_t buf1[BUF];
  __shared__ float sums[4][KEYS];
  __shared__ int starts[DIRECT ? 1 : kMaxSeqPerLaunch + 1];
  __shared__ int wtot[DIRECT ? 1 : 4];
  typedef __attribute__((address_space(3))) void lds_void;
  using std::integral_constant;
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = w % KW, qw = w / KW;
  const int lane = tid & 63, col = lane & 31, h = lane >> 5, lr = lane >> 4;
  const int gsh = __builtin_ctz(p.group), HK = p.num_kv_heads;
  const bool paged = p.block_tables != nullptr;
  const uint32_t qs = (uint32_t)p.q_row_stride * 2u;
  const uint32_t lane_off = (uint32_t)(lr >> gsh) * qs + (uint32_t)((lr & (p.group - 1)) << 8);
  const uint32_t lane_sw = (uint32_t)(((lane & 15) ^ lr) << 4);

  // k-step i of a query fragment (row col of a half, chunk 2 i + h) and the row's lse, in a buffer
  uint32_t frag[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) frag[i] = (uint32_t)(qw * TILE + col * 256 + (((2 * i + h) ^ (col & 15)) << 4));
  const uint32_t lse_at = (uint32_t)(QW * TILE + w * 256 + col * 4);

  // ---- every sequence's first item, and this workgroup's items
  int item = (int)blockIdx.x, step = 1, hi = item + 1;
  if constexpr (!DIRECT) {
    const int total = number_items(p.batch, starts, wtot, [&](int b) {
      const KwSeq s = kw_seq(k, b, gsh);
      int items = 0;
      for (int x = 0; x < s.parts; ++x) items += s.blocks(k, x, gsh);
      return items * HK;
    });
    const int xcd = blockIdx.x % kXcds;
    step = gridDim.x / kXcds;  // (the grid is a multiple of the XCDs)
    item = (int)((int64_t)total * xcd / kXcds) + (int)(blockIdx.x / kXcds);
    hi = (int)((int64_t)total * (xcd + 1) / kXcds);
  }

  for (; item < hi; item += step) {
    // ---- the item's sequence, part, kv head and key block
    int b, x, g, first;
    KwSeq s;
    if constexpr (DIRECT) {
      const int blocks = (k.max_k + KW * KEYS - 1) / (KW * KEYS);
      first = item % blocks * (KW * KEYS);
      x = item / blocks % k.max_parts;
      g = item / blocks / k.max_parts % HK;
      b = item / blocks / k.max_parts / HK;
      s = kw_seq(k, b, gsh);
      if (x >= s.parts || first >= s.blocks(k, x, gsh) * (KW * KEYS)) return;
    } else {
      b = sequence_of(item, p.batch, starts);
      s = kw_seq(k, b, gsh);
      int left = item - starts[b], blocks = s.blocks(k, 0, gsh);
      x = 0;
      while (left >= blocks * HK) {
        left -= blocks * HK;
        blocks = s.blocks(k, ++x, gsh);
      }
      left = __builtin_amdgcn_readfirstlane(left);
      x = __builtin_amdgcn_readfirstlane(x);
      blocks = __builtin_amdgcn_readfirstlane(blocks);
      g = left / blocks;
      first = left % blocks * (KW * KEYS);
    }

    const int jb = first + kw * KEYS;  // this wave's first key
    u32x4 kf[KT][8];
    uint64_t counts = 0;  // bit: key jb + bit takes weight
    // ---- the part's rows that see a key of the item: token tq sees key j when j <= old + tq. Query wave qw takes tiles qw,
    // qw + QW, ... from row `begin` on; a tile is two halves of 32 rows.
    const int end = min(s.n, (x + 1) * k.part_rows);
    const int begin = max(x * k.part_rows, (max(0, first - s.old) << gsh) & ~31);
    const int rounds = (end - begin + kKwRows * QW - 1) / (kKwRows * QW);
    const uint16_t* const qb = p.q + (int64_t)s.q0 * p.q_row_stride + (g << gsh) * kKwD;
    const float* const lb = p.lse + (int64_t)s.q0 * p.num_heads + (g << gsh);
    auto buffer = [&](auto buf) -> uint8_t* { return decltype(buf)::value & 1 ? buf1 : buf0; };
    auto row0 = [&](int t) { return begin + (t * QW + qw) * kKwRows; };
    // Tile t into its buffer (t % 2): rows past the sequence's last read as zeros. A piece is four rows, which start at a
    // multiple of four: its lanes' offsets are the same up to a uniform one, and the chunks' order (as prefill_tile32.h's).
    const int r0 = row0(0) & (p.group - 1);  // every tile starts at this head of its first token
    auto load = [&](int t, auto buf) {
      const int tok0 = row0(t) >> gsh;
      const uint32_t toks = (uint32_t)__builtin_amdgcn_readfirstlane(max(0, min(s.nq - tok0, kKwRows + 1)));
      uint8_t* const to = buffer(buf) + qw * TILE;
      const auto rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(qb + (int64_t)tok0 * p.q_row_stride), (short)0,
                                                        toks * qs, 0x00020000);
      uint32_t at = lane_off, sw = lane_sw;
      asm volatile("" : "+v"(at), "+v"(sw));  // (the pieces' offsets made here, not held in registers over the loop)
#pragma unroll
      for (int i = 0; i < kKwRows / 4 / KW; ++i) {
        const int rr = kw * (kKwRows / KW) + 4 * i, rho = r0 + rr;
        const uint32_t piece = (uint32_t)(rho >> gsh) * qs + (uint32_t)((rho & (p.group - 1)) << 8);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (lds_void*)(to + rr * 256), 16, piece + at + (sw ^ (uint32_t)((i & 3) << 6)),
                                                 0, 0, 0);
      }
      const auto rl = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(lb + (int64_t)tok0 * p.num_heads), (short)0,
                                                        toks * (uint32_t)p.num_heads * 4u, 0x00020000);
      const int rho = r0 + lane;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rl, (lds_void*)(buffer(buf) + QW * TILE + w * 256), 4,
          ((uint32_t)(rho >> gsh) * (uint32_t)p.num_heads + (uint32_t)(rho & (p.group - 1))) * 4u, 0, 0, 0);
    };
    auto arrive = [&]() {  // the tile on its way is there, and every wave has read the one before it
      wait_vmem_all();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    float c[KT];  // (wave-uniform)
    float acc[KT][16];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      c[kt] = p.scale_log2;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[kt][i] = 0.f;
    }
    constexpr int NM = 8 * KT, NE = 16 * KT;
    // the scores (into sn) of half `hn` of the tile in buffer `buf` beside the probabilities of the half before it, whose first
    // row is r0
    auto step = [&](auto masked, auto buf, auto hn, int r0, const f32x16 (&sc)[KT], f32x16 (&sn)[KT], float lse, float& lse_n) {
      constexpr bool MASK = decltype(masked)::value;
      constexpr int HN = decltype(hn)::value;
      const uint8_t* tile = buffer(buf) + HN * 32 * 256;
      u32x4 qf[4];  // (read four k-steps ahead)
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[i] = *reinterpret_cast<const u32x4*>(tile + frag[i]);
      lse_n = *reinterpret_cast<const float*>(buffer(buf) + lse_at + HN * 128);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sn[kt][i] = 0.f;
      // register i: key jb + 32 kt + 8 (i / 4) + 4 h + i % 4; the last key that the row sees, relative to jb + 4 h
      const int rho = r0 + col;
      const int last = rho < end ? s.old + (rho >> gsh) - jb - 4 * h : -1;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        sn[i % KT] = mfma_32x32x16(kf[i % KT][i / KT], qf[i / KT % 4], sn[i % KT]);
        if (i % KT == KT - 1 && i / KT + 4 < 8)
          qf[i / KT % 4] = *reinterpret_cast<const u32x4*>(tile + frag[i / KT + 4]);
#pragma unroll
        for (int y = i * NE / NM; y < (i + 1) * NE / NM; ++y) {
          const int kt = y >> 4, e = y & 15;
          const float pr = fast_exp2(fmaf(sc[kt][e], c[kt], -lse));
          acc[kt][e] += !MASK || 32 * kt + 8 * (e >> 2) + (e & 3) <= last ? pr : 0.f;
          asm volatile("" : "+v"(acc[kt][e]));  // (here: sunk behind the two forms of the step, the adds ran beside no MFMA)
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // step, masked where a row of the half before does not exist or does not see every key of the wave
    auto half = [&](auto buf, auto hn, int r0, const f32x16 (&sc)[KT], f32x16 (&sn)[KT], float lse, float& lse_n) {
      if (r0 + 32 <= end && s.old + (r0 >> gsh) >= jb + KEYS - 1)
        step(std::false_type{}, buf, hn, r0, sc, sn, lse, lse_n);
      else
        step(std::true_type{}, buf, hn, r0, sc, sn, lse, lse_n);
    };
    using C0 = integral_constant<int, 0>;
    using C1 = integral_constant<int, 1>;
    f32x16 sa[KT], sb[KT];
    float la, lx = 0.f;
    load(0, C0{});

    // ---- this wave's keys: key j = jb + 32 kt + col, dims 16 s + 8 h + [0, 8) in kf[kt][s]; keys that do not count are zeros
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int j = jb + 32 * kt + col;
      bool ok = j < s.nk;
      const uint16_t* kr = nullptr;
      const uint8_t *block = nullptr, *code = nullptr;
      int in = 0;
      if (!paged) {
        kr = p.k_src + ((int64_t)s.k0 + (ok ? j : 0)) * p.k_row_stride + g * kKwD;
      } else {
        ok = ok && j < p.max_blocks * p.block_size;
        const int bid = p.block_tables[(int64_t)b * p.bt_stride + (ok ? j / p.block_size : 0)];
        ok = ok && bid >= 0 && bid < p.num_blocks;
        if constexpr (FP4) {
          in = j % p.block_size;
          block = reinterpret_cast<const uint8_t*>(p.k_cache) + (ok ? bid : 0) * fp4::block_bytes(p.block_size, HK);
          code = block + (int64_t)(in * HK + g) * fp4::kHeadCodes;
        } else {
          kr = p.k_cache + (((int64_t)(ok ? bid : 0) * p.block_size + j % p.block_size) * HK + g) * kKwD;
        }
      }
      counts |= (uint64_t)(uint32_t)__builtin_amdgcn_ballot_w64(ok) << (32 * kt);
      if constexpr (FP4) {  // chunk i's 4 bytes: word 2 (i % 2) + h of the 32 channels i / 2
        u32x4 codes[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[i] = *reinterpret_cast<const u32x4*>(code + 16 * i);
        const uint32_t scale = *reinterpret_cast<const uint32_t*>(block + (int64_t)p.block_size * HK * fp4::kHeadCodes +
                                                                  (in * HK + g) * fp4::kHeadScales);
        auto convert = [&](auto&& values) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const u32x4 c4 = codes[i / 2];
            const u32x4 v = values(h ? c4[2 * (i & 1) + 1] : c4[2 * (i & 1)], (scale >> (8 * (i / 2))) & 0xffu);
            kf[kt][i] = ok ? v : zero4();
          }
        };
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(ok && fp4::past_bf16(scale)) != 0, 0)) {
          convert([](uint32_t codes8, uint32_t b) { return fp4::quarter_values8(codes8, b); });
          c[kt] = fminf(4.f * p.scale_log2, FLT_MAX);  // (an infinity would make NaN of a score of 0)
        } else {
          convert([](uint32_t codes8, uint32_t b) { return fp4::values8(codes8, fp4::scale_float(b)); });
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const u32x4 v = ld_g16(kr + 16 * i + 8 * h);
          kf[kt][i] = ok ? v : zero4();
        }
      }
    }
    arrive();
    load(1, C1{});
    {
      la = *reinterpret_cast<const float*>(buf0 + lse_at);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sa[kt][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const u32x4 qf = *reinterpret_cast<const u32x4*>(buf0 + frag[i]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) sa[kt] = mfma_32x32x16(kf[kt][i], qf, sa[kt]);
      }
    }
    // tile t: the scores of its second half, then those of the next tile's first, each beside the probabilities before them;
    // the tile after next is loaded from where tile t is read, over the second of the two and the next tile's first
    auto tile = [&](auto buf, auto other, int t) {
      half(buf, C1{}, row0(t), sa, sb, la, lx);
      arrive();
      load(t + 2, buf);
      half(other, C0{}, row0(t) + 32, sb, sa, lx, la);
    };
    for (int t = 0;;) {
      tile(C0{}, C1{}, t);
      if (++t >= rounds) break;
      tile(C1{}, C0{}, t);
      if (++t >= rounds) break;
    }

    // ---- over the rows' lane columns (the 32 lanes of a half) and the query waves
    int lc = col;
    asm volatile("" : "+v"(lc));  // (sixteen comparisons made here, not held in scalar registers over the loop)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = acc[kt][i];
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));  // row_ror:8, 4, 2, 1
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xF, 0xF, false));
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xF, 0xF, false));
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xF, 0xF, false));
        v = xrow_sum(v);
        mine = lc == i ? v : mine;
      }
      if (lc < 16) sums[w][32 * kt + 8 * (col >> 2) + 4 * h + (col & 3)] = mine;
    }
    wait_vmem_all();  // (tiles behind the last one)
    __syncthreads();
    const int j = jb + lane;
    if (qw == 0 && lane < KEYS && j < s.nk && j < k.width) {
      float got = sums[kw][lane] + sums[kw + KW][lane];
      got = (counts >> lane) & 1u ? got : 0.f;
      if (s.parts > 1) {
        k.partials[((s.first_part(k, gsh) + x) * HK + g) * k.max_k + j] = got;
      } else {
        float* out = k.weights + (s.row * HK + g) * k.width + j;
        *out = j >= s.old ? got : *out + got;
      }
    }
    __syncthreads();  // (sums and tiles are free)
  }
}

// The weights of the sequences in several parts: the sum of those whose rows see the key, in order.
__global__ __launch_bounds__(256) void key_weights_sum_kernel(KeyWeightsArgs k) {
  const int b = blockIdx.y, g = blockIdx.z, j = (int)(blockIdx.x * 256 + threadIdx.x);
  const int gsh = __builtin_ctz(k.a.group);
  const KwSeq s = kw_seq(k, b, gsh);
  if (s.parts <= 1 || j >= s.nk || j >= k.width) return;
  const int64_t apart = (int64_t)k.a.num_kv_heads * k.max_k;
  const float* part = k.partials + s.first_part(k, gsh) * apart + (int64_t)g * k.max_k + j;
  // the first part with a row that sees the key's block
  const int from = (int)(((int64_t)max(0, (j >> k.item_shift << k.item_shift) - s.old) << gsh) / k.part_rows);
  float got = 0.f;
  for (int x = from; x < s.parts; x += 8) {  // (eight loads in flight)
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = part[min(x + i, s.parts - 1) * apart];
#pragma unroll
    for (int i = 0; i < 8; ++i) got += x + i < s.parts ? v[i] : 0.f;
  }
  float* out = k.weights + (s.row * k.a.num_kv_heads + g) * k.width + j;
  *out = j >= s.old ? got : *out + got;
}

// A step with fewer queries than new tokens (a layer that takes the last row of each sequence): the sums above and the decode
// kernels set the queries' own places and add to all before them, so the others of the step start at 0 here. A launch of its
// own ahead of them, for those layers alone; bound by its start (44 sequences of 83-109 tokens 2.7 us).
__global__ __launch_bounds__(256) void clear_new_weights_kernel(ClearWeightsArgs a) {
  const int b = blockIdx.y, g = blockIdx.z;
  const int64_t row = a.rows ? (int64_t)a.rows[b] : b;
  const int64_t nk = min((int64_t)a.cu_k[b + 1] - a.cu_k[b], (int64_t)a.max_keys);
  const int64_t fresh = (int64_t)a.cu_new[b + 1] - a.cu_new[b];
  if (row < 0 || row >= a.row_count) return;
  const int64_t to = min(min(nk, (int64_t)a.max_tokens), a.width);
  float* const w = a.weights + (row * a.num_heads + g) * a.width;
  for (int64_t j = max((int64_t)0, nk - max((int64_t)0, fresh)) + blockIdx.x * 256 + threadIdx.x; j < to; j += (int64_t)gridDim.x * 256)
    w[j] = 0.f;
}

template <bool DIRECT, int KT>
void launch_sums(const KeyWeightsArgs& k, int64_t grid, hipStream_t stream) {
  if (k.fp4)
    key_weights_kernel<DIRECT, KT, true><<<dim3((unsigned)grid), dim3(256), 0, stream>>>(k);
  else
    key_weights_kernel<DIRECT, KT, false><<<dim3((unsigned)grid), dim3(256), 0, stream>>>(k);
}

template <int RG, int KS, bool WALK>
hipError_t launch_lse(const PrefillArgs& a, dim3 grid, hipStream_t stream) {
  const dim3 block(64 * RG * KS);
  if (!a.block_tables)
    prefill32_lse_kernel<pf32::kRows, RG, KS, WALK><<<grid, block, 0, stream>>>(a);
  else
    prefill32_lse_kernel<pf32::kCache, RG, KS, WALK><<<grid, block, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_prefill_lse(const PrefillArgs& a0, int max_seqlen_q, hipStream_t stream) {
  if (max_seqlen_q <= 0 || a0.batch <= 0) return hipSuccess;
  if (!a0.lse || !a0.cu_q || !a0.cu_k || !a0.causal || (a0.block_tables && a0.block_size % pf32::kBK) || 128 % a0.group)
    return hipErrorInvalidValue;
  PrefillArgs a = a0;
  const int64_t tiles = ((int64_t)max_seqlen_q + 128 / a.group - 1) / (128 / a.group);
  const int64_t grid = tiles * a.batch * a.num_kv_heads;
  // WALK (6 x 1000-2000 over 1500-2500: 245 us, the plain grid heavy tiles first 248, in XCD order 255; 44 x 33-59 over 50 13.2
  // against the plain grid's 12.3, 5 x 237-900 27.2 against 25.1)
  if (grid >= 1024 || 4 * a.row_limit <= (int64_t)max_seqlen_q * a.batch) {
    for (int b0 = 0; b0 < a0.batch; b0 += kMaxSeqPerLaunch) {
      a.batch = a0.batch - b0 < kMaxSeqPerLaunch ? a0.batch - b0 : kMaxSeqPerLaunch;
      a.cu_q = a0.cu_q + b0;
      a.cu_k = a0.cu_k + b0;
      if (a.block_tables) a.block_tables = a0.block_tables + (int64_t)b0 * a0.bt_stride;
      // no more tiles than fit the call's rows, and one more a sequence
      const int64_t items = (a.row_limit * a.group / 128 + a.batch) * a.num_kv_heads;
      if (items > INT32_MAX) return hipErrorInvalidValue;
      const hipError_t e = launch_lse<4, 1, true>(a, dim3((unsigned)items), stream);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  // 64 rows a workgroup, two waves on the same ones: halves the chain of key tiles. Two workgroups a CU at once, or two rounds of
  // them where the chains are long (1 x 3000 tokens: 50 us, in 128 rows 59; 44 x 33-59 over 50 15.3 and 12.4). Counted as the call
  // says it, sequences shorter than max_seqlen_q at their full length.
  const bool fits64 = 64 % a.group == 0;
  const int64_t tiles64 = fits64 ? ((int64_t)max_seqlen_q + 64 / a.group - 1) / (64 / a.group) : 0;
  const int64_t grid64 = tiles64 * a.batch * a.num_kv_heads;
  if (fits64 && (grid64 <= 512 || (grid64 <= 1024 && tiles64 >= 16)))
    return launch_lse<2, 2, false>(a, dim3((unsigned)tiles64, (unsigned)a.batch, (unsigned)a.num_kv_heads), stream);
  return launch_lse<4, 1, false>(a, dim3((unsigned)tiles, (unsigned)a.batch, (unsigned)a.num_kv_heads), stream);
}

hipError_t launch_clear_new_weights(const ClearWeightsArgs& a, hipStream_t stream) {
  if (a.batch <= 0 || a.max_tokens <= 0 || a.num_heads <= 0) return hipSuccess;
  const int64_t wgs = ((int64_t)a.max_tokens + 1023) / 1024;
  clear_new_weights_kernel<<<dim3((unsigned)(wgs < 64 ? wgs : 64), (unsigned)a.batch, (unsigned)a.num_heads), dim3(256), 0, stream>>>(a);
  return hipGetLastError();
}

int key_weights_part_rows(int64_t num_tokens, int max_seqlen_q, int max_seqlen_k, int group, int num_kv_heads) {
  // About three items for each workgroup slot (two a CU), of 256 to 4096 rows, and 16 parts at most; one part of up to 640
  // rows, where a second launch costs what it saves. us (with whole key blocks), in parts of 512 rows and eight at most,
  // against this (max_seqlen_k counts a mixed step's decode rows too): prompts of 64 tokens 11.0 (in parts of 256 9.0 + 2.6 and a launch's gap), 100 11.5 + 3.9 and 9.5 + 3.3,
  // 237 12.2 + 3.8 and 9.7 + 3.9, 1000 18.6 + 4.2 and 12.9 + 4.0.
  const int64_t blocks = ((int64_t)max_seqlen_k + kKwKeys - 1) / kKwKeys;
  const int64_t longest = (int64_t)max_seqlen_q * group, least = (longest + 15) / 16;
  const int64_t want = num_tokens * group * num_kv_heads * blocks / 1536;
  int64_t r = want < 256 ? 256 : want > 4096 ? 4096 : want;
  r = r > least ? r : least;
  if (longest <= 640 && r < longest) r = longest;
  r = (r + 127) / 128 * 128;
  return r > INT32_MAX / 2 ? INT32_MAX / 2 / 128 * 128 : (int)r;
}

hipError_t launch_key_weights(const KeyWeightsArgs& k0, hipStream_t stream) {
  KeyWeightsArgs k = k0;
  if (k.max_k <= 0 || k.a.batch <= 0) return hipSuccess;
  if (!k.a.lse || !k.weights || !k.a.cu_q || !k.a.cu_k || k.a.row_limit <= 0 || k.max_q <= 0 || k.part_rows <= 0 || k.part_rows % 128 ||
      (k.max_parts > 1 && !k.partials) || (k.fp4 && !k.a.block_tables))
    return hipErrorInvalidValue;
  const int batch = k0.a.batch;
  for (int b0 = 0; b0 < batch; b0 += kMaxSeqPerLaunch) {  // (the sequences' items are laid out in LDS)
    k.a.batch = batch - b0 < kMaxSeqPerLaunch ? batch - b0 : kMaxSeqPerLaunch;
    k.a.cu_q = k0.a.cu_q + b0;
    k.a.cu_k = k0.a.cu_k + b0;
    if (k.a.block_tables) k.a.block_tables = k0.a.block_tables + (int64_t)b0 * k0.a.bt_stride;
    if (k.rows)
      k.rows = k0.rows + b0;
    else
      k.row0 = k0.row0 + b0;
    const int64_t blocks = ((int64_t)k.max_k + kKwKeys - 1) / kKwKeys;
    int64_t items = blocks * k.max_parts * k.a.batch * k.a.num_kv_heads;
    // Grids of at most a workgroup a CU, which the exponentials of their own rows bound: half the keys each (us, whole and
    // half key blocks: a prompt of 30 tokens 8.6 and 6.8, 64 11.0 and 8.6, 237 9.7 and 7.4, 44 of 33-59 over 50 13.2 and
    // 9.8; past it 5 of 237-900 19.2 and 24.6, 4 of 300 over 700 21.4 and 22.8).
    k.item_shift = items <= 256 ? 6 : 7;
    if (items <= 256) {
      items = ((int64_t)k.max_k + 63) / 64 * k.max_parts * k.a.batch * k.a.num_kv_heads;
      launch_sums<true, 1>(k, items, stream);
    } else if (items <= 1536) {  // (5 prompts of 237-900 tokens, 1200 of them: 23.2 -> 19.2 us)
      launch_sums<true, 2>(k, items, stream);
    } else {  // two workgroups a CU
      launch_sums<false, 2>(k, 512, stream);
    }
    if (k.max_parts > 1)
      key_weights_sum_kernel<<<dim3((unsigned)((k.max_k + 255) / 256), (unsigned)k.a.batch, (unsigned)k.a.num_kv_heads),
                               dim3(256), 0, stream>>>(k);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace vox
