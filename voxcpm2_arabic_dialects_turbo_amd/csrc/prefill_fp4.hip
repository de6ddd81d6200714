// Varlen attention over a 4-bit KV cache through block tables: prompts that go on from cached prefixes, and steps that
// mix prompts with decode rows. Semantics as prefill_attn.hip's paged form: query i of a sequence with nq queries and nk
// keys sees keys j <= nk - nq + i (causal) or all nk; a row that sees no key gives zeros; keys of blocks outside the
// cache have no weight. The format is in fp4_common.h.
//
// A workgroup is four waves over 128 / KS query rows (as many / G tokens x the G query heads of one kv head), and walks
// 64-key tiles (a tile lies inside one block: block_size is a multiple of 64). With KS = 1 a wave has 32 of the rows and
// every key; with KS = 2 two waves share 32 rows, each with half of every tile, and merge (O, m, l) at the end: half the
// work a wave and tile, for grids so short that the chain of tiles is what takes the time (launch_prefill_fp4).
//  * S^T[64 keys x 32 rows] = K Q^T by 32x32x64 MFMAs on the codes as they are stored: a lane's 16 bytes are its
//    operand and have one scale, so K needs no conversion. The query is two fp8 parts, so the scores cost the MFMA time of
//    bf16 ones.
//  * V is converted once a workgroup (a thread 32 channels of a key: 16 exact conversions) into a bf16 LDS tile, double
//    buffered, one barrier a tile. Column w * 4 + c of a row (16 bytes) holds piece w of the key's 32-channel group c, so
//    that the four lanes of a key write consecutive columns.
//  * O^T[128 x 32 rows] += V^T P^T by 32x32x16 MFMAs: P^T is in the B layout as the scores come, k-slot e of half h of
//    step s being key 16 s + 8 (e / 4) + 4 h + e % 4, and the transposed reads gather the same keys.
// A tile's codes (8.5 KB, K and V) go from memory straight into LDS, a quarter by each wave. A tile's softmax and P V run
// beside the next tile's scores and V conversion (step), while the codes of the tile after that are on their way (three
// tiles ahead gave nothing). Probabilities are rounded to bf16 for the MFMA (off by at most 2^-8 of each, as the output
// is); scores, maxima, sums and O are fp32.
// A tile's time is its instructions: about 1.1 us for a wave alone on its SIMD with KS = 1, 0.87 with KS = 2, so short
// prompts are bound by the chain of their tiles (44 x 33-59 tokens over 50 cached: 12.4 us), long ones by MFMA and VALU
// issue: 16 query heads of 2 kv heads, 6 x 1000-2000 over 1500-2500 cached (0.214 PFLOP) 211-223 us, 0.96-1.02 PFLOP/s, where a
// large bf16 product reaches 1.37; 1134 workgroups are 2.2 rounds of 512, whose last costs about a tenth.
#include <algorithm>
#include <climits>

#include "decode_fp4.h"
#include "vox_kernels.h"

namespace vox {

namespace {

namespace pf4 {

constexpr int kD = 128;
constexpr int kBK = 64;         // keys of a tile
constexpr int kHalfChip = 128;  // half the compute units
constexpr int kVRow = kD + 16;  // elements of an LDS row: the four rows a transposed read touches lie in other banks

// A tile's codes as they come from memory: 64 keys x 64 bytes, then the keys' four scales. Of K's 16-byte pieces piece p of
// key r lies in slot p ^ (r / 4 % 4): the eight lanes that an operand read serves at once then hit distinct banks.
constexpr int kCodes = kBK * fp4::kHeadCodes;
constexpr int kTileBytes = kCodes + kBK * fp4::kHeadScales;
typedef __attribute__((address_space(3))) void lds_void;
// Read by scalar loads: as vector loads, behind the transfers into LDS, they could only be waited for with those.
typedef const __attribute__((address_space(4))) int32_t* const_i32;
typedef u32x4 __attribute__((aligned(8))) u32x4_a8;  // output rows are 8-byte aligned

// A workgroup's LDS. s_t0 and s_t1 hold the codes of a tile each, K's, then V's (distinct arrays: the compiler can tell a
// tile's reads from the next one's transfers in flight).
struct Lds {
  uint16_t* v;    // [2][kBK * kVRow]
  uint8_t *t0, *t1;  // [2 * kTileBytes]
  uint8_t* nan;   // [2][key][group]: a tile's scales that are not numbers
  int* nan_at;    // [2]: the first key of the last tile that held any
};

// Query tile qt of sequence b and kv head g. LSE: every row's log2 of the sum its output is divided by goes to p.lse.
template <int KS, bool LSE = false>
__device__ __forceinline__ void prefill_item(const PrefillArgs& p, int b, int g, int qt, const Lds& L) {
  uint8_t* const s_t0 = L.t0;
  uint8_t* const s_t1 = L.t1;
  int* const s_nan_at = L.nan_at;
  // Scalar loads, all at once: the bounds and the first block, which every table row has (left to the compiler, each stands
  // behind the branch before its use: a round trip each)
  const const_i32 bt = (const_i32)(p.block_tables + (int64_t)b * p.bt_stride);
  const const_i32 cu_q = (const_i32)(p.cu_q + b), cu_k = (const_i32)(p.cu_k + b);
  const int q0 = cu_q[0], q1 = cu_q[1], k0 = cu_k[0], k1 = cu_k[1], blk0 = bt[0];
  asm volatile("" ::"s"(q0), "s"(q1), "s"(k0), "s"(k1), "s"(blk0), "s"(p.skip_single), "s"(p.max_blocks), "s"(p.block_size),
               "s"(p.num_blocks), "s"(p.row_limit), "s"(p.q), "s"(p.k_cache), "s"(p.v_cache));
  const int nq = q1 - q0;
  const int HK = p.num_kv_heads;
  const int gsh = __builtin_ctz(p.group);  // the group divides 128: a power of two
  constexpr int ROWS = 128 / KS;           // query rows of the workgroup
  constexpr int KT = 2 / KS;               // 32-key blocks of a tile that a wave takes
  const int bq = ROWS >> gsh;              // query tokens of the workgroup
  if (qt * bq >= nq || (p.skip_single && nq == 1)) return;  // (workgroup-uniform)
  const int nk = max(0, min(k1 - k0, p.max_blocks * p.block_size));

  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 31;
  const int h = lane >> 5;
  const int rg = KS == 1 ? w : w & 1;      // rows 32 rg + [0, 32)
  const int kh = KS == 1 ? 0 : w >> 1;     // keys 32 kh + [0, 32 KT) of every tile
  const int rho = rg * 32 + col;
  const int tq = qt * bq + (rho >> gsh);
  const int head = (g << gsh) + (rho & (p.group - 1));
  const int64_t row = (int64_t)q0 + tq;
  const int tq_last = min(nq, (qt + 1) * bq) - 1;
  const int kv_end = p.causal ? min(nk, nk - nq + tq_last + 1) : nk;  // keys that some row of the workgroup sees
  const int limit = p.causal ? min(nk, nk - nq + tq + 1) : nk;        // keys that this lane's row sees
  const int all_see = p.causal ? nk - nq + qt * bq + 1 : nk;          // keys that every row sees

  const int64_t bb = fp4::block_bytes(p.block_size, HK);
  const int crow = HK * fp4::kHeadCodes, srow = HK * fp4::kHeadScales;
  const int scales = p.block_size * crow;
  // The next tile's codes from memory into LDS at d, a quarter of them by each wave; whether its block is
  // mapped.
  const int key16 = tid >> 2;  // the key of the 16-byte slot that this lane fills
  const int kcode = key16 * crow + (((tid & 3) ^ ((key16 >> 2) & 3)) << 4), vcode = key16 * crow + ((tid & 3) << 4);
  const int word = lane * srow;
  // the next tile: its first key, block (read a tile ahead) and place in the block
  int next_kv = 0, next_col = 0, next_in = 0, next_blk = kv_end > 0 ? blk0 : -1;
  auto issue = [&](uint8_t* d) -> bool {
    const int blk = __builtin_amdgcn_readfirstlane(next_blk);
    const bool ok = blk >= 0 && blk < p.num_blocks;
    const int tok = next_in;
    const int64_t at = ok ? blk * bb : 0;
    const int range = ok ? (int)bb : 0;
    const auto rk = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.k_cache) + at, (short)0, range,
                                                      fp4::kBufferWord3);
    const auto rv = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.v_cache) + at, (short)0, range,
                                                      fp4::kBufferWord3);
    const int c0 = tok * crow + g * fp4::kHeadCodes, s0 = scales + tok * srow + g * fp4::kHeadScales;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(d + w * 1024), 16, kcode, c0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(d + kTileBytes + w * 1024), 16, vcode, c0, 0, 0);
    // (the scales by two waves each: the same words)
    if (w & 1)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(d + kTileBytes + kCodes), 4, word, s0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(d + kCodes), 4, word, s0, 0, 0);
    next_kv += kBK;
    next_in += kBK;
    if (next_in == p.block_size) {
      next_in = 0;
      ++next_col;
    }
    next_blk = next_kv < kv_end ? bt[next_col] : -1;
    return ok;
  };

  // ---- the query's loads, then the first tiles': one round trip for both
  u32x4 qv[8];
  {
    // (a row that is none reads the nearest one that q holds: its loads need no branches, its output is not written)
    const int64_t qrow = max((int64_t)0, min(row, p.row_limit - 1));
    const uint16_t* qb = p.q + qrow * p.q_row_stride + (int64_t)head * kD + h * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) qv[i] = ld_g16(qb + (i >> 1) * 32 + (i & 1) * 8);
  }
  bool ok0 = issue(s_t0);

  // ---- the query in fp8 (fp4_common.h): operand ks holds channels 64 ks + 16 h + [0, 16) and 64 ks + 32 + 16 h + [0, 16)
  fp4::i32x8 qhi[2], qlo[2];
  uint32_t qs;
  {
    uint32_t mb = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mb = max(mb, fp4::max_bits(qv[i]));
    mb = __float_as_uint(xhalf_max(__uint_as_float(mb << 16))) >> 16;
    qs = fp4::query_scale_byte(mb);
    const float scale = fp4::scale_float(qs), inv = fp4::query_inverse(qs);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t* x = reinterpret_cast<const uint32_t*>(&qv[ks * 4 + i / 2]) + (i & 1) * 2;
        int hi, lo;
        fp4::query_parts4(x[0], x[1], scale, inv, hi, lo);
        qhi[ks][i] = hi;
        qlo[ks][i] = lo;
      }
  }

  float m = -INFINITY, lsum = 0.f;
  f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
  const float c = p.scale_log2;
  // this thread's V store and this lane's transposed reads: key rows 4 h + (l % 16) / 4, column 16 (l / 16 % 2) + 4 (l % 4)
  const int vst = (tid >> 2) * kVRow + (tid & 3) * 8;
  const int vtr = (4 * h + ((lane & 15) >> 2)) * kVRow + ((lane >> 4) & 1) * 16 + 4 * (lane & 3);

  // V of tile kv0 (its codes at d, `mapped`) into LDS buffer buf: the scale, then piece q4. Values that are not numbers (or past
  // bf16: held_scale) stay out of the MFMAs, where a masked key's probability of 0 would not hide them: such a group is zeros in
  // LDS, and mark_nan finds the rows that see it (their outputs in the group are NaN).
  u32x4 vcodes;
  float vscale = 0.f;
  auto scale_v = [&](const uint8_t* d, int kv0, bool mapped, int buf) {
    vcodes = *reinterpret_cast<const u32x4*>(d + kTileBytes + tid * 16);
    uint32_t b = mapped && kv0 + (tid >> 2) < nk ? (uint32_t)d[kTileBytes + kCodes + tid] : 0u;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(b >= 253u) != 0, 0)) {
      b = fp4::held_scale(b, vcodes);
      if (__builtin_amdgcn_ballot_w64(b == 255u) != 0) s_nan_at[buf] = kv0;
    }
    const bool nan = b == 255u;
    L.nan[buf * (kBK * 4) + tid] = nan;
    vscale = fp4::scale_float(nan ? 0u : b);
  };
  auto piece_v = [&](int q4, int buf) {
    *reinterpret_cast<u32x4*>(L.v + buf * (kBK * kVRow) + vst + q4 * 32) = fp4::values8(vcodes[q4], vscale);
  };
  uint32_t nan_groups = 0;  // byte c, bit 0: the row has seen such a key in group c
  auto mark_nan = [&](int buf, int seen) {  // seen: the tile's keys that this lane's row sees
#pragma unroll 1
    for (int j = 0; j < kBK; ++j) nan_groups |= j < seen ? reinterpret_cast<const uint32_t*>(L.nan + buf * (kBK * 4))[j] : 0u;
  };
  // Score MFMA i of 4 KT: key block i % KT (of the wave's), the query's high or low parts (i / KT % 2), channels
  // 64 (i / (2 KT)) + [0, 64). Its operand is piece 2 (i / (2 KT)) + h of key 32 (kh + i % KT) + col.
  u32x4 kf[KT];
  uint32_t ksc[KT];
  const int krow = (kh * 32 + col) * fp4::kHeadCodes, kswz = (col >> 2) & 3;  // (32 keys on: the same swizzle)
  auto read_k = [&](const uint8_t* kd, int ks) {
#pragma unroll
    for (int rt = 0; rt < KT; ++rt)
      kf[rt] = *reinterpret_cast<const u32x4*>(kd + rt * 32 * fp4::kHeadCodes + krow + (((2 * ks + h) ^ kswz) << 4));
  };
  auto read_scales = [&](const uint8_t* kd) {  // bytes 0 and 2: the scales of channels 32 h and 64 + 32 h on
#pragma unroll
    for (int rt = 0; rt < KT; ++rt)
      ksc[rt] = *reinterpret_cast<const uint32_t*>(kd + kCodes + ((kh + rt) * 32 + col) * 4) >> (8 * h);
  };
  auto score = [&](int i, f32x16 (&s)[KT]) {
    const int rt = i % KT, ks = i / (2 * KT);
    const fp4::i32x8 q = (i / KT) & 1 ? qlo[ks] : qhi[ks];
    f32x16 z;
#pragma unroll
    for (int j = 0; j < 16; ++j) z[j] = 0.f;
    const f32x16 in = i < KT ? z : s[rt];
    s[rt] = ks == 0 ? fp4::mfma_scores32<0>(kf[rt], ksc[rt], q, qs, in) : fp4::mfma_scores32<2>(kf[rt], ksc[rt], q, qs, in);
  };
  auto mask = [&](f32x16 (&s)[KT], int kv0, bool mapped) -> bool {  // whether something was to be masked
    if (mapped && kv0 + kBK <= min(all_see, nk)) return false;  // workgroup-uniform
    const int lim = mapped ? limit - kv0 - 32 * kh - 4 * h : INT_MIN;  // this half's keys below it are seen
#pragma unroll
    for (int rt = 0; rt < KT; ++rt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[rt][i] = rt * 32 + 8 * (i / 4) + i % 4 < lim ? s[rt][i] : -INFINITY;
    return true;
  };
  auto top_of = [&](const f32x16 (&s)[KT]) {
    float t = s[0][0];
#pragma unroll
    for (int rt = 0; rt < KT; ++rt)
#pragma unroll
      for (int i = 0; i < 16; ++i) t = fmaxf(t, s[rt][i]);
    return t;
  };
  // The running max for scores whose largest (of this lane) is top: it moves where that exceeds it by more than 8 in log2
  // units (p <= 256, exact after the final 1 / l).
  auto raise = [&](float top) {
    const float tm = xhalf_max(top) * c;
    const bool up = tm > m + 8.f;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(up) != 0, 0)) {
      const float alpha = up ? fast_exp2(m - tm) : 1.f;  // exp2(-inf) = 0 on the first update
      m = up ? tm : m;
      lsum *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
    }
  };
  auto tile_barrier = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  // One tile (kv0, its V in buffer buf; the next one's codes at `next`, its own place free for the one after): its softmax
  // and P V beside the next tile's score MFMAs and V conversion, in this order, pinned: an MFMA leaves the wave's issue slots
  // free, for about 2.3 elements' fma, exp, add and half a cvt (a score MFMA, 64 cycles) or 1.1 (a P V one, 32). Left to
  // itself the compiler runs the MFMAs together and the softmax together.
  auto step = [&](int kv0, int buf, f32x16 (&s)[KT], f32x16 (&sn)[KT], const uint8_t* next, uint8_t* own, bool& okn,
                  bool& okd) {
    const bool more = kv0 + kBK < kv_end;
    const int nan_at = s_nan_at[buf];
    constexpr int NS = 4 * KT, NP = 8 * KT, NE = 16 * KT;  // score and P V MFMAs, elements of a lane
    constexpr int E1 = KT == 2 ? 18 : 10;                  // elements beside the score MFMAs; the others ...
    constexpr int SPAN = NP - 4;                           // ... beside the P V ones before the last 16 keys'
    const float mu = m == -INFINITY ? 0.f : m;
    u32x4 pb[2 * KT];
    float e[4];
    float sum = 0.f;
    auto element = [&](int x) {
      e[x & 3] = fast_exp2(fmaf(s[x >> 4][x & 15], c, -mu));
      if (x & 1) pb[x >> 3][(x >> 1) & 3] = pack_bf16x2(e[(x & 3) - 1], e[x & 3]);
      if ((x & 3) == 3) {
        sum += (e[0] + e[1]) + (e[2] + e[3]);
        asm volatile("" : "+v"(sum));  // (here: sunk to the end of the tile, the adds would keep every e alive)
      }
    };
    const uint16_t* vt = L.v + buf * (kBK * kVRow) + vtr + kh * 32 * kVRow;
    u32x4 vf[4];
    auto read_v = [&](int i) {  // operand of P V MFMA i (16-key step i / 4, dims block i % 4)
      const u32x2 u0 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + (16 * (i >> 2)) * kVRow + (i & 3) * 32));
      const u32x2 u1 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + (16 * (i >> 2) + 8) * kVRow + (i & 3) * 32));
      vf[i & 3] = u32x4{u0[0], u0[1], u1[0], u1[1]};
    };
    if (more) {
      read_scales(next);
      read_k(next, 0);
      okd = issue(own);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        score(i, sn);
        if (i == 0) scale_v(next, kv0 + kBK, okn, buf ^ 1);
        if (i == NS / 2 - 1) read_k(next, 1);
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          if (i == (KT == 2 ? q4 + 2 : min(q4 + 1, 3))) piece_v(q4, buf ^ 1);
        if (i >= NS - 2) {
          read_v(2 * (i - (NS - 2)));
          read_v(2 * (i - (NS - 2)) + 1);
        }
#pragma unroll
        for (int x = i * E1 / NS; x < (i + 1) * E1 / NS; ++x) element(x);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) read_v(i);
#pragma unroll
      for (int x = 0; x < E1; ++x) element(x);
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      acc[i & 3] = mfma_32x32x16(vf[i & 3], pb[i >> 2], acc[i & 3]);
      if (i + 4 < NP) read_v(i + 4);
#pragma unroll
      for (int x = E1 + i * (NE - E1) / SPAN; x < E1 + (i + 1) * (NE - E1) / SPAN && x < NE; ++x) element(x);
      if (i >= NP - 4) {  // this lane's largest score of the next tile
#pragma unroll
        for (int x = 4 * KT * (i - (NP - 4)); x < 4 * KT * (i - (NP - 5)); ++x) top = fmaxf(top, sn[x >> 4][x & 15]);
        asm volatile("" : "+v"(top));  // (here)
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    lsum += sum;
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(nan_at) == kv0, 0)) mark_nan(buf, limit - kv0);
    if (more) {
      if (mask(sn, kv0 + kBK, okn)) top = top_of(sn);
      raise(top);
      tile_barrier();
    }
  };

  if (kv_end > 0) {
    f32x16 sa[KT], sb[KT];
#pragma unroll
    for (int rt = 0; rt < KT; ++rt)
#pragma unroll
      for (int i = 0; i < 16; ++i) sb[rt][i] = 0.f;  // (read by the last tile's step, which has no next one)
    if (tid < 2) s_nan_at[tid] = -1;
    tile_barrier();
    bool ok1 = issue(s_t1);
    read_scales(s_t0);
    scale_v(s_t0, 0, ok0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) piece_v(i, 0);
#pragma unroll
    for (int i = 0; i < 4 * KT; ++i) {
      if (i % (2 * KT) == 0) read_k(s_t0, i / (2 * KT));
      score(i, sa);
    }
    mask(sa, 0, ok0);
    raise(top_of(sa));
    tile_barrier();
    for (int kv0 = 0;;) {
      step(kv0, 0, sa, sb, s_t1, s_t0, ok1, ok0);
      if ((kv0 += kBK) >= kv_end) break;
      step(kv0, 1, sb, sa, s_t0, s_t1, ok0, ok1);
      if ((kv0 += kBK) >= kv_end) break;
    }
  }
  wait_vmem_all();  // (no transfer into LDS outlives the workgroup)

  // ---- O through LDS (in the V tiles, which are done with), so that a row leaves in 16-byte pieces side by side: 8-byte
  // stores straight from the accumulators, 32 rows apart, took a third of a short step's time (44 x 33-59 tokens over 50
  // cached: 16.0 us, 11.2 up to here). KS = 2: first the two waves of a row block trade halves: wave kh finishes the dims
  // blocks 2 kh, 2 kh + 1.
  float l = xhalf_sum(lsum);
  constexpr int ND = 4 / KS;  // dims blocks a wave finishes
  constexpr int kORow = kD + 8;
  static_assert(4 / KS * 32 * kORow <= 2 * kBK * kVRow && 4 * 64 * 36 * 2 <= 2 * kBK * kVRow, "they fit the V tiles");
  __syncthreads();
  if constexpr (KS == 2) {
    float* const sx = reinterpret_cast<float*>(L.v);  // [wave][piece of 4 or (m, l)][lane]
    f32x4* const mine = reinterpret_cast<f32x4*>(sx + w * 64 * 36);
    const f32x4* const theirs = reinterpret_cast<const f32x4*>(sx + (w ^ 2) * 64 * 36);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // the blocks that the other wave finishes
        const f32x16& o = kh == 0 ? acc[2 + dt] : acc[dt];
        mine[(dt * 4 + i) * 64 + lane] = f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
      }
    mine[8 * 64 + lane] = f32x4{m, l, __uint_as_float(nan_groups), 0.f};
    __syncthreads();
    const f32x4 x = theirs[8 * 64 + lane];
    const float top = fmaxf(m, x[0]), mu = top == -INFINITY ? 0.f : top;
    const float a0 = fast_exp2(m - mu), a1 = fast_exp2(x[0] - mu);
    l = l * a0 + x[1] * a1;
    if constexpr (LSE) m = top;
    nan_groups |= __float_as_uint(x[2]);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 y = theirs[(dt * 4 + i) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[dt][4 * i + j] = (kh == 0 ? acc[dt][4 * i + j] : acc[2 + dt][4 * i + j]) * a0 + y[j] * a1;
      }
    __syncthreads();
  }
  if constexpr (LSE) {
    if (h == 0 && kh == 0 && tq < nq && row >= 0 && row < p.row_limit)
      p.lse[row * p.num_heads + head] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);  // a row that sees no key: zeros
  uint16_t* const so = L.v + rg * 32 * kORow;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // LDS column 32 dt + 8 i + 4 h + [0, 4): channels 32 i + 8 dt + 4 h + [0, 4)
      const float f = (nan_groups >> (8 * i)) & 1u ? __builtin_nanf("") : inv;
      *reinterpret_cast<u32x2*>(so + col * kORow + i * 32 + (kh * ND + dt) * 8 + 4 * h) =
          u32x2{pack_bf16x2(acc[dt][4 * i] * f, acc[dt][4 * i + 1] * f),
                pack_bf16x2(acc[dt][4 * i + 2] * f, acc[dt][4 * i + 3] * f)};
    }
  if constexpr (KS == 2) __syncthreads();
  else wave_lds_sync();
#pragma unroll
  for (int i = 0; i < 8 / KS; ++i) {
    const int r = (kh * (8 / KS) + i) * 4 + (lane >> 4);
    const int orho = rg * 32 + r;
    const int otq = qt * bq + (orho >> gsh);
    const int64_t orow = (int64_t)q0 + otq;
    const u32x4 x = *reinterpret_cast<const u32x4*>(so + r * kORow + (lane & 15) * 8);
    if (otq < nq && orow >= 0 && orow < p.row_limit)
      *reinterpret_cast<u32x4_a8*>(p.out + orow * p.out_row_stride + (int64_t)((g << gsh) + (orho & (p.group - 1))) * kD +
                                   (lane & 15) * 8) = x;
  }
}

template <int KS, bool LSE>
__global__ __launch_bounds__(256, 2) void prefill_fp4_kernel(PrefillArgs p) {
  __shared__ __attribute__((aligned(16))) uint16_t s_v[2 * kBK * kVRow];
  __shared__ __attribute__((aligned(16))) uint8_t s_t0[2 * kTileBytes], s_t1[2 * kTileBytes];
  __shared__ __attribute__((aligned(4))) uint8_t s_nan[2 * kBK * 4];
  __shared__ int s_nan_at[2];
  // the last tile has the most keys: first
  prefill_item<KS, LSE>(p, (int)blockIdx.y, (int)blockIdx.z, (int)gridDim.x - 1 - (int)blockIdx.x,
                        Lds{s_v, s_t0, s_t1, s_nan, s_nan_at});
}

// ---- steps that mix prompts with decode rows, in one launch: workgroups [0, da.grid) are the decode split of the one-query
// rows (decode_fp4.h, four waves), the others a prefill item each. The decode rows are a stream from memory, the prompts
// chains of key tiles: side by side on a CU each has what the other leaves. Both fit a CU because the decode role's V tiles
// lie where the prefill's do, its tables where the codes are. 16 query heads of 2 kv heads, with the merge, against a launch
// of each: 6 prompts of 300-600 tokens and 120 decode rows over 128-1800 44.7 -> 28.5 us; 4 x 200-400 over 1000 cached and
// 100 over 500-1500 61.0 -> 38.0; one of 40 and 8 over 100-500 18.5 -> 12.9.
constexpr int kMixedSeqs = 256;

// Item x of the launch: (sequence, kv head, query tile) in this order, the last tile of a sequence first; sequences of one
// query have none. Every wave finds it by itself. Returns whether there is one.
__device__ __forceinline__ bool find_item(const PrefillArgs& p, int x, int bq, int& b, int& g, int& qt) {
  const int lane = threadIdx.x & 63;
  int tiles[kMixedSeqs / 64];
#pragma unroll
  for (int i = 0; i < kMixedSeqs / 64; ++i) {
    const int s = i * 64 + lane;
    const int nq = s < p.batch ? p.cu_q[s + 1] - p.cu_q[s] : 0;
    tiles[i] = nq > 1 ? (nq + bq - 1) / bq : 0;
  }
  const int hk = p.num_kv_heads;
  g = x % hk;
  int r = x / hk;  // tiles before it
#pragma unroll
  for (int i = 0; i < kMixedSeqs / 64; ++i) {
    const int incl = wave_incl_scan_dpp(tiles[i]);
    const uint64_t past = __builtin_amdgcn_ballot_w64(incl > r);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      b = i * 64 + l;
      qt = __builtin_amdgcn_readlane(incl, l) - 1 - r;
      return true;
    }
    r -= __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

template <int HK, int KS>
__global__ __launch_bounds__(256, 2) void mixed_fp4_kernel(PrefillArgs pa, DecodeArgs da) {
  using LD = dec::LdsFp4<HK, false, 4, 3>;
  constexpr int kVs = LD::kNW * LD::kVt > 2 * kBK * kVRow ? LD::kNW * LD::kVt : 2 * kBK * kVRow;
  __shared__ __attribute__((aligned(16))) uint16_t s_v[kVs];
  __shared__ __attribute__((aligned(16))) uint8_t s_t0[2 * kTileBytes], s_t1[2 * kTileBytes];
  __shared__ __attribute__((aligned(16))) float s_slot[(LD::kRoundSegs - 1) * kPartialFloats];
  __shared__ __attribute__((aligned(4))) uint8_t s_nan[2 * kBK * 4];
  __shared__ int s_nan_at[2];
  static_assert((LD::kBtInts + dec::kRecTiles) * 4 <= sizeof(s_t0), "records and tile ids");
  static_assert((4 * kMixedSeqs + 1 + 2 * LD::kNW) * 4 <= sizeof(s_t1), "the step's layout");
  if ((int)blockIdx.x < da.grid) {
    int* const i0 = reinterpret_cast<int*>(s_t0);
    int* const i1 = reinterpret_cast<int*>(s_t1);
    const LD L{s_v,
               s_slot,
               i1,
               i1 + kMixedSeqs,
               i1 + 2 * kMixedSeqs,
               i1 + 3 * kMixedSeqs,
               i1 + 4 * kMixedSeqs + 1,
               i1 + 4 * kMixedSeqs + 1 + LD::kNW,
               i0,
               i0 + LD::kBtInts};
    dec::decode_split<HK>(da, (int)blockIdx.x, da.grid, L);
    return;
  }
  int b, g, qt;
  if (!find_item(pa, (int)blockIdx.x - da.grid, 128 / KS / pa.group, b, g, qt)) return;
  __builtin_amdgcn_s_setprio(1);  // the decode waves wait for memory anyway
  prefill_item<KS>(pa, b, g, qt, Lds{s_v, s_t0, s_t1, s_nan, s_nan_at});
}

// Workgroups of `rows` query rows at most: every sequence's tiles, or one tile in part a sequence and the others full.
int64_t most_items(const PrefillArgs& a, int max_seqlen_q, int rows) {
  const int bq = std::max(1, rows / a.group);
  return std::min((int64_t)a.batch * ((max_seqlen_q + bq - 1) / bq), a.row_limit / bq + a.batch) * a.num_kv_heads;
}

}  // namespace pf4

}  // namespace

bool mixed_fp4_fits(const PrefillArgs& a, int max_seqlen_q) {
  return max_seqlen_q > 1 && a.batch <= pf4::kMixedSeqs && pf4::most_items(a, max_seqlen_q, 64) < (1 << 22);
}

hipError_t launch_mixed_fp4(const PrefillArgs& a, int max_seqlen_q, const DecodeArgs& d, hipStream_t stream) {
  // Two waves on the same rows where the prompts (what is left of the rows without one a sequence: nearly all of these are
  // decode rows) are at most half a workgroup a compute unit, as in launch_prefill_fp4. Prompts beside 60-100 decode rows,
  // KS = 1 | 2, 8 query heads of one kv head: 2000 tokens (125 items) 46.3 | 39.5 us, 4 x 200-400 over 1000 (86) 36.1 |
  // 31.4, 400 (25) 18.1 | 16.6, 3 x 1000-1500 (249) 38.0 | 46.8; 16 heads of two: 400 (50) 19.3 | 18.6, 6 x 300-600 (332)
  // 28.5 | 35.7.
  const bool two = a.group <= 64 && (a.row_limit - a.batch) * a.num_kv_heads <= (int64_t)pf4::kHalfChip * (128 / a.group);
  const dim3 grid((unsigned)(d.grid + pf4::most_items(a, max_seqlen_q, two ? 64 : 128)));
  if (a.num_kv_heads == 1)
    two ? pf4::mixed_fp4_kernel<1, 2><<<grid, dim3(256), 0, stream>>>(a, d)
        : pf4::mixed_fp4_kernel<1, 1><<<grid, dim3(256), 0, stream>>>(a, d);
  else
    two ? pf4::mixed_fp4_kernel<2, 2><<<grid, dim3(256), 0, stream>>>(a, d)
        : pf4::mixed_fp4_kernel<2, 1><<<grid, dim3(256), 0, stream>>>(a, d);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  return launch_decode_merge_fp4(d, stream);
}

template <bool LSE>
static hipError_t launch_prefill_fp4_form(const PrefillArgs& a, int max_seqlen_q, hipStream_t stream) {
  // Two waves on the same rows where the launch is at most half a workgroup a compute unit: the chain of tiles is then the
  // time (16 query heads of 2 kv heads, KS = 1 | 2: 1000 tokens over 2000 cached, 126 workgroups of 128 rows, 58.6 | 47.6 us;
  // 4 x 200 over 2000, 104: 44.9 | 36.8; 100 over 300, 14: 13.4 | 11.9). From there on 64-row workgroups stage and convert
  // every tile twice as often for more than they save (156 workgroups 19.5 | 20.8 us, 298: 12.7 | 16.4, 1134: 152 | 177).
  // (group 128: 64 rows would be half a token)
  const bool two = a.group <= 64 && pf4::most_items(a, max_seqlen_q, 128) <= pf4::kHalfChip;
  const int bq_ks = (two ? 64 : 128) / a.group;
  const dim3 grid((unsigned)((max_seqlen_q + bq_ks - 1) / bq_ks), (unsigned)a.batch, (unsigned)a.num_kv_heads);
  if (two)
    pf4::prefill_fp4_kernel<2, LSE><<<grid, dim3(256), 0, stream>>>(a);
  else
    pf4::prefill_fp4_kernel<1, LSE><<<grid, dim3(256), 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_prefill_fp4(const PrefillArgs& a, int max_seqlen_q, hipStream_t stream) {
  return launch_prefill_fp4_form<false>(a, max_seqlen_q, stream);
}

hipError_t launch_prefill_lse_fp4(const PrefillArgs& a, int max_seqlen_q, hipStream_t stream) {
  if (max_seqlen_q <= 0 || a.batch <= 0) return hipSuccess;
  if (!a.lse || !a.causal) return hipErrorInvalidValue;
  return launch_prefill_fp4_form<true>(a, max_seqlen_q, stream);
}

}  // namespace vox
