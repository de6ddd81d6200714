// The walk of a wave over 4-bit keys and values (fp4_common.h has the format): what decode_split's LDS policy brings
// where the cache is not bf16. The layout, the plan records, the rounds and the merges are decode_body.h's.
//
// A wave takes its share in chunks of two 16-token steps of one sequence (the second may be missing).
//  * Scores: the codes go from memory into the MFMA as they are (fp4, lane = token r16, channels 32 jq + [0, 32), one
//    scale a lane), against the query in fp8. A query value needs two fp8 (mfma_scores16): with HK = 2 the 16 columns are
//    the high parts of a kv head's 8 query heads and their low parts, one MFMA per kv head and step, and lane c adds
//    column c ^ 8; with HK = 1 they are the 16 heads, high and low parts by an MFMA each. No conversion of K at all.
//  * Values: a lane's 16 bytes are 32 channels of one token and kv head and share one scale: 16 conversions to bf16
//    (exact), then LDS, one kv head at a time in the same tile. Piece w of group c of a row (8 channels) goes to 16-byte
//    column 4 w + c, so that the four lanes of a token write consecutive columns (in channel order they would be 64 bytes
//    apart, a four-way bank conflict); the transposed reads then hand out the channels in that order, and put() writes
//    them where they belong.
//  * O^T += V^T P^T by 16x16x32 MFMAs, both steps at once.
// 136 HK bytes a key: bound by HBM over long contexts (24 streams of 20000-32768 tokens, 177 MB: 36-40 us, 4.4-4.9 TB/s; the
// bf16 cache's kernel takes 107 us), by fixed costs over short ones: start, layout, one round trip of loads and the merge of
// the waves (one of 420: 7.9 us; 150 of 256-2048, 46 MB: 22 us). A chunk's key loads sent ahead of its
// softmax, the values' one head at a time, in place of all at its end: 25.4 -> 26.3 us and 41 -> 42.7 with the merge.
// Eight waves a workgroup over long ranges (launch_split): one wave's conversions, LDS reads and MFMAs wait for each other
// most of the time (with four, VALU and MFMA were busy for under a third of it each), and two to a SIMD fill each other's
// gaps.
// The scales are loaded as words, four a lane, and shifted where they are used: a byte load's zero extension, an
// instruction of its own, was put behind the loads of the next chunk and waited for all of them.
// Loads are buffer loads whose descriptor ends with the cache block and is empty for a step that is not there: nothing
// outside the block is read, and every chunk issues the same loads.
#pragma once

#include "decode_body.h"
#include "fp4_common.h"

namespace vox {

namespace {

namespace dec {

constexpr int kSteps = 2;  // steps of a chunk

template <int HK>
struct Chunk {
  u32x4 k[kSteps][HK];      // codes: token r16 of the step, kv head g, channels 32 jq + [0, 32)
  uint32_t ks[kSteps][HK];  // the token's four scales of kv head g, the lane's in byte jq
  u32x4 v[kSteps][HK];      // codes: token lane / 4 of the step, kv head g, channels 32 (lane % 4) + [0, 32)
  uint32_t vs[kSteps][HK];  // the token's four scales of kv head g, the lane's in byte lane % 4
  bool ok[kSteps];          // the step exists and its block is mapped
  int fresh;                // store mode: the chunk's token that is the step's new one (-1: none), its row in `piece`
  u32x4 piece;              // 8 channels: lanes [0, 16 HK) of its key row, [16 HK, 32 HK) of its value row
};

template <int HK, bool BTL, int NW, int SEGS = 6, bool SCORES = false>
struct LdsFp4 {
  static constexpr bool kOwnWalk = true;
  static constexpr int kNW = NW;
  static constexpr int kGet = 8 / NW;
  static constexpr int kRoundSegs = SEGS;
  static constexpr bool kBtl = BTL;
  static constexpr int kBtInts = BTL ? (kBtLds > kPlanRecInts ? kBtLds : kPlanRecInts) : kPlanRecInts;
  static constexpr int VROW = kD + 32;  // elements of an LDS row: four rows' 64-byte runs, and the reads', in distinct banks
  static constexpr int kVt = kSteps * kTile * VROW;  // one wave's V tile
  static_assert(kVt * 2 >= kPartialFloats * 4, "a V tile holds a partial");
  uint16_t* vt_all;  // [kNW][kVt]
  float* slots;      // [kRoundSegs - 1][kPartialFloats]
  int *ctx, *row, *snew, *start, *wtot, *wmax, *bt, *rtiles;
  __device__ __forceinline__ uint16_t* vt(int w) const { return vt_all + w * kVt; }
  // A wave's partial of segment k of the round: of its share's last segment in its V tile, which it has done with; of the
  // others in slot k (a segment ends in one wave's share, so only that wave leaves it before its last).
  __device__ __forceinline__ float* partial(int w, int k, bool last) const {
    return last ? reinterpret_cast<float*>(vt(w)) : slots + k * kPartialFloats;
  }
  // head hh's part: accumulator a, rows jq*4 + [0, 4) are 4 channels
  __device__ __forceinline__ void put4(float* sl, int hh, int jq, const f32x4 (&acc)[8], float m, float l) const {
#pragma unroll
    for (int a = 0; a < 8; ++a)
      *reinterpret_cast<f32x4*>(&sl[hh * kD + (2 * (a & 1) + (jq >> 1)) * 32 + (a >> 1) * 8 + (jq & 1) * 4]) = acc[a];
    if (jq == 0) {
      sl[kMOff + hh] = m;
      sl[kLOff + hh] = l;
    }
  }
  __device__ __forceinline__ void get(int w, int k, bool last, int hh, int d0, f32x4 (&o)[kGet], float& m,
                                      float& l) const {
    const float* sl = partial(w, min(k, kRoundSegs - 2), last);  // (a pair that is none reads any slot: it is not used)
    m = sl[kMOff + hh];
    l = sl[kLOff + hh];
#pragma unroll
    for (int i = 0; i < kGet; ++i) o[i] = *reinterpret_cast<const f32x4*>(&sl[hh * kD + d0 + 4 * i]);
  }

  // Wave w's share [t_lo, t_hi) of a round, from window lane k on, the kc-th segment of the round; a partial for each
  // segment goes where partial() says. win: the window's values of a lane (st, en, ctx, row).
  template <class BlockAt, class NextSeg, class Win>
  __device__ __forceinline__ void walk(const DecodeArgs& p, int w_, int t_lo_, int t_hi_, int k_, int kc_,
                                       BlockAt block_at, NextSeg next_seg, Win win) const {
    // (in scalar registers: the descriptors of the loads are made from them)
    const int w = uniform(w_), t_lo = uniform(t_lo_), t_hi = uniform(t_hi_);
    int k = uniform(k_), kc = uniform(kc_);
    const int lane = threadIdx.x & 63;
    const int r16 = lane & 15;
    const int jq = lane >> 4;
    const int64_t bb = fp4::block_bytes(p.block_size, HK);
    const int scales = p.block_size * HK * fp4::kHeadCodes;  // where a block's scales start
    const int kcode = r16 * HK * fp4::kHeadCodes + jq * 16, kscale = r16 * HK * fp4::kHeadScales;
    const int vcode = (lane >> 2) * HK * fp4::kHeadCodes + (lane & 3) * 16, vscale = (lane >> 2) * HK * fp4::kHeadScales;

    const bool store = p.slot_mapping != nullptr;  // (never in varlen mode: slots are a row's own)
    // ---- the next chunk to load: step ti of window lane ki, whose sequence ends (in this share) at step ei, at slot `in`
    // of the block in table column `col`
    int ki = k, ti = t_lo, ei = 0, col = 0, in = 0;
    auto enter = [&]() {
      ei = min(t_hi, win.en(ki));
      const int tok = (ti - win.st(ki)) * kTile;
      col = tok / p.block_size;
      in = tok - col * p.block_size;
    };
    enter();
    auto issue = [&](Chunk<HK>& T) {
      const int fresh_slot = store ? win.snew(ki) : -1;
      T.fresh = -1;
      const int64_t nrow = win.row(ki);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bool there = ti < ei;
        const int blk = there ? uniform((int)block_at(ki, ti, col)) : -1;
        T.ok[s] = blk >= 0 && blk < p.num_blocks;
        if (store) {
          const int64_t d = (int64_t)fresh_slot - ((int64_t)blk * p.block_size + in);
          if (T.ok[s] && d >= 0 && d < kTile) T.fresh = s * kTile + (int)d;
        }
        const int range = T.ok[s] ? (int)bb : 0;
        const int64_t at = T.ok[s] ? blk * bb : 0;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.k_cache) + at, (short)0, range,
                                                          fp4::kBufferWord3);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.v_cache) + at, (short)0, range,
                                                          fp4::kBufferWord3);
        const int c0 = in * HK * fp4::kHeadCodes, s0 = scales + in * HK * fp4::kHeadScales;
        ti += there ? 1 : 0;
        in += kTile;
        if (in == p.block_size) {
          in = 0;
          ++col;
        }
#pragma unroll
        for (int g = 0; g < HK; ++g) {
          T.k[s][g] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, kcode + g * fp4::kHeadCodes, c0, 0));
          T.ks[s][g] = __builtin_amdgcn_raw_buffer_load_b32(rk, kscale + g * fp4::kHeadScales, s0, 0);
        }
#pragma unroll
        for (int g = 0; g < HK; ++g) {
          T.v[s][g] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, vcode + g * fp4::kHeadCodes, c0, 0));
          T.vs[s][g] = __builtin_amdgcn_raw_buffer_load_b32(rv, vscale + g * fp4::kHeadScales, s0, 0);
        }
      }
      if (T.fresh >= 0) {
        const int at = (lane & (16 * HK - 1)) * 8;
        T.piece = ld_g16((lane & (16 * HK) ? p.new_v + nrow * p.new_v_stride : p.new_k + nrow * p.new_k_stride) + at);
      }
      if (ti == ei && ti < t_hi) {
        ki = next_seg(ki);
        enter();
      }
    };

    // what lane c ^ 8 of the 16 gives
    auto other_part = [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x128, 0xF, 0xF, false); };
    // ---- the query of a sequence: column r16 of kv head g's operand is a part of head (HK == 2: g * group + r16 % 8)
    // With HK == 2 lanes c and c ^ 8 hold parts of the same values: each loads and splits half of them (channels 16 jq +
    // [0, 16), or 64 on) and they trade.
    constexpr int QL = HK == 2 ? 2 : 4;  // 16-byte loads of a lane
    auto load_q = [&](u32x4 (&qv)[HK][QL], int ks) {
#pragma unroll
      for (int g = 0; g < HK; ++g) {
        const int c = HK == 2 ? (r16 & 7) : r16;
        const int hd = HK == 2 ? g * p.group + (c < p.group ? c : 0) : (c < p.num_heads ? c : 0);
        const uint16_t* qb = p.q + (int64_t)win.row(ks) * p.q_row_stride + (int64_t)hd * kD + jq * 16 +
                             (HK == 2 ? (r16 >> 3) * 64 : 0);
#pragma unroll
        for (int i = 0; i < QL; ++i) qv[g][i] = ld_g16(qb + (i >> 1) * 64 + (i & 1) * 8);
      }
    };
    // qop[g]: HK == 2: high parts of kv head g's heads in columns 0-7, low parts in 8-15; HK == 1: qop[0] high, qop[1] low
    fp4::i32x8 qop[2];
    uint32_t qs[HK];
    auto make_q = [&](const u32x4 (&qv)[HK][QL]) {
#pragma unroll
      for (int g = 0; g < HK; ++g) {
        uint32_t mb = 0;
#pragma unroll
        for (int i = 0; i < QL; ++i) mb = max(mb, fp4::max_bits(qv[g][i]));
        if constexpr (HK == 2) mb = max(mb, (uint32_t)other_part((int)mb));
        mb = __float_as_uint(col_max4(__uint_as_float(mb << 16))) >> 16;  // the whole row
        qs[g] = fp4::query_scale_byte(mb);
        const float scale = fp4::scale_float(qs[g]), inv = fp4::query_inverse(qs[g]);
#pragma unroll
        for (int i = 0; i < 2 * QL; ++i) {
          int hi, lo;
          fp4::query_parts4(qv[g][i / 2][(i & 1) * 2], qv[g][i / 2][(i & 1) * 2 + 1], scale, inv, hi, lo);
          if constexpr (HK == 2) {
            const int keep = r16 < 8 ? hi : lo, got = other_part(r16 < 8 ? lo : hi);
            qop[g][i] = r16 < 8 ? keep : got;
            qop[g][i + 4] = r16 < 8 ? got : keep;
          } else {
            qop[0][i] = hi;
            qop[1][i] = lo;
          }
        }
      }
    };
    const int hc = HK == 2 ? (r16 & 7) : r16;
    const bool head_ok = HK == 2 ? hc < p.group : hc < p.num_heads;
    const int head = HK == 2 ? (r16 >> 3) * p.group + hc : hc;
    const int hg = HK == 2 ? r16 >> 3 : 0;

    float m = -INFINITY;
    float lsum = 0.f;
    uint32_t nan_groups = 0;  // bit (kv head, 32-channel group): a value of the sequence is not a number
    f32x4 acc[8];
#pragma unroll
    for (int a = 0; a < 8; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint16_t* vt_w = vt(w);
    uint16_t* vst = vt_w + (lane >> 2) * VROW + (lane & 3) * 8;                  // stores
    const uint16_t* vtr = vt_w + (jq * 4 + (r16 >> 2)) * VROW + 4 * (r16 & 3);   // transposed reads
    const float c = p.scale_log2;

    // Store mode: the new token as the cache will hold it, in the place of what was loaded for it (its row is stored by the
    // merge kernel, after every read). The wave quantises the row once (a lane 8 channels, as store_fp4_kernel) and hands
    // codes and scales out through its V tile.
    auto take_fresh = [&](Chunk<HK>& T) {
      uint32_t codes, b;
      fp4::quantise8(T.piece, codes, b);
      uint8_t* const s = reinterpret_cast<uint8_t*>(vt_w);
      constexpr int kRow = HK * fp4::kHeadCodes, kScales = 2 * kRow;  // key codes, value codes, then their scales
      if (lane < 32 * HK) {
        *reinterpret_cast<uint32_t*>(s + lane * 4) = codes;
        if ((lane & 3) == 0) s[kScales + (lane >> 2)] = (uint8_t)b;
      }
      wave_lds_sync();
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const int r = T.fresh - st * kTile;
#pragma unroll
        for (int g = 0; g < HK; ++g) {
          const u32x4 kc = *reinterpret_cast<const u32x4*>(s + g * fp4::kHeadCodes + jq * 16);
          const u32x4 vc = *reinterpret_cast<const u32x4*>(s + kRow + g * fp4::kHeadCodes + (lane & 3) * 16);
          const uint32_t ks = *reinterpret_cast<const uint32_t*>(s + kScales + g * 4);
          const uint32_t vs = *reinterpret_cast<const uint32_t*>(s + kScales + HK * 4 + g * 4);
          T.k[st][g] = r16 == r ? kc : T.k[st][g];
          T.ks[st][g] = r16 == r ? ks : T.ks[st][g];
          T.v[st][g] = lane >> 2 == r ? vc : T.v[st][g];
          T.vs[st][g] = lane >> 2 == r ? vs : T.vs[st][g];
        }
      }
      wave_lds_sync();
    };

    // A chunk whose first token is t0, of a sequence that ends at tok_end: scores, online softmax (the running max moves
    // when the chunk's exceeds it by more than 8 in log2 units, as in decode_body.h) and P V, one kv head after the other.
    // `between`: called when the chunk's registers are free. SCORES: the scores of its steps, from step t on and below `en`, go
    // to p.scores as decode_split's do, behind the next chunk's loads.
    auto compute = [&](Chunk<HK>& T, int t, int en, int t0, int tok_end, auto&& between) {
      if (T.fresh >= 0) take_fresh(T);
      int lim[kSteps];  // tokens of each step that count
#pragma unroll
      for (int s = 0; s < kSteps; ++s) lim[s] = T.ok[s] ? tok_end - t0 - s * kTile : 0;
      float x[kSteps * 4];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const f32x4 z = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 y;
        uint32_t sc[HK];
#pragma unroll
        for (int g = 0; g < HK; ++g) sc[g] = T.ks[s][g] >> (8 * jq);
        if constexpr (HK == 2) {
          const f32x4 y0 = fp4::mfma_scores16(T.k[s][0], sc[0], qop[0], qs[0], z);
          const f32x4 y1 = fp4::mfma_scores16(T.k[s][1], sc[1], qop[1], qs[1], z);
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // lane c keeps kv head c / 8 and adds the other part, in lane c ^ 8
            const float give = r16 < 8 ? y1[i] : y0[i], keep = r16 < 8 ? y0[i] : y1[i];
            y[i] = keep + __int_as_float(other_part(__float_as_int(give)));
          }
        } else {
          y = fp4::mfma_scores16(T.k[s][0], sc[0], qop[0], qs[0], z);
          y = fp4::mfma_scores16(T.k[s][0], sc[0], qop[1], qs[0], y);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[s * 4 + i] = jq * 4 + i < lim[s] ? y[i] : -INFINITY;
      }
      // The values of kv head g into LDS as bf16. Groups that are not numbers (or past bf16: held_scale) stay out of the MFMAs
      // (the zeros that keep the kv heads apart would not hide them): the sequence's heads of that kv head are NaN in the group.
      auto store_v = [&](int g) {
        uint32_t b[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) b[s] = (lane >> 2) < lim[s] ? (T.vs[s][g] >> (8 * (lane & 3))) & 0xffu : 0u;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(max(b[0], b[1]) >= 253u) != 0, 0)) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) b[s] = fp4::held_scale(b[s], T.v[s][g]);
          uint64_t bad = __builtin_amdgcn_ballot_w64(max(b[0], b[1]) == 255u);
#pragma unroll
          for (int i = 32; i >= 4; i >>= 1) bad |= bad >> i;
          nan_groups |= ((uint32_t)bad & 15u) << (4 * g);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) b[s] = b[s] == 255u ? 0u : b[s];
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<u32x4*>(vst + s * kTile * VROW + q4 * 32) =
                fp4::values8(T.v[s][g][q4], fp4::scale_float(b[s]));
        wave_lds_sync();
      };
      store_v(0);
      float raw[SCORES ? kSteps * 4 : 1];
      if constexpr (SCORES) {
#pragma unroll
        for (int i = 0; i < kSteps * 4; ++i) raw[i] = x[i];
      }

      float tm = x[0];
#pragma unroll
      for (int i = 1; i < kSteps * 4; ++i) tm = fmaxf(tm, x[i]);
      tm = col_max4(tm) * c;
      const bool up = tm > m + 8.f;
      if (__builtin_amdgcn_ballot_w64(up) != 0) {  // wave-uniform
        const float alpha = up ? fast_exp2(m - tm) : 1.f;  // exp2(-inf) = 0 on the first update
        m = up ? tm : m;
        lsum *= alpha;
#pragma unroll
        for (int a = 0; a < 8; ++a) acc[a] *= alpha;
      }
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < kSteps * 4; ++i) {
        x[i] = fast_exp2(fmaf(x[i], c, -mu));
        lsum += x[i];
      }
      // P^T in bf16 (off by at most 2^-8 of each, as the output is): k-slots 4 s + i = token 16 s + 4 jq + i
      u32x4 pv;
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
#pragma unroll
      for (int g = 0; g < HK; ++g) {
        if (g > 0) store_v(g);
        if (g == HK - 1) {
          between();
          if constexpr (SCORES) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
              if (head_ok && t + s < en)
                *reinterpret_cast<f32x4*>(p.scores + ((int64_t)(t + s) * p.num_heads + head) * kTile + jq * 4) =
                    f32x4{raw[4 * s], raw[4 * s + 1], raw[4 * s + 2], raw[4 * s + 3]};
          }
        }
        const u32x4 pb = HK == 1 || hg == g ? pv : zero4();
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          const u32x2 u0 = __builtin_bit_cast(u32x2, lds_read_tr16(vtr + a * 16));
          const u32x2 u1 = __builtin_bit_cast(u32x2, lds_read_tr16(vtr + kTile * VROW + a * 16));
          acc[a] = mfma_16x16x32(u32x4{u0[0], u0[1], u1[0], u1[1]}, pb, acc[a]);
        }
        wave_lds_sync();
      }
    };

    // ---- one chunk in registers; the next one's loads go out as soon as they are free
    Chunk<HK> T;
    u32x4 qv[HK][QL];
    load_q(qv, k);
    issue(T);
    make_q(qv);
    int t = t_lo;
    for (;;) {
      const int en = min(t_hi, win.en(k));
      const bool last = t + kSteps >= en;  // of the segment
      int kn = k;
      if (last && en < t_hi) {
        kn = next_seg(k);
        load_q(qv, kn);
      }
      compute(T, t, en, (t - win.st(k)) * kTile, win.ctx(k), [&]() { issue(T); });
      t += kSteps;
      if (!last) continue;
      const float l = col_sum4(lsum);
      if (__builtin_expect(nan_groups != 0, 0)) {
#pragma unroll
        for (int a = 0; a < 8; ++a)
          if ((nan_groups >> (hg * 4 + 2 * (a & 1) + (jq >> 1))) & 1u)
            acc[a] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
      }
      if (head_ok) put4(partial(w, kc, en >= t_hi), head, jq, acc, m, l);
      if (en >= t_hi) break;
      m = -INFINITY;
      lsum = 0.f;
      nan_groups = 0;
#pragma unroll
      for (int a = 0; a < 8; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
      make_q(qv);
      t = en;
      k = kn;
      ++kc;
    }
  }
};

}  // namespace dec

}  // namespace

}  // namespace vox
