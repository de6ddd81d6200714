// The walk of a wave over 4-bit keys and values (fp4_common.h has the format): what decode_split's LDS policy brings
// where the cache is not bf16. The layout, the plan records, the rounds and the merges are decode_body.h's.
//
// A wave takes its share in chunks of two 16-token steps of one sequence (the second may be missing).
//  * Scores: the codes go from memory into the MFMA as they are (fp4, lane = token r16, channels 32 jq + [0, 32), one
//    scale a lane), against the query in fp8. A query value needs two fp8 (mfma_scores16): with HK = 2 the 16 columns are
//    the high parts of a kv head's 8 query heads and their low parts, one MFMA per kv head and step, and lane c adds
//    column c ^ 8; with HK = 1 they are the 16 heads, high and low parts by an MFMA each. No conversion of K at all.
//  * Values: a lane's 16 bytes are 32 channels of one token and share one scale: 16 conversions to bf16 (exact), then LDS.
//    Piece w of chunk c of a row (8 channels) goes to 16-byte column w CPR + c, so that the lanes of one store write
//    consecutive columns (in channel order they would be 64 bytes apart, a four-way bank conflict); the transposed reads
//    then hand out the channels in that order, and put() writes them where they belong.
//  * O^T += V^T P^T by 16x16x32 MFMAs, both steps at once.
// Loads are buffer loads whose descriptor ends with the cache block and is empty for a step that is not there: nothing
// outside the block is read, and every chunk issues the same loads, so the waits count them exactly.
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
  uint32_t ks[kSteps][HK];  // their scales
  u32x4 v[kSteps][HK];      // codes: the step's 16-byte pieces i * 64 + lane
  uint32_t vs[kSteps][HK];  // their scales
  bool ok[kSteps];          // the step exists and its block is mapped
};

template <int HK, bool BTL>
struct LdsFp4 {
  static constexpr bool kOwnWalk = true;
  static constexpr int kRoundSegs = 5;
  static constexpr int kSlots = kRoundSegs + kWaves - 1;
  static constexpr bool kBtl = BTL;
  static constexpr int kBtInts = BTL ? (kBtLds > kPlanRecInts ? kBtLds : kPlanRecInts) : kPlanRecInts;
  static constexpr int CPR = HK * 4;  // 16-byte pieces of a token's codes: its groups of 32 channels
  static constexpr int VROW = Tile<HK>::VROW;
  static constexpr int kVt = kSteps * kTile * VROW;  // one wave's V tile
  uint16_t* vt_all;  // [kWaves][kVt]
  float* slots;      // [kSlots][kPartialFloats]
  int *ctx, *row, *snew, *start, *wtot, *wmax, *bt, *rtiles;
  __device__ __forceinline__ uint16_t* vt(int w) const { return vt_all + w * kVt; }
  // head hh's part of a wave partial into slot si: accumulator a, rows jq*4 + [0, 4) are 4 channels from chan(a) on
  __device__ __forceinline__ void put4(int si, int hh, int jq, const f32x4 (&acc)[8], float m, float l) const {
    float* sl = slots + si * kPartialFloats;
#pragma unroll
    for (int a = 0; a < 8; ++a)
      *reinterpret_cast<f32x4*>(&sl[hh * kD + (2 * (a & 1) + (jq >> 1)) * 32 + (a >> 1) * 8 + (jq & 1) * 4]) = acc[a];
    if (jq == 0) {
      sl[kMOff + hh] = m;
      sl[kLOff + hh] = l;
    }
  }
  __device__ __forceinline__ void get(int si, int hh, int d0, f32x4 (&o)[2], float& m, float& l) const {
    const float* sl = slots + si * kPartialFloats;
    m = sl[kMOff + hh];
    l = sl[kLOff + hh];
    o[0] = *reinterpret_cast<const f32x4*>(&sl[hh * kD + d0]);
    o[1] = *reinterpret_cast<const f32x4*>(&sl[hh * kD + d0 + 4]);
  }

  // Wave w's share [t_lo, t_hi) of a round, from window lane k on, the kc-th segment of the round; a partial for each
  // segment goes to slot w + its number. win: the window's values of a lane (st, en, ctx, row).
  template <class BlockOf, class NextSeg, class Win>
  __device__ __forceinline__ void walk(const DecodeArgs& p, int w, int t_lo, int t_hi, int k, int kc, BlockOf block_of,
                                       NextSeg next_seg, Win win) const {
    constexpr int kRing = 2;  // chunks in flight
    const int lane = threadIdx.x & 63;
    const int r16 = lane & 15;
    const int jq = lane >> 4;
    const int64_t bb = fp4::block_bytes(p.block_size, HK);
    const int scales = p.block_size * HK * fp4::kHeadCodes;  // where a block's scales start
    const int kcode = r16 * CPR * 16 + jq * 16, kscale = r16 * CPR + jq;

    auto issue = [&](Chunk<HK>& T, bool any, int ks, int t) {
      const int end = min(t_hi, any ? win.en(ks) : 0);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bool in = any && t + s < end;
        const int64_t blk = in ? block_of(ks, t + s) : -1;
        T.ok[s] = blk >= 0 && blk < p.num_blocks;
        const int tok = in ? ((t + s - win.st(ks)) * kTile) % p.block_size : 0;
        const int range = T.ok[s] ? (int)bb : 0;
        const int64_t at = T.ok[s] ? blk * bb : 0;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.k_cache) + at, (short)0, range,
                                                          fp4::kBufferWord3);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.v_cache) + at, (short)0, range,
                                                          fp4::kBufferWord3);
        const int c0 = tok * HK * fp4::kHeadCodes, s0 = scales + tok * HK * fp4::kHeadScales;
#pragma unroll
        for (int g = 0; g < HK; ++g) {
          T.k[s][g] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, kcode + g * fp4::kHeadCodes, c0, fp4::kStream));
          T.ks[s][g] = __builtin_amdgcn_raw_buffer_load_b8(rk, kscale + g * fp4::kHeadScales, s0, fp4::kStream);
        }
#pragma unroll
        for (int i = 0; i < HK; ++i) {
          T.v[s][i] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, (i * 64 + lane) * 16, c0, fp4::kStream));
          T.vs[s][i] = __builtin_amdgcn_raw_buffer_load_b8(rv, i * 64 + lane, s0, fp4::kStream);
        }
      }
    };

    // ---- the query of a sequence: column r16 of kv head g's operand is a part of head (HK == 2: g * group + r16 % 8)
    auto load_q = [&](u32x4 (&qv)[HK][4], int ks) {
#pragma unroll
      for (int g = 0; g < HK; ++g) {
        const int c = HK == 2 ? (r16 & 7) : r16;
        const int hd = HK == 2 ? g * p.group + (c < p.group ? c : 0) : (c < p.num_heads ? c : 0);
        const uint16_t* qb = p.q + (int64_t)win.row(ks) * p.q_row_stride + (int64_t)hd * kD + jq * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) qv[g][i] = ld_g16(qb + (i >> 1) * 64 + (i & 1) * 8);
      }
    };
    // qop[g]: HK == 2: high parts of kv head g's heads in columns 0-7, low parts in 8-15; HK == 1: qop[0] high, qop[1] low
    fp4::i32x8 qop[2];
    uint32_t qs[HK];
    auto make_q = [&](const u32x4 (&qv)[HK][4]) {
#pragma unroll
      for (int g = 0; g < HK; ++g) {
        uint32_t mb = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) mb = max(mb, fp4::max_bits(qv[g][i]));
        mb = __float_as_uint(col_max4(__uint_as_float(mb << 16))) >> 16;  // the whole row: four lanes hold it
        qs[g] = fp4::query_scale_byte(mb);
        const float inv = fp4::query_inverse(qs[g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t a = qv[g][i / 2][(i & 1) * 2], b = qv[g][i / 2][(i & 1) * 2 + 1];
          const float x0 = __uint_as_float(a << 16) * inv, x1 = __uint_as_float(a & 0xffff0000u) * inv;
          const float x2 = __uint_as_float(b << 16) * inv, x3 = __uint_as_float(b & 0xffff0000u) * inv;
          if constexpr (HK == 2) {
            qop[g][i] = fp4::query_part4(x0, x1, x2, x3, r16 >= 8);
          } else {
            qop[0][i] = fp4::query_part4(x0, x1, x2, x3, false);
            qop[1][i] = fp4::query_part4(x0, x1, x2, x3, true);
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
    uint16_t* vst = vt_w + (lane / CPR) * VROW + (lane % CPR) * 8;                      // stores
    const uint16_t* vtr = vt_w + (jq * 4 + (r16 >> 2)) * VROW + 4 * (r16 & 3);          // transposed reads
    const float c = p.scale_log2;

    // Scores, online softmax and P V of a chunk whose first token is t0, of a sequence that ends at tok_end (as in
    // decode_body.h: the running max moves when the chunk's exceeds it by more than 8 in log2 units).
    auto compute = [&](const Chunk<HK>& T, int t0, int tok_end, auto&& between) {
      const bool full = T.ok[0] && T.ok[1] && t0 + kSteps * kTile <= tok_end;  // wave-uniform
      float x[kSteps * 4];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const f32x4 z = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 y;
        if constexpr (HK == 2) {
          const f32x4 y0 = fp4::mfma_scores16(T.k[s][0], T.ks[s][0], qop[0], qs[0], z);
          const f32x4 y1 = fp4::mfma_scores16(T.k[s][1], T.ks[s][1], qop[1], qs[1], z);
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // lane c keeps kv head c / 8 and adds the other part, in lane c ^ 8
            const float give = r16 < 8 ? y1[i] : y0[i], keep = r16 < 8 ? y0[i] : y1[i];
            y[i] = keep + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(give), 0x128, 0xF, 0xF, false));
          }
        } else {
          y = fp4::mfma_scores16(T.k[s][0], T.ks[s][0], qop[0], qs[0], z);
          y = fp4::mfma_scores16(T.k[s][0], T.ks[s][0], qop[1], qs[0], y);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[s * 4 + i] = full || (T.ok[s] && t0 + s * kTile + jq * 4 + i < tok_end) ? y[i] : -INFINITY;
      }
      // V into LDS as bf16. Groups that are not numbers stay out of the MFMAs (the zeros that keep the kv heads apart
      // would not hide them): the sequence's heads of that kv head are NaN in the group, which put() is told of.
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < HK; ++i) {
          const int tr = s * kTile + i * (64 / CPR);  // LDS row of the piece, less the lane's
          const uint32_t b = full || (T.ok[s] && t0 + tr + lane / CPR < tok_end) ? T.vs[s][i] : 0u;
          uint64_t bad = __builtin_amdgcn_ballot_w64(b == 255u);
          if (__builtin_expect(bad != 0, 0)) {
            bad |= bad >> 32;
            bad |= bad >> 16;
            bad |= bad >> 8;
            if (CPR == 4) bad |= bad >> 4;
            nan_groups |= (uint32_t)bad & ((1u << CPR) - 1u);
          }
          const float sc = fp4::scale_float(b == 255u ? 0u : b);
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<u32x4*>(vst + tr * VROW + q4 * CPR * 8) = fp4::values8(T.v[s][i][q4], sc);
        }
      wave_lds_sync();
      between();  // the chunk's registers are free: the next one's loads go out

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
      // P^T in bf16 (rounded by 2^-9, as the output is): k-slots 4 s + i = token 16 s + 4 jq + i
      u32x4 pv;
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
#pragma unroll
      for (int gk = 0; gk < HK; ++gk) {
        const u32x4 pb = HK == 1 || hg == gk ? pv : zero4();
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          const int col = HK == 2 ? (a >> 1) * 4 + gk * 2 + (a & 1) : a;  // the 16 LDS columns of accumulator a
          const s16x4 v0 = lds_read_tr16(vtr + col * 16);
          const s16x4 v1 = lds_read_tr16(vtr + kTile * VROW + col * 16);
          const u32x2 u0 = __builtin_bit_cast(u32x2, v0), u1 = __builtin_bit_cast(u32x2, v1);
          acc[a] = mfma_16x16x32(u32x4{u0[0], u0[1], u1[0], u1[1]}, pb, acc[a]);
        }
      }
      wave_lds_sync();
    };

    // ---- the ring: chunk registers T[u], refilled with the chunk kRing further on as soon as they are used
    Chunk<HK> T[kRing];
    u32x4 qv[HK][4];
    load_q(qv, k);
    int ki = k, ti = t_lo;  // the next chunk to load
    auto next = [&](Chunk<HK>& C) {
      const bool any = ti < t_hi;
      issue(C, any, ki, ti);
      if (any) {
        const int en = win.en(ki);
        ti += kSteps;
        if (ti >= en) {
          ti = en;
          if (ti < t_hi) ki = next_seg(ki);
        }
      }
    };
#pragma unroll
    for (int u = 0; u < kRing; ++u) next(T[u]);
    make_q(qv);
    int t = t_lo;
    bool more = true;
    while (more) {
#pragma unroll
      for (int u = 0; u < kRing; ++u) {
        if (!more) break;
        const int en = min(t_hi, win.en(k));
        const bool last = t + kSteps >= en;
        int kn = k;
        if (last && en < t_hi) {
          kn = next_seg(k);
          load_q(qv, kn);
        }
        compute(T[u], (t - win.st(k)) * kTile, win.ctx(k), [&]() { next(T[u]); });
        t = last ? en : t + kSteps;
        if (last) {
          const float l = col_sum4(lsum);
          if (__builtin_expect(nan_groups != 0, 0)) {
#pragma unroll
            for (int a = 0; a < 8; ++a)
              if ((nan_groups >> (hg * 4 + 2 * (a & 1) + (jq >> 1))) & 1u)
                acc[a] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
          }
          if (head_ok) put4(w + kc, head, jq, acc, m, l);
          more = en < t_hi;
          if (more) {
            m = -INFINITY;
            lsum = 0.f;
            nan_groups = 0;
#pragma unroll
            for (int a = 0; a < 8; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
            make_q(qv);
            k = kn;
            ++kc;
          }
        }
      }
    }
  }
};

}  // namespace dec

}  // namespace

}  // namespace vox
