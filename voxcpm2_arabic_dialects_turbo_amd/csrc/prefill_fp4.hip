// Varlen attention over a 4-bit KV cache through block tables: prompts that go on from cached prefixes, and steps that
// mix prompts with decode rows. Semantics as prefill_attn.hip's paged form: query i of a sequence with nq queries and nk
// keys sees keys j <= nk - nq + i (causal) or all nk; a row that sees no key gives zeros; keys of blocks outside the
// cache have no weight. The format is in fp4_common.h.
//
// A workgroup is four waves over 128 query rows (128 / G tokens x the G query heads of one kv head), a wave 32 of them,
// and walks 64-key tiles (a tile lies inside one block: block_size is a multiple of 64).
//  * S^T[64 keys x 32 rows] = K Q^T by 32x32x64 MFMAs on the codes as they are stored: a lane's 16 bytes are its
//    operand and have one scale, so K needs no conversion and no LDS; each wave loads the tile's 4 KB for itself (three
//    of the four from the CU's cache). The query is two fp8 parts, so the scores cost the MFMA time of bf16 ones.
//  * V is converted once a workgroup (a thread 32 channels of a key: 16 exact conversions) into a bf16 LDS tile, double
//    buffered, one barrier a tile. Column w * 4 + c of a row (16 bytes) holds piece w of the key's 32-channel group c, so
//    that the four lanes of a key write consecutive columns.
//  * O^T[128 x 32 rows] += V^T P^T by 32x32x16 MFMAs: P^T is in the B layout as the scores come, k-slot e of half h of
//    step s being key 16 s + 8 (e / 4) + 4 h + e % 4, and the transposed reads gather the same keys.
// The next tile's codes (20 registers a lane) are loaded while a tile is computed.
#include <climits>

#include "fp4_common.h"
#include "vox_kernels.h"

namespace vox {

namespace {

namespace pf4 {

constexpr int kD = 128;
constexpr int kRows = 128;  // query rows of a workgroup
constexpr int kBK = 64;     // keys of a tile
constexpr int kVRow = kD + 16;  // elements of an LDS row: the four rows a transposed read touches lie in other banks

struct TileRegs {
  u32x4 k[2][2];    // keys 32 rt + l % 32, channels 64 ks + 32 (l / 32) + [0, 32)
  uint32_t ks[2];   // their keys' four scales
  u32x4 v;          // key tid / 4, channels 32 (tid % 4) + [0, 32)
  uint32_t vs;      // their scale
  bool ok;          // the tile's block is mapped
};

__global__ __launch_bounds__(256, 2) void prefill_fp4_kernel(PrefillArgs p) {
  __shared__ __attribute__((aligned(16))) uint16_t s_v[2][kBK * kVRow];
  __shared__ __attribute__((aligned(4))) uint8_t s_nan[2][kBK * 4];  // a tile's groups whose scale is not a number: [key][32-channel group]
  __shared__ int s_nan_at[2];            // the first key of the last tile that held any
  const int b = blockIdx.y, g = blockIdx.z;
  const int q0 = p.cu_q[b], nq = p.cu_q[b + 1] - q0;
  const int HK = p.num_kv_heads;
  const int gsh = __builtin_ctz(p.group);  // the group divides 128: a power of two
  const int bq = kRows >> gsh;             // query tokens of a workgroup
  const int qt = (int)gridDim.x - 1 - (int)blockIdx.x;  // the last tile has the most keys: first
  if (qt * bq >= nq || (p.skip_single && nq == 1)) return;  // (workgroup-uniform)
  const int nk = max(0, min(p.cu_k[b + 1] - p.cu_k[b], p.max_blocks * p.block_size));

  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int col = lane & 31;
  const int h = lane >> 5;
  const int rho = w * 32 + col;
  const int tq = qt * bq + (rho >> gsh);
  const int head = (g << gsh) + (rho & (p.group - 1));
  const int64_t row = (int64_t)q0 + tq;
  const bool row_ok = tq < nq && row >= 0 && row < p.row_limit;
  const int tq_last = min(nq, (qt + 1) * bq) - 1;
  const int kv_end = p.causal ? min(nk, nk - nq + tq_last + 1) : nk;  // keys that some row of the workgroup sees
  const int limit = p.causal ? min(nk, nk - nq + tq + 1) : nk;        // keys that this lane's row sees
  const int all_see = p.causal ? nk - nq + qt * bq + 1 : nk;          // keys that every row sees

  const int64_t bb = fp4::block_bytes(p.block_size, HK);
  const int crow = HK * fp4::kHeadCodes, srow = HK * fp4::kHeadScales;
  const int scales = p.block_size * crow;
  const int32_t* bt = p.block_tables + (int64_t)b * p.bt_stride;
  auto issue = [&](TileRegs& T, int kv0) {
    const int blk = __builtin_amdgcn_readfirstlane(kv0 < kv_end ? bt[kv0 / p.block_size] : -1);
    T.ok = blk >= 0 && blk < p.num_blocks;
    const int tok = T.ok ? kv0 % p.block_size : 0;
    const int64_t at = T.ok ? blk * bb : 0;
    const int range = T.ok ? (int)bb : 0;
    const auto rk = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.k_cache) + at, (short)0, range,
                                                      fp4::kBufferWord3);
    const auto rv = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<uint16_t*>(p.v_cache) + at, (short)0, range,
                                                      fp4::kBufferWord3);
    const int c0 = tok * crow + g * fp4::kHeadCodes, s0 = scales + tok * srow + g * fp4::kHeadScales;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        T.k[rt][ks] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, (rt * 32 + col) * crow + ks * 32 + h * 16, c0, 0));
      T.ks[rt] = __builtin_amdgcn_raw_buffer_load_b32(rk, (rt * 32 + col) * srow, s0, 0);
    }
    T.v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, (tid >> 2) * crow + (tid & 3) * 16, c0, 0));
    T.vs = __builtin_amdgcn_raw_buffer_load_b8(rv, (tid >> 2) * srow + (tid & 3), s0, 0);
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
  TileRegs T0, T1;
  issue(T0, 0);
  issue(T1, kBK);

  // ---- the query in fp8 (fp4_common.h): operand ks holds channels 64 ks + 16 h + [0, 16) and 64 ks + 32 + 16 h + [0, 16)
  fp4::i32x8 qhi[2], qlo[2];
  uint32_t qs;
  {
    uint32_t mb = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mb = max(mb, fp4::max_bits(qv[i]));
    mb = __float_as_uint(xhalf_max(__uint_as_float(mb << 16))) >> 16;
    qs = fp4::query_scale_byte(mb);
    const float inv = fp4::query_inverse(qs);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = qv[ks * 4 + i / 2][(i & 1) * 2], c = qv[ks * 4 + i / 2][(i & 1) * 2 + 1];
        const float x0 = __uint_as_float(a << 16) * inv, x1 = __uint_as_float(a & 0xffff0000u) * inv;
        const float x2 = __uint_as_float(c << 16) * inv, x3 = __uint_as_float(c & 0xffff0000u) * inv;
        qhi[ks][i] = fp4::query_part4(x0, x1, x2, x3, false);
        qlo[ks][i] = fp4::query_part4(x0, x1, x2, x3, true);
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

  // Values that are not numbers stay out of the MFMAs, where a masked key's probability of 0 would not hide them: such a
  // group is zeros in LDS, and mark_nan finds the rows that see it (their outputs in the group are NaN).
  auto store_v = [&](const TileRegs& T, int kv0, int buf) {
    uint16_t* d = s_v[buf];
    const uint32_t b = T.ok && kv0 + (tid >> 2) < nk ? T.vs : 0u;
    const bool nan = b == 255u;
    s_nan[buf][tid] = nan;
    if (__builtin_amdgcn_ballot_w64(nan) != 0) s_nan_at[buf] = kv0;
    const float sc = fp4::scale_float(nan ? 0u : b);
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) *reinterpret_cast<u32x4*>(d + vst + q4 * 32) = fp4::values8(T.v[q4], sc);
  };
  uint32_t nan_groups = 0;  // byte c, bit 0: the row has seen such a key in group c
  auto mark_nan = [&](int buf, int seen) {  // seen: the tile's keys that this lane's row sees
#pragma unroll 1
    for (int j = 0; j < kBK; ++j) nan_groups |= j < seen ? reinterpret_cast<const uint32_t*>(s_nan[buf])[j] : 0u;
  };
  auto compute = [&](const TileRegs& T, int kv0, int buf, auto&& between) {
    const uint16_t* vt = s_v[buf];
    f32x16 s[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[rt][i] = 0.f;
      const uint32_t ksc = T.ks[rt] >> (8 * h);  // bytes 0 and 2: the scales of channels 32 h and 64 + 32 h on
      s[rt] = fp4::mfma_scores32<0>(T.k[rt][0], ksc, qhi[0], qs, s[rt]);
      s[rt] = fp4::mfma_scores32<2>(T.k[rt][1], ksc, qhi[1], qs, s[rt]);
      s[rt] = fp4::mfma_scores32<0>(T.k[rt][0], ksc, qlo[0], qs, s[rt]);
      s[rt] = fp4::mfma_scores32<2>(T.k[rt][1], ksc, qlo[1], qs, s[rt]);
    }
    const bool full = T.ok && kv0 + kBK <= min(all_see, nk);  // workgroup-uniform
    const int lim = T.ok ? limit - kv0 - 4 * h : INT_MIN;     // this half's keys below it are seen
    between();  // the tile's registers are free
    if (!full) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[rt][i] = rt * 32 + 8 * (i / 4) + i % 4 < lim ? s[rt][i] : -INFINITY;
    }
    float tm = s[0][0];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int i = 0; i < 16; ++i) tm = fmaxf(tm, s[rt][i]);
    tm = xhalf_max(tm) * c;
    const bool up = tm > m + 8.f;
    if (__builtin_amdgcn_ballot_w64(up) != 0) {
      const float alpha = up ? fast_exp2(m - tm) : 1.f;
      m = up ? tm : m;
      lsum *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.f : m;
    u32x4 pb[4];
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = (st & 1) * 8 + 2 * e;
        const float x0 = fast_exp2(fmaf(s[st >> 1][i], c, -mu)), x1 = fast_exp2(fmaf(s[st >> 1][i + 1], c, -mu));
        lsum += x0 + x1;
        pb[st][e] = pack_bf16x2(x0, x1);
      }
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        const u32x2 u0 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + vtr + (16 * st) * kVRow + dt * 32));
        const u32x2 u1 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + vtr + (16 * st + 8) * kVRow + dt * 32));
        acc[dt] = mfma_32x32x16(u32x4{u0[0], u0[1], u1[0], u1[1]}, pb[st], acc[dt]);
      }
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(s_nan_at[buf]) == kv0, 0)) mark_nan(buf, limit - kv0);
  };

  if (kv_end > 0) {
    if (tid < 2) s_nan_at[tid] = -1;
    __syncthreads();
    store_v(T0, 0, 0);
    __syncthreads();
    for (int kv0 = 0; kv0 < kv_end; kv0 += 2 * kBK) {
      compute(T0, kv0, 0, [&]() {
        store_v(T1, kv0 + kBK, 1);
        issue(T0, kv0 + 2 * kBK);
      });
      __syncthreads();
      if (kv0 + kBK >= kv_end) break;
      compute(T1, kv0 + kBK, 1, [&]() {
        store_v(T0, kv0 + 2 * kBK, 0);
        issue(T1, kv0 + 3 * kBK);
      });
      __syncthreads();
    }
  }

  const float l = xhalf_sum(lsum);
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);  // a row that sees no key: zeros
  if (!row_ok) return;
  uint16_t* ob = p.out + row * p.out_row_stride + (int64_t)head * kD + 4 * h;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // LDS column 32 dt + 8 i + 4 h + [0, 4): channels 32 i + 8 dt + 4 h + [0, 4)
      const float f = (nan_groups >> (8 * i)) & 1u ? __builtin_nanf("") : inv;
      *reinterpret_cast<u32x2*>(ob + i * 32 + dt * 8) =
          u32x2{pack_bf16x2(acc[dt][4 * i] * f, acc[dt][4 * i + 1] * f),
                pack_bf16x2(acc[dt][4 * i + 2] * f, acc[dt][4 * i + 3] * f)};
    }
}

}  // namespace pf4

}  // namespace

hipError_t launch_prefill_fp4(const PrefillArgs& a, int max_seqlen_q, hipStream_t stream) {
  const int bq = pf4::kRows / a.group;
  const dim3 grid((unsigned)((max_seqlen_q + bq - 1) / bq), (unsigned)a.batch, (unsigned)a.num_kv_heads);
  pf4::prefill_fp4_kernel<<<grid, dim3(256), 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace vox
