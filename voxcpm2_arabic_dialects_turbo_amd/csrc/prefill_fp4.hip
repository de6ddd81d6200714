// Varlen attention over a 4-bit KV cache through block tables: prompts that go on from cached prefixes, and steps that
// mix prompts with decode rows. Semantics as prefill_attn.hip's paged form: query i of a sequence with nq queries and nk
// keys sees keys j <= nk - nq + i (causal) or all nk; a row that sees no key gives zeros; keys of blocks outside the
// cache have no weight. The format is in fp4_common.h.
//
// A workgroup is four waves over 128 query rows (128 / G tokens x the G query heads of one kv head), a wave 32 of them,
// and walks 64-key tiles (a tile lies inside one block: block_size is a multiple of 64).
//  * S^T[64 keys x 32 rows] = K Q^T by 32x32x64 MFMAs on the codes as they are stored: a lane's 16 bytes are its
//    operand and have one scale, so K needs no conversion. The query is two fp8 parts, so the scores cost the MFMA time of
//    bf16 ones.
//  * V is converted once a workgroup (a thread 32 channels of a key: 16 exact conversions) into a bf16 LDS tile, double
//    buffered, one barrier a tile. Column w * 4 + c of a row (16 bytes) holds piece w of the key's 32-channel group c, so
//    that the four lanes of a key write consecutive columns.
//  * O^T[128 x 32 rows] += V^T P^T by 32x32x16 MFMAs: P^T is in the B layout as the scores come, k-slot e of half h of
//    step s being key 16 s + 8 (e / 4) + 4 h + e % 4, and the transposed reads gather the same keys.
// A tile's codes (8.5 KB, K and V) go from memory straight into LDS, a quarter by each wave. A tile's softmax and P V run
// beside the next tile's scores and V conversion (step), while the codes of the tile after that are on their way.
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

// A tile's codes as they come from memory: 64 keys x 64 bytes, then the keys' four scales. Of K's 16-byte pieces piece p of
// key r lies in slot p ^ (r / 4 % 4): the eight lanes that an operand read serves at once then hit distinct banks.
constexpr int kCodes = kBK * fp4::kHeadCodes;
constexpr int kTileBytes = kCodes + kBK * fp4::kHeadScales;
typedef __attribute__((address_space(3))) void lds_void;
typedef u32x4 __attribute__((aligned(8))) u32x4_a8;  // output rows are 8-byte aligned

__global__ __launch_bounds__(256, 2) void prefill_fp4_kernel(PrefillArgs p) {
  __shared__ __attribute__((aligned(16))) uint16_t s_v[2][kBK * kVRow];
  // (distinct arrays: the compiler can tell a tile's reads from the next one's transfers in flight)
  __shared__ __attribute__((aligned(16))) uint8_t s_k0[kTileBytes], s_k1[kTileBytes], s_c0[kTileBytes], s_c1[kTileBytes];
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
  const int tq_last = min(nq, (qt + 1) * bq) - 1;
  const int kv_end = p.causal ? min(nk, nk - nq + tq_last + 1) : nk;  // keys that some row of the workgroup sees
  const int limit = p.causal ? min(nk, nk - nq + tq + 1) : nk;        // keys that this lane's row sees
  const int all_see = p.causal ? nk - nq + qt * bq + 1 : nk;          // keys that every row sees

  const int64_t bb = fp4::block_bytes(p.block_size, HK);
  const int crow = HK * fp4::kHeadCodes, srow = HK * fp4::kHeadScales;
  const int scales = p.block_size * crow;
  const int32_t* bt = p.block_tables + (int64_t)b * p.bt_stride;
  // The next tile's codes from memory into LDS (K's to kd, V's to vd), a quarter of them by each wave; whether its block is
  // mapped.
  const int key16 = tid >> 2;  // the key of the 16-byte slot that this lane fills
  const int kcode = key16 * crow + (((tid & 3) ^ ((key16 >> 2) & 3)) << 4), vcode = key16 * crow + ((tid & 3) << 4);
  const int word = lane * srow;
  // the next tile: its first key, block (read a tile ahead) and place in the block
  int next_kv = 0, next_col = 0, next_in = 0, next_blk = kv_end > 0 ? bt[0] : -1;
  auto issue = [&](uint8_t* kd, uint8_t* vd) -> bool {
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
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(kd + w * 1024), 16, kcode, c0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(vd + w * 1024), 16, vcode, c0, 0, 0);
    // (the scales by two waves each: the same words)
    if (w & 1)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(vd + kCodes), 4, word, s0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(kd + kCodes), 4, word, s0, 0, 0);
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
  bool ok0 = issue(s_k0, s_c0);

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

  // V of tile kv0 (in registers, `mapped`) into LDS buffer buf: the scale, then piece q4. Values that are not numbers stay
  // out of the MFMAs, where a masked key's probability of 0 would not hide them: such a group is zeros in LDS, and mark_nan
  // finds the rows that see it (their outputs in the group are NaN).
  u32x4 vcodes;
  float vscale = 0.f;
  auto scale_v = [&](const uint8_t* vd, int kv0, bool mapped, int buf) {
    vcodes = *reinterpret_cast<const u32x4*>(vd + tid * 16);
    const uint32_t b = mapped && kv0 + (tid >> 2) < nk ? (uint32_t)vd[kCodes + tid] : 0u;
    const bool nan = b == 255u;
    s_nan[buf][tid] = nan;
    if (__builtin_amdgcn_ballot_w64(nan) != 0) s_nan_at[buf] = kv0;
    vscale = fp4::scale_float(nan ? 0u : b);
  };
  auto piece_v = [&](int q4, int buf) {
    *reinterpret_cast<u32x4*>(s_v[buf] + vst + q4 * 32) = fp4::values8(vcodes[q4], vscale);
  };
  uint32_t nan_groups = 0;  // byte c, bit 0: the row has seen such a key in group c
  auto mark_nan = [&](int buf, int seen) {  // seen: the tile's keys that this lane's row sees
#pragma unroll 1
    for (int j = 0; j < kBK; ++j) nan_groups |= j < seen ? reinterpret_cast<const uint32_t*>(s_nan[buf])[j] : 0u;
  };
  // Score MFMA i of 8: channels 64 (i / 4) + [0, 64), the query's high or low parts (i / 2 % 2), key block i % 2. Its
  // operand is piece 2 (i / 4) + h of key 32 (i % 2) + col.
  u32x4 kf[2];
  uint32_t ksc[2];
  const int krow = col * fp4::kHeadCodes, kswz = (col >> 2) & 3;  // (32 keys on: the same swizzle)
  auto read_k = [&](const uint8_t* kd, int ks) {
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
      kf[rt] = *reinterpret_cast<const u32x4*>(kd + rt * 32 * fp4::kHeadCodes + krow + (((2 * ks + h) ^ kswz) << 4));
  };
  auto read_scales = [&](const uint8_t* kd) {  // bytes 0 and 2: the scales of channels 32 h and 64 + 32 h on
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
      ksc[rt] = *reinterpret_cast<const uint32_t*>(kd + kCodes + (rt * 32 + col) * 4) >> (8 * h);
  };
  auto score = [&](int i, f32x16 (&s)[2]) {
    const int rt = i & 1, ks = i >> 2;
    const fp4::i32x8 q = i & 2 ? qlo[ks] : qhi[ks];
    f32x16 z;
#pragma unroll
    for (int j = 0; j < 16; ++j) z[j] = 0.f;
    const f32x16 in = i < 2 ? z : s[rt];
    s[rt] = ks == 0 ? fp4::mfma_scores32<0>(kf[rt], ksc[rt], q, qs, in) : fp4::mfma_scores32<2>(kf[rt], ksc[rt], q, qs, in);
  };
  auto mask = [&](f32x16 (&s)[2], int kv0, bool mapped) -> bool {  // whether something was to be masked
    if (mapped && kv0 + kBK <= min(all_see, nk)) return false;  // workgroup-uniform
    const int lim = mapped ? limit - kv0 - 4 * h : INT_MIN;     // this half's keys below it are seen
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[rt][i] = rt * 32 + 8 * (i / 4) + i % 4 < lim ? s[rt][i] : -INFINITY;
    return true;
  };
  auto top_of = [&](const f32x16 (&s)[2]) {
    float t = s[0][0];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
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

  // One tile (kv0, its V in buffer buf; the next one's codes in kn, vn, the places kd, vd free): its softmax and P V beside the next tile's score MFMAs and V conversion, in this
  // order, pinned: an MFMA leaves the wave's issue slots free, for about 2.3 elements' fma, exp, add and half a cvt (a score
  // MFMA, 64 cycles) or 1.1 (a P V one, 32). Left to itself the compiler runs the MFMAs together and the softmax together.
  auto step = [&](int kv0, int buf, f32x16 (&s)[2], f32x16 (&sn)[2], const uint8_t* kn, const uint8_t* vn, uint8_t* kd,
                  uint8_t* vd, bool& okn, bool& okd) {
    const bool more = kv0 + kBK < kv_end;
    const int nan_at = s_nan_at[buf];
    const float mu = m == -INFINITY ? 0.f : m;
    u32x4 pb[4];
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
    const uint16_t* vt = s_v[buf] + vtr;
    u32x4 vf[4];
    auto read_v = [&](int i) {  // operand of P V MFMA i (16-key step i / 4, dims block i % 4)
      const u32x2 u0 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + (16 * (i >> 2)) * kVRow + (i & 3) * 32));
      const u32x2 u1 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + (16 * (i >> 2) + 8) * kVRow + (i & 3) * 32));
      vf[i & 3] = u32x4{u0[0], u0[1], u1[0], u1[1]};
    };
    if (more) {
      read_scales(kn);
      read_k(kn, 0);
      okd = issue(kd, vd);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        score(i, sn);
        if (i == 0) scale_v(vn, kv0 + kBK, okn, buf ^ 1);
        if (i == 3) read_k(kn, 1);
        if (i >= 2 && i <= 5) piece_v(i - 2, buf ^ 1);
        if (i >= 6) {
          read_v(2 * (i - 6));
          read_v(2 * (i - 6) + 1);
        }
#pragma unroll
        for (int x = i * 18 / 8; x < (i + 1) * 18 / 8; ++x) element(x);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) read_v(i);
#pragma unroll
      for (int x = 0; x < 18; ++x) element(x);
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      acc[i & 3] = mfma_32x32x16(vf[i & 3], pb[i >> 2], acc[i & 3]);
      if (i + 4 < 16) read_v(i + 4);
#pragma unroll
      for (int x = 18 + i * 14 / 12; x < 18 + (i + 1) * 14 / 12 && x < 32; ++x) element(x);
      if (i >= 12) {  // this lane's largest score of the next tile
#pragma unroll
        for (int x = 8 * (i - 12); x < 8 * (i - 11); ++x) top = fmaxf(top, sn[x >> 4][x & 15]);
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
    f32x16 sa[2], sb[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int i = 0; i < 16; ++i) sb[rt][i] = 0.f;  // (read by the last tile's step, which has no next one)
    if (tid < 2) s_nan_at[tid] = -1;
    tile_barrier();
    bool ok1 = issue(s_k1, s_c1);
    read_scales(s_k0);
    scale_v(s_c0, 0, ok0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i % 4 == 0) read_k(s_k0, i / 4);
      score(i, sa);
      if (i < 4) piece_v(i, 0);
    }
    mask(sa, 0, ok0);
    raise(top_of(sa));
    tile_barrier();
    for (int kv0 = 0;;) {
      step(kv0, 0, sa, sb, s_k1, s_c1, s_k0, s_c0, ok1, ok0);
      kv0 += kBK;
      if (kv0 >= kv_end) break;
      step(kv0, 1, sb, sa, s_k0, s_c0, s_k1, s_c1, ok0, ok1);
      kv0 += kBK;
      if (kv0 >= kv_end) break;
    }
  } else {
    wait_vmem_all();  // (no transfer into LDS outlives the workgroup)
  }

  const float l = xhalf_sum(lsum);
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);  // a row that sees no key: zeros
  // O through LDS (each wave in a part of its own of the V tiles, which are done with), so that a row leaves in 16-byte
  // pieces side by side: 8-byte stores straight from the accumulators, 32 rows apart, took a third of a short step's time
  // (44 x 33-59 tokens over 50 cached: 16.0 us, 11.2 up to here).
  constexpr int kORow = kD + 8;
  static_assert(4 * 32 * kORow <= 2 * kBK * kVRow, "four waves' rows fit the V tiles");
  __syncthreads();
  uint16_t* const so = s_v[0] + w * 32 * kORow;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // LDS column 32 dt + 8 i + 4 h + [0, 4): channels 32 i + 8 dt + 4 h + [0, 4)
      const float f = (nan_groups >> (8 * i)) & 1u ? __builtin_nanf("") : inv;
      *reinterpret_cast<u32x2*>(so + col * kORow + i * 32 + dt * 8 + 4 * h) =
          u32x2{pack_bf16x2(acc[dt][4 * i] * f, acc[dt][4 * i + 1] * f),
                pack_bf16x2(acc[dt][4 * i + 2] * f, acc[dt][4 * i + 3] * f)};
    }
  wave_lds_sync();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 4);
    const int orho = w * 32 + r;
    const int otq = qt * bq + (orho >> gsh);
    const int64_t orow = (int64_t)q0 + otq;
    const u32x4 x = *reinterpret_cast<const u32x4*>(so + r * kORow + (lane & 15) * 8);
    if (otq < nq && orow >= 0 && orow < p.row_limit)
      *reinterpret_cast<u32x4_a8*>(p.out + orow * p.out_row_stride + (int64_t)((g << gsh) + (orho & (p.group - 1))) * kD +
                                   (lane & 15) * 8) = x;
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
