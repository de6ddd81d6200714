// What every key of a causal varlen call receives: for sequence b, kv head g and key j
//   got[g, j] = sum over b's queries i that see j and the query heads h of g of exp2(c q_ih . k_j - lse_ih),
// c the log2-scaled softmax scale, lse_ih = log2 sum_j exp2(c q_ih . k_j): the column sums of the attention's probabilities.
// Two launches. The attention (prefill_tile32.h) leaves every row's lse behind; then key_weights_kernel makes the scores
// again, a key block at a time over all queries that see it, which needs neither atomics nor partial sums in memory: every
// key's sum is one workgroup's, in a fixed order, fp32. A new key's weight is set, a cached one's grows.
//
// A workgroup is (KW x 32 keys, sequence, kv head), as KW x QW waves: wave (kw, qw) holds its 32 keys' K rows in registers
// (the A operand of the score MFMA) and takes the 32-row query tiles qw, qw + QW, ... from the first that sees its keys.
// Rows are (token, query head of g), so S^T[32 keys x 32 rows] has a row's scores in one lane column and its lse in one
// register; 16 fma, exp2 and adds a tile behind 8 MFMAs. The lanes' sums meet in LDS at the end.
#include "prefill_tile32.h"
#include "vox_common.h"
#include "vox_kernels.h"

namespace vox {

namespace {

constexpr int kKwD = 128;

template <int SRC, int RG, int KS>
__global__ __launch_bounds__(64 * RG * KS, 2) void prefill32_lse_kernel(PrefillArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t kt0[pf32::kTB];
  __shared__ __attribute__((aligned(1024))) uint8_t kt1[pf32::kTB];
  __shared__ __attribute__((aligned(1024))) uint8_t vt0[pf32::kTB];
  __shared__ __attribute__((aligned(1024))) uint8_t vt1[pf32::kTB];
  __shared__ float red[KS == 2 ? 256 : 1];
  const pf32::Bufs bufs{kt0, kt1, vt0, vt1, red};
  int qt, b, g;
  grid_item(p, qt, b, g);
  pf32::tile<SRC, RG, KS, true>(p, qt, b, g, bufs);
}

template <int KW, int QW>
__global__ __launch_bounds__(64 * KW * QW) void key_weights_kernel(KeyWeightsArgs k) {
  const PrefillArgs& p = k.a;
  __shared__ float sums[KW * QW][32][33];  // [wave][key][row column]
  const int b = blockIdx.y, g = blockIdx.z;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int kw = w % KW, qw = w / KW;
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int q0 = p.cu_q[b], nq = p.cu_q[b + 1] - q0;
  const int k0 = p.cu_k[b], nk = p.cu_k[b + 1] - k0;
  const int64_t row = k.rows ? (int64_t)k.rows[b] : b;
  const int first = (int)blockIdx.x * (32 * KW);  // the workgroup's first key
  if (nq <= 0 || first >= nk || first >= k.width || row < 0 || row >= k.row_count) return;

  // ---- this wave's keys: key j = jb + col, dims 16 s + 8 h + [0, 8) in kf[s]; keys that do not count read row 0
  const int jb = first + kw * 32, j = jb + col;
  const bool paged = p.block_tables != nullptr;
  const uint16_t* kr = nullptr;
  if (j < nk && !paged) {
    kr = p.k_src + ((int64_t)k0 + j) * p.k_row_stride + g * kKwD;
  } else if (j < nk && j < p.max_blocks * p.block_size) {
    const int bid = p.block_tables[(int64_t)b * p.bt_stride + j / p.block_size];
    if (bid >= 0 && bid < p.num_blocks)
      kr = p.k_cache + (((int64_t)bid * p.block_size + j % p.block_size) * p.num_kv_heads + g) * kKwD;
  }
  const uint32_t counts = (uint32_t)__builtin_amdgcn_ballot_w64(kr != nullptr);  // bit: key jb + bit takes weight
  u32x4 kf[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) kf[s] = kr ? ld_g16(kr + 16 * s + 8 * h) : zero4();

  // ---- the query tiles that see a key of the wave: token tq sees key j when j <= nk - nq + tq
  const int gsh = __builtin_ctz(p.group), n = nq << gsh;
  const int first_row = max(0, jb - (nk - nq)) << gsh;
  float acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  const float c = p.scale_log2;
  for (int r0 = (first_row & ~31) + 32 * qw; r0 < n; r0 += 32 * QW) {
    const int rho = r0 + col, tq = rho >> gsh, head = (g << gsh) + (rho & (p.group - 1));
    const bool ok = rho < n && (p.row_limit <= 0 || (int64_t)q0 + tq < p.row_limit);
    u32x4 qf[8];
    const uint16_t* qr = p.q + ((int64_t)q0 + (ok ? tq : 0)) * p.q_row_stride + head * kKwD + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[s] = ok ? ld_g16(qr + 16 * s) : zero4();
    const float lse = ok ? p.lse[((int64_t)q0 + tq) * p.num_heads + head] : INFINITY;
    f32x16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) sc = mfma_32x32x16(kf[s], qf[s], sc);
    // register i: key jb + 8 (i / 4) + 4 h + i % 4; the last key that the row sees, relative to jb + 4 h
    const int last = ok ? min(nk - 1, nk - nq + tq) - jb - 4 * h : -1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = fast_exp2(fmaf(sc[i], c, -lse));
      acc[i] += 8 * (i >> 2) + (i & 3) <= last ? e : 0.f;
    }
  }

  // ---- over the rows' lane columns and the workgroup's query waves
#pragma unroll
  for (int i = 0; i < 16; ++i) sums[w][8 * (i >> 2) + 4 * h + (i & 3)][col] = acc[i];
  __syncthreads();
  if (qw != 0 || lane >= 32) return;
  float got = 0.f;
  for (int x = 0; x < QW; ++x)
    for (int y = 0; y < 32; ++y) got += sums[kw + x * KW][col][y];
  if (j >= nk || j >= k.width) return;
  float* out = k.weights + (row * p.num_kv_heads + g) * k.width + j;
  got = (counts >> col) & 1u ? got : 0.f;
  *out = j >= nk - nq ? got : *out + got;
}

template <int RG, int KS>
hipError_t launch_lse(const PrefillArgs& a, dim3 grid, hipStream_t stream) {
  const dim3 block(64 * RG * KS);
  if (!a.block_tables)
    prefill32_lse_kernel<pf32::kRows, RG, KS><<<grid, block, 0, stream>>>(a);
  else
    prefill32_lse_kernel<pf32::kCache, RG, KS><<<grid, block, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_prefill_lse(const PrefillArgs& a0, int max_seqlen_q, hipStream_t stream) {
  if (max_seqlen_q <= 0 || a0.batch <= 0) return hipSuccess;
  if (!a0.lse || !a0.cu_q || !a0.cu_k || !a0.causal || (a0.block_tables && a0.block_size % pf32::kBK) || 128 % a0.group)
    return hipErrorInvalidValue;
  PrefillArgs a = a0;
  const bool small = 64 % a.group == 0;
  const int64_t tiles64 = small ? ((int64_t)max_seqlen_q + 64 / a.group - 1) / (64 / a.group) : 0;
  if (small && tiles64 * a.batch * a.num_kv_heads <= 512)
    return launch_lse<2, 2>(a, dim3((unsigned)tiles64, (unsigned)a.batch, (unsigned)a.num_kv_heads), stream);
  const int64_t tiles = ((int64_t)max_seqlen_q + 128 / a.group - 1) / (128 / a.group);
  a.xcd_order = tiles * a.batch * a.num_kv_heads >= 1024;
  return launch_lse<4, 1>(a, dim3((unsigned)tiles, (unsigned)a.batch, (unsigned)a.num_kv_heads), stream);
}

hipError_t launch_key_weights(const KeyWeightsArgs& k, int max_seqlen_k, hipStream_t stream) {
  if (max_seqlen_k <= 0 || k.a.batch <= 0) return hipSuccess;
  if (!k.a.lse || !k.weights || !k.a.cu_q || !k.a.cu_k) return hipErrorInvalidValue;
  constexpr int KW = 2, QW = 4;
  const dim3 grid((unsigned)((max_seqlen_k + 32 * KW - 1) / (32 * KW)), (unsigned)k.a.batch, (unsigned)k.a.num_kv_heads);
  key_weights_kernel<KW, QW><<<grid, dim3(64 * KW * QW), 0, stream>>>(k);
  return hipGetLastError();
}

}  // namespace vox
