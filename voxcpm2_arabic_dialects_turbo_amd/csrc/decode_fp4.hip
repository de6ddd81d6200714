// Paged decode attention over a 4-bit KV cache: decode_split (decode_body.h) with the walk of decode_fp4.h, then the
// merge of the sequences it cut (decode_merge_kernel: the partials are the bf16 cache's).
#include "decode_fp4.h"

namespace vox {

namespace {

using namespace dec;

constexpr int kThreadsFp4 = LdsFp4<1, true>::kNW * kWave;

template <int HK, bool BTL>
__global__ __launch_bounds__(kThreadsFp4) void decode_fp4_kernel(DecodeArgs p) {
  using LDS = LdsFp4<HK, BTL>;
  __shared__ __attribute__((aligned(16))) uint16_t s_vt[LDS::kNW * LDS::kVt];                  // per-wave V tiles (bf16)
  __shared__ __attribute__((aligned(16))) float s_slot[(LDS::kRoundSegs - 1) * kPartialFloats];  // segments' partials
  __shared__ int s_ctx[kMaxSeqPerLaunch];        // as in decode_kernel
  __shared__ int s_row[kMaxSeqPerLaunch];
  __shared__ int s_snew[kMaxSeqPerLaunch];
  __shared__ int s_start[kMaxSeqPerLaunch + 1];
  __shared__ int s_wtot[LDS::kNW];
  __shared__ int s_wmax[LDS::kNW];
  __shared__ __attribute__((aligned(16))) int s_bt[LDS::kBtInts];
  __shared__ int s_rtiles[kRecTiles];
  const LDS L{s_vt, s_slot, s_ctx, s_row, s_snew, s_start, s_wtot, s_wmax, s_bt, s_rtiles};
  decode_split<HK>(p, (int)blockIdx.x, (int)gridDim.x, L);
}

}  // namespace

hipError_t launch_decode_fp4(const DecodeArgs& a, int num_kv_heads, hipStream_t stream) {
  const dim3 grid((unsigned)a.grid);
  const bool btl = (int64_t)a.batch * a.max_blocks <= kBtLds;
  if (num_kv_heads == 1 && btl)
    decode_fp4_kernel<1, true><<<grid, dim3(kThreadsFp4), 0, stream>>>(a);
  else if (num_kv_heads == 1)
    decode_fp4_kernel<1, false><<<grid, dim3(kThreadsFp4), 0, stream>>>(a);
  else if (btl)
    decode_fp4_kernel<2, true><<<grid, dim3(kThreadsFp4), 0, stream>>>(a);
  else
    decode_fp4_kernel<2, false><<<grid, dim3(kThreadsFp4), 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  return launch_decode_merge_fp4(a, stream);
}

}  // namespace vox
