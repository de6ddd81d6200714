// Paged decode attention over a 4-bit KV cache: decode_split (decode_body.h) with the walk of decode_fp4.h, then the
// merge of the sequences it cut (decode_merge_kernel: the partials are the bf16 cache's).
#include "decode_fp4.h"

namespace vox {

namespace {

using namespace dec;

template <int HK, bool BTL, int NW, bool SCORES>
__global__ __launch_bounds__(NW * kWave) void decode_fp4_kernel(DecodeArgs p) {
  using LDS = LdsFp4<HK, BTL, NW, 6, SCORES>;
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
  decode_split<HK, LDS, SCORES>(p, (int)blockIdx.x, (int)gridDim.x, L);
}

// Four waves a workgroup where the tables reach at most 8192 steps, 32 a compute unit: a short share is start-up, the
// layout's scan and merges, and each costs less with half the waves. Beyond, eight keep the loads going (decode_fp4.h).
// 16 query heads of 2 kv heads, four | eight waves with the merge, streams x tokens (steps the tables reach): 1 x 420 (32)
// 11.2 | 11.9 us, 16 x 100-500 (512) 12.3 | 14.1, 64 x 500-1000 (4096) 15.8 | 18.1, 256 x 100-500 (8192) 18.9 | 20.3,
// 16 x 4000-8000 (7936) 19.4 | 19.2, 64 x 1500-2500 (10240) 21.3 | 20.7, 150 x 1500-2500 (24000) 30.5 | 27.5,
// 24 x 20000-32768 (49152) 47.5 | 38.4. The lengths are known on the device only. (A function of a plan's key: its record
// and its reader take the same.)
template <int HK, bool BTL, bool SCORES>
void launch_split(const DecodeArgs& a, hipStream_t stream) {
  constexpr int kShort = 8192;
  static_assert(kShort / (64 / kTile) <= kBtLds, "their block tables fit LDS");
  if (BTL && (int64_t)a.batch * a.max_blocks * (a.block_size / kTile) <= kShort)
    decode_fp4_kernel<HK, true, 4, SCORES><<<dim3((unsigned)a.grid), dim3(4 * kWave), 0, stream>>>(a);
  else
    decode_fp4_kernel<HK, BTL, 8, SCORES><<<dim3((unsigned)a.grid), dim3(8 * kWave), 0, stream>>>(a);
}

template <bool SCORES>
hipError_t launch_split(const DecodeArgs& a, int num_kv_heads, hipStream_t stream) {
  const bool btl = (int64_t)a.batch * a.max_blocks <= kBtLds;
  if (num_kv_heads == 1)
    btl ? launch_split<1, true, SCORES>(a, stream) : launch_split<1, false, SCORES>(a, stream);
  else
    btl ? launch_split<2, true, SCORES>(a, stream) : launch_split<2, false, SCORES>(a, stream);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_decode_fp4(const DecodeArgs& a, int num_kv_heads, hipStream_t stream) {
  const hipError_t e = launch_split<false>(a, num_kv_heads, stream);
  if (e != hipSuccess) return e;
  return launch_decode_merge_fp4(a, stream);
}

hipError_t launch_decode_weights_fp4(const DecodeArgs& a, int num_kv_heads, hipStream_t stream) {
  if (!a.scores || !a.weights) return hipErrorInvalidValue;
  const hipError_t e = launch_split<true>(a, num_kv_heads, stream);
  if (e != hipSuccess) return e;
  return launch_decode_merge_weights(a, true, stream);
}

}  // namespace vox
