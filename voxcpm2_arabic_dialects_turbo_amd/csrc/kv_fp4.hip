// Rows of a 4-bit KV cache: quantised into their slots (store) and read back as bf16 (load). The format and the layout of
// a block are in fp4_common.h.
//
// store: for every token i whose slot s = slot_mapping[i] lies in [0, num_slots), its key row (HK heads of 128 bf16, rows
// key_row_stride apart) becomes 64 bytes of codes and 4 scales a head at slot s, and likewise the value row; other slots
// (-1: a padded row) store nothing. The scale is a power of two, so x / scale is exact and the codes depend on nothing
// but the rule in scale_byte and one rounding.
//
// A thread takes 8 channels: one 16-byte load, so a wave reads 1 KB runs; the four lanes of a 32-channel group agree on
// the largest magnitude by two DPP steps and each writes 4 bytes of codes (the lane that starts the group also its
// scale). Flattened over (token, K / V, piece); bound by the launch at a step's rows and by HBM beyond: 512 HK bytes
// read and 136 HK written a token. 8 rows of 2 kv heads: 2.0 us to store, 2.0 to load; 60001 rows (78 MB each way): 19.0 us
// (4.1 TB/s) and 17.3 us (4.5 TB/s).
#include "fp4_common.h"
#include "vox_kernels.h"

namespace vox {

namespace {

constexpr int kThreadsKv = 256;

template <bool VEC16>
__global__ __launch_bounds__(kThreadsKv) void store_fp4_kernel(Fp4RowsArgs a) {
  const int pieces = a.num_kv_heads * (fp4::kD / 8);  // of a token's key (or value) row
  const int64_t total = a.num_tokens * 2 * pieces;
  for (int64_t idx = (int64_t)blockIdx.x * kThreadsKv + threadIdx.x; idx < total;
       idx += (int64_t)gridDim.x * kThreadsKv) {
    const int64_t tok = idx / (2 * pieces);
    const int rem = (int)(idx - tok * 2 * pieces);
    const bool is_v = rem >= pieces;
    const int piece = is_v ? rem - pieces : rem;
    const uint16_t* src = (is_v ? a.value + tok * a.value_row_stride : a.key + tok * a.key_row_stride) + piece * 8;
    u32x4 x;
    if constexpr (VEC16) {
      x = ld_g16(src);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (uint32_t)src[2 * i] | ((uint32_t)src[2 * i + 1] << 16);
    }
    const int64_t slot = a.slots[tok];
    // (the four lanes of the group: total is a multiple of 4, so they leave the loop together)
    uint32_t codes, b;
    fp4::quantise8(x, codes, b);
    if (slot < 0 || slot >= a.num_slots) continue;
    const int64_t blk = slot / a.block_size;
    const int64_t in = slot - blk * a.block_size;
    uint8_t* base = (is_v ? a.v_cache : a.k_cache) + blk * fp4::block_bytes(a.block_size, a.num_kv_heads);
    *reinterpret_cast<uint32_t*>(base + in * a.num_kv_heads * fp4::kHeadCodes + piece * 4) = codes;
    if ((piece & 3) == 0)
      base[((int64_t)a.block_size * fp4::kHeadCodes + in * fp4::kHeadScales) * a.num_kv_heads + (piece >> 2)] = (uint8_t)b;
  }
}

// Row i of key / value (contiguous [num_tokens, HK, 128] bf16) = the values held at slots[i]; zeros where it is outside
// the cache. Exact. A thread makes 8 channels from 4 bytes of codes and their scale.
__global__ __launch_bounds__(kThreadsKv) void load_fp4_kernel(Fp4RowsArgs a) {
  const int pieces = a.num_kv_heads * (fp4::kD / 8);
  const int64_t total = a.num_tokens * 2 * pieces;
  for (int64_t idx = (int64_t)blockIdx.x * kThreadsKv + threadIdx.x; idx < total;
       idx += (int64_t)gridDim.x * kThreadsKv) {
    const int64_t tok = idx / (2 * pieces);
    const int rem = (int)(idx - tok * 2 * pieces);
    const bool is_v = rem >= pieces;
    const int piece = is_v ? rem - pieces : rem;
    const int64_t slot = a.slots[tok];
    u32x4 x = zero4();
    if (slot >= 0 && slot < a.num_slots) {
      const int64_t blk = slot / a.block_size;
      const int64_t in = slot - blk * a.block_size;
      const uint8_t* base = (is_v ? a.v_cache : a.k_cache) + blk * fp4::block_bytes(a.block_size, a.num_kv_heads);
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(base + in * a.num_kv_heads * fp4::kHeadCodes + piece * 4);
      const uint32_t b =
          base[((int64_t)a.block_size * fp4::kHeadCodes + in * fp4::kHeadScales) * a.num_kv_heads + (piece >> 2)];
      x = fp4::values8(codes, fp4::scale_float(b));
    }
    uint16_t* dst = const_cast<uint16_t*>(is_v ? a.value : a.key) + tok * (int64_t)a.num_kv_heads * fp4::kD + piece * 8;
    *reinterpret_cast<u32x4*>(dst) = x;
  }
}

unsigned grid_of(const Fp4RowsArgs& a) {
  const int64_t total = a.num_tokens * 2 * a.num_kv_heads * (fp4::kD / 8);
  const int64_t blocks = (total + kThreadsKv - 1) / kThreadsKv;
  return (unsigned)(blocks < 65536 ? blocks : 65536);  // the loop covers the rest
}

}  // namespace

hipError_t launch_store_fp4(const Fp4RowsArgs& a, bool vec16, hipStream_t stream) {
  if (a.num_tokens == 0) return hipSuccess;
  if (vec16)
    store_fp4_kernel<true><<<dim3(grid_of(a)), dim3(kThreadsKv), 0, stream>>>(a);
  else
    store_fp4_kernel<false><<<dim3(grid_of(a)), dim3(kThreadsKv), 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_load_fp4(const Fp4RowsArgs& a, hipStream_t stream) {
  if (a.num_tokens == 0) return hipSuccess;
  load_fp4_kernel<<<dim3(grid_of(a)), dim3(kThreadsKv), 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace vox
