// C-ABI entry points of libvoxattn.so (declared in include/vox_attn.h).
//
// Every entry point validates its arguments on the host, launches on the caller's stream, checks the launch, and
// returns a status (VOX_OK, VOX_EINVAL, VOX_EHIP) instead of throwing; vox_last_error() gives the calling thread's
// message for the last failure. Nothing here allocates, frees or synchronizes, so every call can be captured into
// a HIP graph.
#include <cfloat>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "vox_kernels.h"
#include "../../include/vox_attn.h"

namespace {

thread_local char g_err[512] = "";
int g_decode_grid_override = 0;

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int hip_status(hipError_t e, const char* what) {
  if (e == hipSuccess) return VOX_OK;
  return fail(VOX_EHIP, "%s: %s", what, hipGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }


constexpr int kHeadDim = 128;
constexpr int kMaxHeads = 16;

}  // namespace

extern "C" {

const char* vox_last_error(void) { return g_err; }

int vox_abi_version(void) { return VOX_ABI_VERSION; }

int vox_store_kvcache(const void* key, const void* value, int64_t key_row_stride, int64_t value_row_stride,
                      void* k_cache, void* v_cache, int64_t num_slots, const int32_t* slot_mapping,
                      int64_t num_tokens, int num_kv_heads, int head_dim, void* stream) {
  if (num_tokens < 0) return fail(VOX_EINVAL, "store_kvcache: num_tokens %lld < 0", (long long)num_tokens);
  if (num_tokens == 0) return VOX_OK;
  if (!key || !value || !k_cache || !v_cache || !slot_mapping)
    return fail(VOX_EINVAL, "store_kvcache: null pointer argument");
  if (num_kv_heads <= 0 || head_dim <= 0) return fail(VOX_EINVAL, "store_kvcache: bad head shape");
  if (num_slots <= 0) return fail(VOX_EINVAL, "store_kvcache: empty cache");
  const int row = num_kv_heads * head_dim;
  if (key_row_stride < row || value_row_stride < row)
    return fail(VOX_EINVAL, "store_kvcache: row stride smaller than num_kv_heads * head_dim");
  const bool vec16 = (row % 8 == 0) && (key_row_stride % 8 == 0) && (value_row_stride % 8 == 0) &&
                     aligned16(key) && aligned16(value) && aligned16(k_cache) && aligned16(v_cache);
  return hip_status(vox::launch_store_kvcache(key, value, key_row_stride, value_row_stride, k_cache, v_cache,
                                              num_slots, slot_mapping, num_tokens, row, vec16,
                                              (hipStream_t)stream),
                    "store_kvcache launch");
}

int vox_decode_workgroups(void) {
  if (g_decode_grid_override > 0) return g_decode_grid_override;
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) {
    (void)hipGetLastError();
    cus = 256;  // MI355X
  }
  return cus;  // one 4-wave workgroup per CU: the split kernel's ranges are balanced over every CU
}

void vox_set_decode_workgroups(int workgroups) { g_decode_grid_override = workgroups > 0 ? workgroups : 0; }

namespace {
// Workspace of decode launches of up to `slice` sequences over `grid` workgroups, each part 256-byte aligned: the fp32
// split-KV partials [slice + grid][kPartialFloats], the int32 step layout [slice + 2] (first step of every sequence,
// the total, the active workgroup count) that the merge kernel reads, then the plan records [grid][kPlanRecInts].
struct DecodeWorkspace {
  size_t partials, steps, plan, total;
};
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
DecodeWorkspace decode_workspace(int slice, int grid) {
  DecodeWorkspace w;
  w.partials = 0;
  w.steps = round256((size_t)(slice + grid) * vox::kPartialFloats * 4);
  w.plan = w.steps + round256((size_t)(slice + 2) * 4);
  w.total = w.plan + round256((size_t)grid * vox::kPlanRecInts * 4);
  return w;
}
}  // namespace

size_t vox_decode_workspace_bytes(int batch) {
  if (batch <= 0) return 0;
  const int slice = batch < vox::kMaxSeqPerLaunch ? batch : vox::kMaxSeqPerLaunch;
  return decode_workspace(slice, vox_decode_workgroups()).total;
}

}  // extern "C"

namespace {
// Launches the decode kernel over `batch` sequences in slices of kMaxSeqPerLaunch (each slice's step layout lives
// in LDS), all sharing the workspace; `a` describes the whole batch. A call of several slices runs unplanned (the
// workspace holds one plan).
// a's split-KV scratch and plan records in the workspace, for launches of up to `slice` sequences
vox::DecodeArgs with_workspace(const vox::DecodeArgs& a, int slice, int plan_mode, void* workspace) {
  const DecodeWorkspace ws = decode_workspace(slice, a.grid);
  vox::DecodeArgs d = a;
  d.partials = (float*)((char*)workspace + ws.partials);
  d.steps = (int32_t*)((char*)workspace + ws.steps);
  d.plan = (int32_t*)((char*)workspace + ws.plan);
  d.plan_mode = plan_mode;
  return d;
}

int launch_decode_slices(const vox::DecodeArgs& a, int batch, int num_kv_heads, int plan, void* workspace,
                         hipStream_t stream,
                         hipError_t (*launch)(const vox::DecodeArgs&, int, hipStream_t) = vox::launch_decode) {
  const int slice_max = batch < vox::kMaxSeqPerLaunch ? batch : vox::kMaxSeqPerLaunch;
  const vox::DecodeArgs base =
      with_workspace(a, slice_max, batch <= vox::kMaxSeqPerLaunch ? plan : vox::kPlanNone, workspace);
  for (int b0 = 0; b0 < batch; b0 += vox::kMaxSeqPerLaunch) {
    vox::DecodeArgs s = base;
    s.batch = batch - b0 < vox::kMaxSeqPerLaunch ? batch - b0 : vox::kMaxSeqPerLaunch;
    s.block_tables = base.block_tables + (int64_t)b0 * base.bt_stride;
    if (base.weight_rows) s.weight_rows = base.weight_rows + b0;
    s.weight_row0 = base.weight_row0 + b0;
    if (base.cu_q) {  // varlen: rows are absolute (cu_seqlens_q), only the sequence arrays move
      s.cu_q = base.cu_q + b0;
      s.cu_k = base.cu_k + b0;
    } else {
      s.q = base.q + (int64_t)b0 * base.q_row_stride;
      s.context_lens = base.context_lens + b0;
      s.out = base.out + (int64_t)b0 * base.out_row_stride;
      if (base.slot_mapping) {
        s.slot_mapping = base.slot_mapping + b0;
        s.new_k = base.new_k + (int64_t)b0 * base.new_k_stride;
        s.new_v = base.new_v + (int64_t)b0 * base.new_v_stride;
      }
    }
    const int st = hip_status(launch(s, num_kv_heads, stream), "decode launch");
    if (st != VOX_OK) return st;
  }
  return VOX_OK;
}
}  // namespace

extern "C" {

}  // extern "C"

namespace {
// Validates a decode call's arguments (batch > 0) and fills its launch descriptor.
int decode_setup(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache, int64_t num_blocks,
                 int block_size, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                 const int32_t* context_lens, int batch, int num_heads, int num_kv_heads, int head_dim,
                 float softmax_scale, void* workspace, size_t workspace_bytes, void* out, vox::DecodeArgs* out_args) {
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out)
    return fail(VOX_EINVAL, "decode_attn: null pointer argument");
  if (head_dim != kHeadDim) return fail(VOX_EINVAL, "decode_attn: head_dim %d unsupported (128 only)", head_dim);
  if (num_kv_heads != 1 && num_kv_heads != 2)
    return fail(VOX_EINVAL, "decode_attn: num_kv_heads %d unsupported (1 or 2)", num_kv_heads);
  if (num_heads <= 0 || num_heads > kMaxHeads || num_heads % num_kv_heads)
    return fail(VOX_EINVAL, "decode_attn: num_heads %d must be <= 16 and a multiple of num_kv_heads", num_heads);
  if (block_size <= 0 || block_size % 32)
    return fail(VOX_EINVAL, "decode_attn: block_size %d must be a positive multiple of 32", block_size);
  if (max_blocks <= 0 || bt_stride < max_blocks) return fail(VOX_EINVAL, "decode_attn: bad block table shape");
  if (num_blocks <= 0) return fail(VOX_EINVAL, "decode_attn: empty cache");
  if (q_row_stride < (int64_t)num_heads * head_dim || q_row_stride % 8)
    return fail(VOX_EINVAL, "decode_attn: q row stride %lld", (long long)q_row_stride);
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || !aligned16(workspace))
    return fail(VOX_EINVAL, "decode_attn: q, caches, out and workspace must be 16-byte aligned");
  if (!std::isfinite(softmax_scale)) return fail(VOX_EINVAL, "decode_attn: softmax_scale is not finite");
  if ((int64_t)max_blocks * block_size > (1 << 30)) return fail(VOX_EINVAL, "decode_attn: block table too wide");
  const int grid = vox_decode_workgroups();
  const size_t need = vox_decode_workspace_bytes(batch);
  if (workspace_bytes < need || !workspace)
    return fail(VOX_EINVAL, "decode_attn: workspace of %zu bytes, %zu needed", workspace_bytes, need);

  vox::DecodeArgs& a = *out_args;
  a = vox::DecodeArgs{};
  a.q = (const uint16_t*)q;
  a.q_row_stride = q_row_stride;
  a.k_cache = (const uint16_t*)k_cache;
  a.v_cache = (const uint16_t*)v_cache;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks;
  a.context_lens = context_lens;
  a.batch = batch;
  a.num_heads = num_heads;
  a.group = num_heads / num_kv_heads;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.grid = grid;
  a.out = (uint16_t*)out;
  a.out_row_stride = (int64_t)num_heads * head_dim;
  return VOX_OK;
}
}  // namespace

extern "C" {

int vox_decode_attn(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                    int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                    int max_blocks, const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                    int head_dim, float softmax_scale, int plan, void* workspace, size_t workspace_bytes,
                    void* out, void* stream) {
  if (batch < 0) return fail(VOX_EINVAL, "decode_attn: batch < 0");
  if (plan != VOX_PLAN_NONE && plan != VOX_PLAN_RECORD && plan != VOX_PLAN_REUSE)
    return fail(VOX_EINVAL, "decode_attn: plan mode %d", plan);
  if (batch == 0) return VOX_OK;
  vox::DecodeArgs a;
  const int st = decode_setup(q, q_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride,
                              max_blocks, context_lens, batch, num_heads, num_kv_heads, head_dim, softmax_scale,
                              workspace, workspace_bytes, out, &a);
  if (st != VOX_OK) return st;
  // batches beyond one launch's LDS step layout run as consecutive launches on the stream (shared workspace)
  return launch_decode_slices(a, batch, num_kv_heads, plan, workspace, (hipStream_t)stream);
}

int vox_decode_attn_store(const void* q, int64_t q_row_stride, const void* key, const void* value,
                          int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                          void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                          const int32_t* block_tables, int64_t bt_stride, int max_blocks, const int32_t* context_lens,
                          int batch, int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int plan,
                          void* workspace, size_t workspace_bytes, void* out, void* stream) {
  if (batch < 0) return fail(VOX_EINVAL, "decode_attn_store: batch < 0");
  if (plan != VOX_PLAN_NONE && plan != VOX_PLAN_RECORD && plan != VOX_PLAN_REUSE)
    return fail(VOX_EINVAL, "decode_attn_store: plan mode %d", plan);
  if (batch == 0) return VOX_OK;
  if (!key || !value || !slot_mapping) return fail(VOX_EINVAL, "decode_attn_store: null key, value or slot_mapping");
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key_row_stride < row || value_row_stride < row || key_row_stride % 8 || value_row_stride % 8 ||
      !aligned16(key) || !aligned16(value))
    return fail(VOX_EINVAL, "decode_attn_store: key / value rows must be 16-byte aligned, strides multiples of 8 "
                            "elements and at least num_kv_heads * head_dim");
  vox::DecodeArgs a;
  const int st = decode_setup(q, q_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride,
                              max_blocks, context_lens, batch, num_heads, num_kv_heads, head_dim, softmax_scale,
                              workspace, workspace_bytes, out, &a);
  if (st != VOX_OK) return st;
  a.slot_mapping = slot_mapping;
  a.new_k = (const uint16_t*)key;
  a.new_v = (const uint16_t*)value;
  a.new_k_stride = key_row_stride;
  a.new_v_stride = value_row_stride;
  return launch_decode_slices(a, batch, num_kv_heads, plan, workspace, (hipStream_t)stream);
}

size_t vox_prefill_workspace_bytes(int batch) { return vox_decode_workspace_bytes(batch); }

}  // extern "C"

// ---- allocation-free decode: the split-KV scratch in a static device array ----------------------------------------
//
// vox_decode_attn_noalloc serves callers that cannot allocate (code under HIP graph capture that must not touch an
// allocator, tight serving loops): the workspace vox_decode_attn takes as an argument lives in `scratch`, a
// file-scope device array that every GPU the library runs on holds until the process ends. In host code `scratch`
// names a host-side stand-in, not the device array: its device address on each GPU comes from hipGetSymbolAddress,
// looked up once per device with that device current, and only that address is handed to kernels.
namespace {
constexpr int kMaxDevices = 64;
constexpr size_t kScratchBytes = size_t(16) << 20;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];
void* g_scratch_ptr[kMaxDevices] = {};
std::mutex g_scratch_mu;

// This device's address of `scratch` (nullptr and an error message on failure).
void* scratch_on_current_device() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    (void)hipGetLastError();
    fail(VOX_EHIP, "decode_attn_noalloc: no current device");
    return nullptr;
  }
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* ptr = nullptr;
    const hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !ptr) {
      (void)hipGetLastError();
      fail(VOX_EHIP, "decode_attn_noalloc: hipGetSymbolAddress(scratch): %s", hipGetErrorString(e));
      return nullptr;
    }
    g_scratch_ptr[dev] = ptr;
  }
  return g_scratch_ptr[dev];
}
}  // namespace

extern "C" {

int vox_decode_attn_noalloc(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                            int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                            int max_blocks, const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                            int head_dim, float softmax_scale, void* out, void* stream) {
  if (batch < 0) return fail(VOX_EINVAL, "decode_attn_noalloc: batch < 0");
  if (batch == 0) return VOX_OK;
  const size_t need = vox_decode_workspace_bytes(batch);
  if (need > kScratchBytes)
    return fail(VOX_EINVAL, "decode_attn_noalloc: needs %zu bytes of scratch, the static array holds %zu", need,
                kScratchBytes);
  void* ws = scratch_on_current_device();
  if (!ws) return VOX_EHIP;
  return vox_decode_attn(q, q_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride,
                         max_blocks, context_lens, batch, num_heads, num_kv_heads, head_dim, softmax_scale,
                         VOX_PLAN_NONE, ws, kScratchBytes, out, stream);
}

}  // extern "C"

namespace {
// Validates a prefill call's shared arguments (all but the output) and fills its launch descriptor.
int prefill_setup(const char* fn, const void* q, int64_t q_row_stride, const void* key, const void* value,
                  int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                  int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                  const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                  int uniform_seqlen_q, int uniform_seqlen_k, int num_heads, int num_kv_heads, int head_dim,
                  float softmax_scale, int causal, vox::PrefillArgs* a) {
  if (!q) return fail(VOX_EINVAL, "%s: null q", fn);
  if (head_dim != kHeadDim) return fail(VOX_EINVAL, "%s: head_dim %d unsupported (128 only)", fn, head_dim);
  if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads)
    return fail(VOX_EINVAL, "%s: num_heads %d not a multiple of num_kv_heads %d", fn, num_heads, num_kv_heads);
  const int group = num_heads / num_kv_heads;
  if (128 % group) return fail(VOX_EINVAL, "%s: group size %d must divide 128", fn, group);
  if ((cu_seqlens_q == nullptr) != (cu_seqlens_k == nullptr))
    return fail(VOX_EINVAL, "%s: give both cu_seqlens or neither", fn);
  if (!cu_seqlens_q && (uniform_seqlen_q <= 0 || uniform_seqlen_k <= 0))
    return fail(VOX_EINVAL, "%s: uniform lengths must be positive without cu_seqlens", fn);
  if (!cu_seqlens_q && max_seqlen_q != uniform_seqlen_q)
    return fail(VOX_EINVAL, "%s: max_seqlen_q must equal the uniform length", fn);
  if (q_row_stride < (int64_t)num_heads * head_dim || q_row_stride % 8 || !aligned16(q))
    return fail(VOX_EINVAL, "%s: q must be 16-byte aligned with a row stride >= H*D, multiple of 8", fn);
  if (!std::isfinite(softmax_scale)) return fail(VOX_EINVAL, "%s: softmax_scale is not finite", fn);
  if (block_tables) {
    if (!k_cache || !v_cache) return fail(VOX_EINVAL, "%s: block tables without caches", fn);
    if (block_size <= 0 || max_blocks <= 0 || bt_stride < max_blocks || num_blocks <= 0)
      return fail(VOX_EINVAL, "%s: bad block table or cache shape", fn);
    if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(VOX_EINVAL, "%s: caches not aligned", fn);
  } else {
    if (!key || !value) return fail(VOX_EINVAL, "%s: null key/value without block tables", fn);
    if (key_row_stride < (int64_t)num_kv_heads * head_dim || value_row_stride < (int64_t)num_kv_heads * head_dim ||
        key_row_stride % 8 || value_row_stride % 8 || !aligned16(key) || !aligned16(value))
      return fail(VOX_EINVAL, "%s: key/value must be 16-byte aligned rows, stride multiple of 8", fn);
    if (key_row_stride >= (1 << 24) || value_row_stride >= (1 << 24))
      return fail(VOX_EINVAL, "%s: key/value row stride must be below 2^24 elements", fn);
  }
  *a = vox::PrefillArgs{};
  a->q = (const uint16_t*)q;
  a->q_row_stride = q_row_stride;
  a->k_src = (const uint16_t*)key;
  a->v_src = (const uint16_t*)value;
  a->k_row_stride = key_row_stride;
  a->v_row_stride = value_row_stride;
  a->k_cache = (const uint16_t*)k_cache;
  a->v_cache = (const uint16_t*)v_cache;
  a->num_blocks = num_blocks;
  a->block_size = block_size;
  a->block_tables = block_tables;
  a->bt_stride = bt_stride;
  a->max_blocks = max_blocks;
  a->cu_q = cu_seqlens_q;
  a->cu_k = cu_seqlens_k;
  a->uniform_q = uniform_seqlen_q;
  a->uniform_k = uniform_seqlen_k;
  a->batch = batch;
  a->num_heads = num_heads;
  a->num_kv_heads = num_kv_heads;
  a->group = group;
  a->scale_log2 = softmax_scale * 1.4426950408889634f;
  a->causal = causal ? 1 : 0;
  return VOX_OK;
}

// Whether a varlen call's one-query rows can run on the split-KV decode kernels (paged keys, cu_seqlens, the
// decode kernels' head and block shapes, an output the merge kernel can write with 16-byte stores, the workspace).
bool varlen_decode_rows(const vox::PrefillArgs& a, const void* workspace, int num_kv_heads) {
  return workspace && a.block_tables && a.cu_q && a.num_heads <= kMaxHeads && (num_kv_heads == 1 || num_kv_heads == 2) &&
         a.block_size % 32 == 0 && (int64_t)a.max_blocks * a.block_size <= (1 << 30) && a.out_row_stride % 8 == 0 &&
         ((uintptr_t)a.out & 15u) == 0;
}
int check_varlen_workspace(const char* fn, int batch, int plan, const void* workspace, size_t workspace_bytes) {
  const size_t need = vox_prefill_workspace_bytes(batch);
  if (workspace_bytes < need || !aligned16(workspace))
    return fail(VOX_EINVAL, "%s: workspace of %zu bytes (16-byte aligned), %zu needed", fn, workspace_bytes, need);
  if (plan != VOX_PLAN_NONE && plan != VOX_PLAN_RECORD && plan != VOX_PLAN_REUSE)
    return fail(VOX_EINVAL, "%s: plan mode %d", fn, plan);
  return VOX_OK;
}
// the decode kernels' arguments for the one-query rows of the paged varlen call a (varlen mode: rows from cu_seqlens)
vox::DecodeArgs varlen_decode_args(const vox::PrefillArgs& a, int64_t q_row_stride, int64_t num_blocks, int num_heads,
                                   int num_kv_heads) {
  vox::DecodeArgs d{};
  d.q = a.q;
  d.q_row_stride = q_row_stride;
  d.k_cache = a.k_cache;
  d.v_cache = a.v_cache;
  d.num_blocks = num_blocks;
  d.block_size = a.block_size;
  d.block_tables = a.block_tables;
  d.bt_stride = a.bt_stride;
  d.max_blocks = a.max_blocks;
  d.batch = a.batch;
  d.num_heads = num_heads;
  d.group = num_heads / num_kv_heads;
  d.scale_log2 = a.scale_log2;
  d.grid = vox_decode_workgroups();
  d.out = a.out;
  d.out_row_stride = a.out_row_stride;
  d.cu_q = a.cu_q;
  d.cu_k = a.cu_k;
  return d;
}
}  // namespace

extern "C" {

int vox_prefill_attn(const void* q, int64_t q_row_stride, const void* key, const void* value,
                     int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                     int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                     int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                     int max_seqlen_q, int uniform_seqlen_q, int uniform_seqlen_k, int num_heads, int num_kv_heads,
                     int head_dim, float softmax_scale, int causal, void* out, int64_t out_row_stride, int plan,
                     void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 0 || max_seqlen_q < 0) return fail(VOX_EINVAL, "prefill_attn: negative batch or max_seqlen_q");
  if (batch == 0 || max_seqlen_q == 0) return VOX_OK;
  if (!out) return fail(VOX_EINVAL, "prefill_attn: null out");
  if (out_row_stride < (int64_t)num_heads * head_dim || out_row_stride % 4 || ((uintptr_t)out & 7u))
    return fail(VOX_EINVAL, "prefill_attn: bad out row stride or alignment");
  vox::PrefillArgs a;
  const int st = prefill_setup("prefill_attn", q, q_row_stride, key, value, key_row_stride, value_row_stride, k_cache,
                               v_cache, num_blocks, block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q,
                               cu_seqlens_k, batch, max_seqlen_q, uniform_seqlen_q, uniform_seqlen_k, num_heads,
                               num_kv_heads, head_dim, softmax_scale, causal, &a);
  if (st != VOX_OK) return st;
  a.out = (uint16_t*)out;
  a.out_row_stride = out_row_stride;
  const hipStream_t s = (hipStream_t)stream;
  // One-query sequences of a paged varlen call (the decode rows of a mixed step) go to the split-KV decode kernels,
  // which spread long contexts over every CU; the prefill kernel takes the rest. Needs the workspace and the decode
  // kernels' shapes; otherwise the prefill kernel takes every row.
  if (varlen_decode_rows(a, workspace, num_kv_heads)) {
    const int sw = check_varlen_workspace("prefill_attn", batch, plan, workspace, workspace_bytes);
    if (sw != VOX_OK) return sw;
    a.skip_single = 1;
    a.persistent = 1;  // the (q tile, sequence) grid would be mostly the decode rows' empty tiles
    const vox::DecodeArgs d = varlen_decode_args(a, q_row_stride, num_blocks, num_heads, num_kv_heads);
    if (max_seqlen_q > 1 && vox::mixed_launch_fits(a, num_kv_heads)) {
      // both kinds of rows in one launch, sharing the CUs (then the merge kernel)
      const vox::DecodeArgs dw = with_workspace(d, batch, plan, workspace);
      return hip_status(vox::launch_mixed(a, max_seqlen_q, dw, num_kv_heads, s), "prefill_attn mixed launch");
    }
    if (max_seqlen_q > 1) {
      const int sp = hip_status(vox::launch_prefill(a, max_seqlen_q, s), "prefill_attn launch");
      if (sp != VOX_OK) return sp;
    }
    return launch_decode_slices(d, batch, num_kv_heads, plan, workspace, s);
  }
  return hip_status(vox::launch_prefill(a, max_seqlen_q, s), "prefill_attn launch");
}

int vox_prefill_attn_store(const void* q, int64_t q_row_stride, const void* key, const void* value,
                           int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                           void* k_cache, void* v_cache, int64_t num_slots, int64_t num_tokens,
                           const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                           int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int causal, void* out,
                           int64_t out_row_stride, void* stream) {
  if (batch < 0 || max_seqlen_q < 0 || num_tokens < 0)
    return fail(VOX_EINVAL, "prefill_attn_store: negative batch, max_seqlen_q or num_tokens");
  if (!key || !value || !k_cache || !v_cache || !slot_mapping || !cu_seqlens_q || !cu_seqlens_k)
    return fail(VOX_EINVAL, "prefill_attn_store: null pointer argument");
  if (num_slots <= 0) return fail(VOX_EINVAL, "prefill_attn_store: empty cache");
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (num_kv_heads <= 0 || head_dim <= 0 || key_row_stride < row || value_row_stride < row)
    return fail(VOX_EINVAL, "prefill_attn_store: key / value row strides smaller than num_kv_heads * head_dim");
  // every argument is checked before anything is launched
  const bool attend = batch > 0 && max_seqlen_q > 0;
  vox::PrefillArgs a;
  if (attend) {
    if (!out) return fail(VOX_EINVAL, "prefill_attn_store: null out");
    if (out_row_stride < (int64_t)num_heads * head_dim || out_row_stride % 4 || ((uintptr_t)out & 7u))
      return fail(VOX_EINVAL, "prefill_attn_store: bad out row stride or alignment");
    const int st = prefill_setup("prefill_attn_store", q, q_row_stride, key, value, key_row_stride,
                                 value_row_stride, nullptr, nullptr, 0, 0, nullptr, 0, 0, cu_seqlens_q, cu_seqlens_k,
                                 batch, max_seqlen_q, 0, 0, num_heads, num_kv_heads, head_dim, softmax_scale, causal,
                                 &a);
    if (st != VOX_OK) return st;
  }
  const bool vec16 = row % 8 == 0 && key_row_stride % 8 == 0 && value_row_stride % 8 == 0 && aligned16(key) &&
                     aligned16(value) && aligned16(k_cache) && aligned16(v_cache);
  if (!attend || !vec16 || num_tokens == 0) {
    // no launch to ride in, nothing to store, or rows the 16-byte copy cannot move: the two calls
    const int st = vox_store_kvcache(key, value, key_row_stride, value_row_stride, k_cache, v_cache, num_slots,
                                     slot_mapping, num_tokens, num_kv_heads, head_dim, stream);
    if (st != VOX_OK || !attend) return st;
    return vox_prefill_attn(q, q_row_stride, key, value, key_row_stride, value_row_stride, nullptr, nullptr, 0, 0,
                            nullptr, 0, 0, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q, 0, 0, num_heads,
                            num_kv_heads, head_dim, softmax_scale, causal, out, out_row_stride, VOX_PLAN_NONE,
                            nullptr, 0, stream);
  }
  a.out = (uint16_t*)out;
  a.out_row_stride = out_row_stride;
  a.store_slots = slot_mapping;
  a.store_k_cache = (uint16_t*)k_cache;
  a.store_v_cache = (uint16_t*)v_cache;
  a.store_rows = num_tokens;
  a.store_num_slots = num_slots;
  return hip_status(vox::launch_prefill(a, max_seqlen_q, (hipStream_t)stream), "prefill_attn_store launch");
}

int vox_prefill_attn_store_paged(const void* q, int64_t q_row_stride, const void* key, const void* value,
                                 int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                                 int64_t num_tokens, void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                                 const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                 const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                                 int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int causal,
                                 void* out, int64_t out_row_stride, int plan, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (batch < 0 || max_seqlen_q < 0 || num_tokens < 0)
    return fail(VOX_EINVAL, "prefill_attn_store_paged: negative batch, max_seqlen_q or num_tokens");
  if (!key || !value || !k_cache || !v_cache || !slot_mapping || !block_tables || !cu_seqlens_q || !cu_seqlens_k)
    return fail(VOX_EINVAL, "prefill_attn_store_paged: null pointer argument");
  if (num_blocks <= 0 || block_size <= 0) return fail(VOX_EINVAL, "prefill_attn_store_paged: empty cache");
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (num_kv_heads <= 0 || head_dim <= 0 || key_row_stride < row || value_row_stride < row)
    return fail(VOX_EINVAL, "prefill_attn_store_paged: key / value row strides smaller than num_kv_heads * head_dim");
  // every argument is checked before anything is launched
  const bool attend = batch > 0 && max_seqlen_q > 0;
  vox::PrefillArgs a;
  if (attend) {
    if (!out) return fail(VOX_EINVAL, "prefill_attn_store_paged: null out");
    if (out_row_stride < (int64_t)num_heads * head_dim || out_row_stride % 4 || ((uintptr_t)out & 7u))
      return fail(VOX_EINVAL, "prefill_attn_store_paged: bad out row stride or alignment");
    const int st = prefill_setup("prefill_attn_store_paged", q, q_row_stride, key, value, key_row_stride,
                                 value_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride,
                                 max_blocks, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q, 0, 0, num_heads,
                                 num_kv_heads, head_dim, softmax_scale, causal, &a);
    if (st != VOX_OK) return st;
    a.out = (uint16_t*)out;
    a.out_row_stride = out_row_stride;
    if (varlen_decode_rows(a, workspace, num_kv_heads)) {
      const int sw = check_varlen_workspace("prefill_attn_store_paged", batch, plan, workspace, workspace_bytes);
      if (sw != VOX_OK) return sw;
    }
  }
  if (plan != VOX_PLAN_NONE && plan != VOX_PLAN_RECORD && plan != VOX_PLAN_REUSE)
    return fail(VOX_EINVAL, "prefill_attn_store_paged: plan mode %d", plan);
  // The store rides in the attention launch: in a mixed launch both roles read each sequence's new keys from the rows
  // (by position) and the merge kernel's extra workgroups write the rows into the caches after every read. Else the
  // two calls.
  const bool vec16 = row % 8 == 0 && key_row_stride % 8 == 0 && value_row_stride % 8 == 0 && aligned16(key) &&
                     aligned16(value) && aligned16(k_cache) && aligned16(v_cache) &&
                     key_row_stride < (1 << 24) && value_row_stride < (1 << 24);
  const bool decode_rows = attend && varlen_decode_rows(a, workspace, num_kv_heads);
  const bool fold_mixed = attend && num_tokens > 0 && max_seqlen_q > 1 && vec16 && decode_rows &&
                          vox::mixed_launch_fits(a, num_kv_heads);
  // without the decode rows' workspace the prefill kernel takes every row: the store rides in its launch as in the
  // packed form (workgroups that have done their item, or have none, copy the rows beside the others' reads), and the
  // new keys are read from the rows alone
  const bool fold_plain = attend && num_tokens > 0 && vec16 && !decode_rows && block_size % 64 == 0;
  if (fold_plain) {
    a.k_src = (const uint16_t*)key;
    a.v_src = (const uint16_t*)value;
    a.k_row_stride = key_row_stride;
    a.v_row_stride = value_row_stride;
    a.new_from_rows = 1;
    a.store_slots = slot_mapping;
    a.store_k_cache = (uint16_t*)k_cache;
    a.store_v_cache = (uint16_t*)v_cache;
    a.store_rows = num_tokens;
    a.store_num_slots = num_blocks * block_size;
    return hip_status(vox::launch_prefill(a, max_seqlen_q, (hipStream_t)stream), "prefill_attn_store_paged launch");
  }
  if (!fold_mixed) {
    const int st = vox_store_kvcache(key, value, key_row_stride, value_row_stride, k_cache, v_cache,
                                     num_blocks * block_size, slot_mapping, num_tokens, num_kv_heads, head_dim, stream);
    if (st != VOX_OK || !attend) return st;
    return vox_prefill_attn(q, q_row_stride, key, value, key_row_stride, value_row_stride, k_cache, v_cache, num_blocks,
                            block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q, cu_seqlens_k, batch,
                            max_seqlen_q, 0, 0, num_heads, num_kv_heads, head_dim, softmax_scale, causal, out,
                            out_row_stride, plan, workspace, workspace_bytes, stream);
  }
  a.skip_single = 1;
  a.persistent = 1;
  a.k_src = (const uint16_t*)key;
  a.v_src = (const uint16_t*)value;
  a.k_row_stride = key_row_stride;
  a.v_row_stride = value_row_stride;
  a.new_from_rows = 1;
  vox::DecodeArgs d = varlen_decode_args(a, q_row_stride, num_blocks, num_heads, num_kv_heads);
  d.slot_mapping = slot_mapping;
  d.new_k = (const uint16_t*)key;
  d.new_v = (const uint16_t*)value;
  d.new_k_stride = key_row_stride;
  d.new_v_stride = value_row_stride;
  d.copy_rows = num_tokens;
  // about one batch of 16-byte copies per thread of a 256-thread workgroup (16 rows of 2 x 256 bf16), at most 256
  const int64_t per_wg = 4 * 256 / (2 * row / 8);
  const int64_t cw = (num_tokens + per_wg - 1) / per_wg;
  d.copy_wgs = (int)(cw < 256 ? cw : 256);
  const vox::DecodeArgs dw = with_workspace(d, batch, plan, workspace);
  return hip_status(vox::launch_mixed(a, max_seqlen_q, dw, num_kv_heads, (hipStream_t)stream),
                    "prefill_attn_store_paged mixed launch");
}

}  // extern "C"

namespace {
// A KV store riding in an int8 prefill launch (vox_prefill_attn_int8_store): rows [0, rows) of the key / value rows
// to slot_mapping's slots
struct RidingStore {
  const int32_t* slot_mapping;
  void* k_cache;
  void* v_cache;
  int64_t num_slots;
  int64_t rows;
  bool paged;  // paged tiles: the launch reads each sequence's new keys from the rows
};

int prefill_int8(const char* fn, const void* q, int64_t q_row_stride, const void* key, const void* value,
                 int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                 int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                 const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                 int uniform_seqlen_q, int uniform_seqlen_k, int num_heads, int num_kv_heads, int head_dim,
                 float softmax_scale, int causal, const float* inv_smooth, void* out_q, int64_t out_q_row_stride,
                 float* out_scale, int64_t num_tokens, void* workspace, size_t workspace_bytes,
                 const RidingStore* store, bool launch, hipStream_t stream) {
  if (!out_q || !out_scale) return fail(VOX_EINVAL, "%s: null out_q or out_scale", fn);
  if (num_kv_heads != 1 && num_kv_heads != 2)
    return fail(VOX_EINVAL, "%s: num_kv_heads %d unsupported (1 or 2)", fn, num_kv_heads);
  if (out_q_row_stride < (int64_t)num_heads * head_dim || out_q_row_stride % 4 || ((uintptr_t)out_q & 3u))
    return fail(VOX_EINVAL, "%s: bad out_q row stride or alignment", fn);
  if (((uintptr_t)out_scale & 3u) || (inv_smooth && !aligned16(inv_smooth)))
    return fail(VOX_EINVAL, "%s: out_scale must be 4-byte and inv_smooth 16-byte aligned", fn);
  vox::PrefillArgs a;
  const int st = prefill_setup(fn, q, q_row_stride, key, value, key_row_stride, value_row_stride, k_cache, v_cache,
                               num_blocks, block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q,
                               cu_seqlens_k, batch, max_seqlen_q, uniform_seqlen_q, uniform_seqlen_k, num_heads,
                               num_kv_heads, head_dim, softmax_scale, causal, &a);
  if (st != VOX_OK) return st;
  if (!cu_seqlens_q && num_tokens != (int64_t)batch * uniform_seqlen_q)
    return fail(VOX_EINVAL, "%s: num_tokens %lld != batch x uniform_seqlen_q", fn, (long long)num_tokens);
  // rows at or past num_tokens are never read or written, whatever cu_seqlens_q (device memory the host cannot
  // check here) says: the outputs and the two-pass scratch are sized by num_tokens
  a.row_limit = num_tokens;
  const size_t need = workspace ? vox_prefill_int8_workspace_bytes(num_tokens, batch, max_seqlen_q, num_heads,
                                                                   num_kv_heads, head_dim, causal)
                                : 0;
  if (need && (workspace_bytes < need || !aligned16(workspace)))
    return fail(VOX_EINVAL, "%s: workspace of %zu bytes (16-byte aligned), %zu needed", fn, workspace_bytes, need);
  if (!launch) return VOX_OK;  // (arguments checked only)
  if (store) {
    if (store->paged) {
      a.k_src = (const uint16_t*)key;
      a.v_src = (const uint16_t*)value;
      a.k_row_stride = key_row_stride;
      a.v_row_stride = value_row_stride;
      a.new_from_rows = 1;
    }
    a.store_slots = store->slot_mapping;
    a.store_k_cache = (uint16_t*)store->k_cache;
    a.store_v_cache = (uint16_t*)store->v_cache;
    a.store_rows = store->rows;
    a.store_num_slots = store->num_slots;
  }
  if (need) {
    // two passes: the bf16 kernel into the workspace ([T, H * 128] bf16; a riding store copied in that launch), then
    // the per-token quantization
    a.out = (uint16_t*)workspace;
    a.out_row_stride = (int64_t)num_heads * head_dim;
    const int st1 = hip_status(vox::launch_prefill(a, max_seqlen_q, stream), "prefill_attn_int8 launch");
    if (st1 != VOX_OK) return st1;
    return hip_status(vox::launch_quantize_rows((const uint16_t*)workspace, num_tokens, num_heads * head_dim,
                                                inv_smooth, (int8_t*)out_q, out_q_row_stride, out_scale, stream),
                      "prefill_attn_int8 quantization launch");
  }
  a.inv_smooth = inv_smooth;
  a.out_q = (int8_t*)out_q;
  a.out_row_stride = out_q_row_stride;
  a.out_scale = out_scale;
  return hip_status(vox::launch_prefill_int8(a, max_seqlen_q, stream), "prefill_attn_int8 launch");
}
}  // namespace

extern "C" {

int vox_prefill_attn_int8(const void* q, int64_t q_row_stride, const void* key, const void* value,
                          int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                          int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                          int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                          int max_seqlen_q, int uniform_seqlen_q, int uniform_seqlen_k, int num_heads,
                          int num_kv_heads, int head_dim, float softmax_scale, int causal, const float* inv_smooth,
                          void* out_q, int64_t out_q_row_stride, float* out_scale, int64_t num_tokens,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 0 || max_seqlen_q < 0 || num_tokens < 0)
    return fail(VOX_EINVAL, "prefill_attn_int8: negative batch, max_seqlen_q or num_tokens");
  if (batch == 0 || max_seqlen_q == 0 || num_tokens == 0) return VOX_OK;
  return prefill_int8("prefill_attn_int8", q, q_row_stride, key, value, key_row_stride, value_row_stride, k_cache,
                      v_cache, num_blocks, block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q,
                      cu_seqlens_k, batch, max_seqlen_q, uniform_seqlen_q, uniform_seqlen_k, num_heads, num_kv_heads,
                      head_dim, softmax_scale, causal, inv_smooth, out_q, out_q_row_stride, out_scale, num_tokens,
                      workspace, workspace_bytes, nullptr, true, (hipStream_t)stream);
}

int vox_prefill_attn_int8_store(const void* q, int64_t q_row_stride, const void* key, const void* value,
                                int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                                int64_t store_rows, void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                                const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                                int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int causal,
                                const float* inv_smooth, void* out_q, int64_t out_q_row_stride, float* out_scale,
                                int64_t num_tokens, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "prefill_attn_int8_store";
  if (batch < 0 || max_seqlen_q < 0 || num_tokens < 0 || store_rows < 0)
    return fail(VOX_EINVAL, "%s: negative batch, max_seqlen_q, num_tokens or store_rows", fn);
  if (!key || !value || !k_cache || !v_cache || !slot_mapping || !cu_seqlens_q || !cu_seqlens_k)
    return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  if (num_blocks <= 0 || block_size <= 0) return fail(VOX_EINVAL, "%s: empty cache", fn);
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (num_kv_heads <= 0 || head_dim <= 0 || key_row_stride < row || value_row_stride < row)
    return fail(VOX_EINVAL, "%s: key / value row strides smaller than num_kv_heads * head_dim", fn);
  // every argument is checked before anything is launched
  const bool paged = block_tables != nullptr;
  const bool attend = batch > 0 && max_seqlen_q > 0 && num_tokens > 0;
  const void* kc_read = paged ? k_cache : nullptr;
  const void* vc_read = paged ? v_cache : nullptr;
  if (attend) {
    const int st = prefill_int8(fn, q, q_row_stride, key, value, key_row_stride, value_row_stride, kc_read, vc_read,
                                num_blocks, block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q,
                                cu_seqlens_k, batch, max_seqlen_q, 0, 0, num_heads, num_kv_heads, head_dim,
                                softmax_scale, causal, inv_smooth, out_q, out_q_row_stride, out_scale, num_tokens,
                                workspace, workspace_bytes, nullptr, false, nullptr);
    if (st != VOX_OK) return st;
  }
  // the store rides in the launch over packed keys, or over paged tiles that read the new keys from the rows
  const bool vec16 = row % 8 == 0 && key_row_stride % 8 == 0 && value_row_stride % 8 == 0 && aligned16(key) &&
                     aligned16(value) && aligned16(k_cache) && aligned16(v_cache) && key_row_stride < (1 << 24) &&
                     value_row_stride < (1 << 24);
  if (!attend || !vec16 || store_rows == 0 || (paged && block_size % 64 != 0)) {
    // no launch to ride in, nothing to store, or rows / blocks the riding copy does not take: the two calls
    const int st = vox_store_kvcache(key, value, key_row_stride, value_row_stride, k_cache, v_cache,
                                     num_blocks * block_size, slot_mapping, store_rows, num_kv_heads, head_dim, stream);
    if (st != VOX_OK || !attend) return st;
    return vox_prefill_attn_int8(q, q_row_stride, key, value, key_row_stride, value_row_stride, kc_read, vc_read,
                                 num_blocks, block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q,
                                 cu_seqlens_k, batch, max_seqlen_q, 0, 0, num_heads, num_kv_heads, head_dim,
                                 softmax_scale, causal, inv_smooth, out_q, out_q_row_stride, out_scale, num_tokens,
                                 workspace, workspace_bytes, stream);
  }
  const RidingStore rs{slot_mapping, k_cache, v_cache, num_blocks * block_size, store_rows, paged};
  return prefill_int8(fn, q, q_row_stride, key, value, key_row_stride, value_row_stride, kc_read, vc_read, num_blocks,
                      block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q,
                      0, 0, num_heads, num_kv_heads, head_dim, softmax_scale, causal, inv_smooth, out_q,
                      out_q_row_stride, out_scale, num_tokens, workspace, workspace_bytes, &rs, true,
                      (hipStream_t)stream);
}

size_t vox_prefill_int8_workspace_bytes(int64_t num_tokens, int batch, int max_seqlen_q, int num_heads,
                                        int num_kv_heads, int head_dim, int causal) {
  if (num_tokens <= 0 || head_dim != kHeadDim || num_heads <= 0 || num_heads * head_dim > 2048) return 0;
  if (!vox::prefill_int8_two_pass(batch, max_seqlen_q, num_heads, num_kv_heads, causal)) return 0;
  return (size_t)num_tokens * num_heads * head_dim * 2;
}

int vox_copy_kv_block_prefix(void* kv, int64_t num_planes, int64_t num_blocks, int block_size,
                              int64_t per_token, int elem_bytes, const int32_t* entries, int num_entries,
                              int max_tokens, void* stream) {
  if (num_entries < 0 || num_planes < 0) return fail(VOX_EINVAL, "copy_kv_block_prefix: negative count");
  if (num_entries == 0 || num_planes == 0 || max_tokens <= 0) return VOX_OK;
  if (!kv || !entries) return fail(VOX_EINVAL, "copy_kv_block_prefix: null kv or entries");
  if (elem_bytes != 2) return fail(VOX_EINVAL, "copy_kv_block_prefix: %d-byte elements unsupported (2 only)", elem_bytes);
  if (num_blocks <= 0 || block_size <= 0 || per_token <= 0)
    return fail(VOX_EINVAL, "copy_kv_block_prefix: bad cache shape");
  if (num_planes > 65535) return fail(VOX_EINVAL, "copy_kv_block_prefix: more than 65535 planes");
  if (max_tokens > block_size) max_tokens = block_size;
  vox::CopyArgs a;
  a.kv = kv;
  a.num_planes = num_planes;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.per_token = per_token;
  a.entries = entries;
  a.num_entries = num_entries;
  const bool vec16 = per_token % 8 == 0 && aligned16(kv);
  return hip_status(vox::launch_copy_block_prefix(a, max_tokens, vec16, (hipStream_t)stream),
                    "copy_kv_block_prefix launch");
}

}  // extern "C"

// ---- 4-bit caches and the care of a cache's blocks

namespace {
// What every call over 4-bit caches needs of them.
int fp4_cache(const char* fn, const void* k_cache, const void* v_cache, int64_t num_blocks, int block_size,
              int num_kv_heads, int head_dim) {
  if (!k_cache || !v_cache) return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  if (head_dim != kHeadDim) return fail(VOX_EINVAL, "%s: head_dim %d unsupported (128 only)", fn, head_dim);
  if (num_kv_heads <= 0 || num_kv_heads > 128) return fail(VOX_EINVAL, "%s: num_kv_heads %d", fn, num_kv_heads);
  if (block_size <= 0 || block_size % 64)
    return fail(VOX_EINVAL, "%s: block_size %d must be a positive multiple of 64", fn, block_size);
  if (num_blocks <= 0) return fail(VOX_EINVAL, "%s: empty cache", fn);
  // a block's byte offsets are 32-bit, its slots int32
  if ((int64_t)block_size * num_kv_heads * 68 > (1 << 30) || num_blocks > INT32_MAX / block_size)
    return fail(VOX_EINVAL, "%s: %lld blocks of %d slots are more than int32 slots reach", fn, (long long)num_blocks,
                block_size);
  if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(VOX_EINVAL, "%s: caches must be 16-byte aligned", fn);
  return VOX_OK;
}

// Of the attention calls: masked scores are -infinity before the scale, so it has to keep them there.
int fp4_softmax(const char* fn, float softmax_scale) {
  if (!(softmax_scale >= 2 * FLT_MIN && softmax_scale <= FLT_MAX / 2))
    return fail(VOX_EINVAL, "%s: softmax_scale %g must be positive", fn, (double)softmax_scale);
  return VOX_OK;
}

// A cache's planes as bytes, for the call fn.
int pages_setup(const char* fn, void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t slot_bytes,
                int64_t scale_bytes, vox::PagesArgs* out) {
  if (!kv) return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  if (num_planes <= 0 || num_planes > 65535) return fail(VOX_EINVAL, "%s: %lld planes", fn, (long long)num_planes);
  if (num_blocks <= 0 || block_size <= 0 || slot_bytes <= 0 || scale_bytes < 0)
    return fail(VOX_EINVAL, "%s: bad cache shape", fn);
  if (num_blocks > INT32_MAX / block_size || slot_bytes > (1 << 20) || scale_bytes > (1 << 20) ||
      (int64_t)block_size * (slot_bytes + scale_bytes) > (1 << 29))
    return fail(VOX_EINVAL, "%s: cache shape out of range", fn);
  if (!aligned16(kv) || (int64_t)block_size * slot_bytes % 16 || (int64_t)block_size * scale_bytes % 16)
    return fail(VOX_EINVAL, "%s: the cache and the runs of a block must be 16-byte aligned", fn);
  out->kv = (uint8_t*)kv;
  out->num_planes = num_planes;
  out->num_blocks = num_blocks;
  out->block_size = block_size;
  out->slot_bytes = slot_bytes;
  out->scale_bytes = scale_bytes;
  return VOX_OK;
}
}  // namespace

extern "C" {

int vox_store_kvcache_fp4(const void* key, const void* value, int64_t key_row_stride, int64_t value_row_stride,
                          void* k_cache, void* v_cache, int64_t num_blocks, int block_size, const int32_t* slot_mapping,
                          int64_t num_tokens, int num_kv_heads, int head_dim, void* stream) {
  const char* fn = "store_kvcache_fp4";
  if (num_tokens < 0) return fail(VOX_EINVAL, "%s: num_tokens %lld < 0", fn, (long long)num_tokens);
  if (num_tokens == 0) return VOX_OK;
  if (!key || !value || !slot_mapping) return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  const int st = fp4_cache(fn, k_cache, v_cache, num_blocks, block_size, num_kv_heads, head_dim);
  if (st != VOX_OK) return st;
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key_row_stride < row || value_row_stride < row)
    return fail(VOX_EINVAL, "%s: row stride smaller than num_kv_heads * head_dim", fn);
  const vox::Fp4RowsArgs a{(const uint16_t*)key, (const uint16_t*)value, key_row_stride, value_row_stride,
                           (uint8_t*)k_cache, (uint8_t*)v_cache, num_blocks * block_size, block_size, num_kv_heads,
                           slot_mapping, num_tokens};
  const bool vec16 = key_row_stride % 8 == 0 && value_row_stride % 8 == 0 && aligned16(key) && aligned16(value);
  return hip_status(vox::launch_store_fp4(a, vec16, (hipStream_t)stream), "store_kvcache_fp4 launch");
}

int vox_load_kvcache_fp4(const void* k_cache, const void* v_cache, int64_t num_blocks, int block_size,
                         const int32_t* slots, int64_t num_tokens, int num_kv_heads, int head_dim, void* key,
                         void* value, void* stream) {
  const char* fn = "load_kvcache_fp4";
  if (num_tokens < 0) return fail(VOX_EINVAL, "%s: num_tokens %lld < 0", fn, (long long)num_tokens);
  if (num_tokens == 0) return VOX_OK;
  if (!key || !value || !slots) return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  const int st = fp4_cache(fn, k_cache, v_cache, num_blocks, block_size, num_kv_heads, head_dim);
  if (st != VOX_OK) return st;
  if (!aligned16(key) || !aligned16(value)) return fail(VOX_EINVAL, "%s: key and value must be 16-byte aligned", fn);
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  const vox::Fp4RowsArgs a{(const uint16_t*)key, (const uint16_t*)value, row, row, (uint8_t*)k_cache,
                           (uint8_t*)v_cache, num_blocks * block_size, block_size, num_kv_heads, slots, num_tokens};
  return hip_status(vox::launch_load_fp4(a, (hipStream_t)stream), "load_kvcache_fp4 launch");
}

int vox_decode_attn_fp4(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                        int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                        int max_blocks, const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                        int head_dim, float softmax_scale, int plan, void* workspace, size_t workspace_bytes,
                        void* out, void* stream) {
  if (batch < 0) return fail(VOX_EINVAL, "decode_attn_fp4: batch < 0");
  if (plan != VOX_PLAN_NONE && plan != VOX_PLAN_RECORD && plan != VOX_PLAN_REUSE)
    return fail(VOX_EINVAL, "decode_attn_fp4: plan mode %d", plan);
  if (batch == 0) return VOX_OK;
  int st = fp4_cache("decode_attn_fp4", k_cache, v_cache, num_blocks, block_size, num_kv_heads, head_dim);
  if (st == VOX_OK) st = fp4_softmax("decode_attn_fp4", softmax_scale);
  if (st != VOX_OK) return st;
  vox::DecodeArgs a;
  st = decode_setup(q, q_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride, max_blocks,
                    context_lens, batch, num_heads, num_kv_heads, head_dim, softmax_scale, workspace, workspace_bytes,
                    out, &a);
  if (st != VOX_OK) return st;
  return launch_decode_slices(a, batch, num_kv_heads, plan, workspace, (hipStream_t)stream, vox::launch_decode_fp4);
}

int vox_decode_attn_store_fp4(const void* q, int64_t q_row_stride, const void* key, const void* value,
                              int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                              void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                              const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                              const int32_t* context_lens, int batch, int num_heads, int num_kv_heads, int head_dim,
                              float softmax_scale, int plan, void* workspace, size_t workspace_bytes, void* out,
                              void* stream) {
  if (batch < 0) return fail(VOX_EINVAL, "decode_attn_store_fp4: batch < 0");
  if (plan != VOX_PLAN_NONE && plan != VOX_PLAN_RECORD && plan != VOX_PLAN_REUSE)
    return fail(VOX_EINVAL, "decode_attn_store_fp4: plan mode %d", plan);
  if (batch == 0) return VOX_OK;
  if (!key || !value || !slot_mapping)
    return fail(VOX_EINVAL, "decode_attn_store_fp4: null key, value or slot_mapping");
  int st = fp4_cache("decode_attn_store_fp4", k_cache, v_cache, num_blocks, block_size, num_kv_heads, head_dim);
  if (st == VOX_OK) st = fp4_softmax("decode_attn_store_fp4", softmax_scale);
  if (st != VOX_OK) return st;
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key_row_stride < row || value_row_stride < row)
    return fail(VOX_EINVAL, "decode_attn_store_fp4: row stride smaller than num_kv_heads * head_dim");
  // every argument is checked before anything is launched
  vox::DecodeArgs a;
  st = decode_setup(q, q_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride, max_blocks,
                    context_lens, batch, num_heads, num_kv_heads, head_dim, softmax_scale, workspace, workspace_bytes,
                    out, &a);
  if (st != VOX_OK) return st;
  if (key_row_stride % 8 || value_row_stride % 8 || !aligned16(key) || !aligned16(value)) {
    // rows that the decode kernels' 16-byte loads cannot take: the two calls
    st = vox_store_kvcache_fp4(key, value, key_row_stride, value_row_stride, k_cache, v_cache, num_blocks, block_size,
                               slot_mapping, batch, num_kv_heads, head_dim, stream);
    if (st != VOX_OK) return st;
  } else {
    a.slot_mapping = slot_mapping;
    a.new_k = (const uint16_t*)key;
    a.new_v = (const uint16_t*)value;
    a.new_k_stride = key_row_stride;
    a.new_v_stride = value_row_stride;
  }
  return launch_decode_slices(a, batch, num_kv_heads, plan, workspace, (hipStream_t)stream, vox::launch_decode_fp4);
}

int vox_prefill_attn_fp4(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                         int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                         int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                         int max_seqlen_q, int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim,
                         float softmax_scale, int causal, void* out, int64_t out_row_stride, int plan, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const char* fn = "prefill_attn_fp4";
  if (batch < 0 || max_seqlen_q < 0 || num_tokens < 0)
    return fail(VOX_EINVAL, "%s: negative batch, max_seqlen_q or num_tokens", fn);
  if (batch == 0 || max_seqlen_q == 0 || num_tokens == 0) return VOX_OK;
  if (!block_tables || !cu_seqlens_q || !cu_seqlens_k || !out)
    return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  int st = fp4_cache(fn, k_cache, v_cache, num_blocks, block_size, num_kv_heads, head_dim);
  if (st == VOX_OK) st = fp4_softmax(fn, softmax_scale);
  if (st != VOX_OK) return st;
  if (out_row_stride < (int64_t)num_heads * head_dim || out_row_stride % 4 || ((uintptr_t)out & 7u))
    return fail(VOX_EINVAL, "%s: bad out row stride or alignment", fn);
  if (batch > 65535) return fail(VOX_EINVAL, "%s: more than 65535 sequences", fn);
  if ((int64_t)max_blocks * block_size > (1 << 30)) return fail(VOX_EINVAL, "%s: block table too wide", fn);
  vox::PrefillArgs a;
  st = prefill_setup(fn, q, q_row_stride, nullptr, nullptr, 0, 0, k_cache, v_cache, num_blocks, block_size,
                     block_tables, bt_stride, max_blocks, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q, 0, 0,
                     num_heads, num_kv_heads, head_dim, softmax_scale, causal, &a);
  if (st != VOX_OK) return st;
  a.out = (uint16_t*)out;
  a.out_row_stride = out_row_stride;
  a.row_limit = num_tokens;
  const hipStream_t s = (hipStream_t)stream;
  if (!varlen_decode_rows(a, workspace, num_kv_heads))
    return hip_status(vox::launch_prefill_fp4(a, max_seqlen_q, s), "prefill_attn_fp4 launch");
  // the one-query rows on the decode kernels, which spread a long context over every CU
  st = check_varlen_workspace(fn, batch, plan, workspace, workspace_bytes);
  if (st != VOX_OK) return st;
  a.skip_single = 1;
  const vox::DecodeArgs d = varlen_decode_args(a, q_row_stride, num_blocks, num_heads, num_kv_heads);
  if (vox::mixed_fp4_fits(a, max_seqlen_q))
    return hip_status(vox::launch_mixed_fp4(a, max_seqlen_q, with_workspace(d, batch, plan, workspace), s),
                      "prefill_attn_fp4 mixed launch");
  if (max_seqlen_q > 1) {
    st = hip_status(vox::launch_prefill_fp4(a, max_seqlen_q, s), "prefill_attn_fp4 launch");
    if (st != VOX_OK) return st;
  }
  return launch_decode_slices(d, batch, num_kv_heads, plan, workspace, s, vox::launch_decode_fp4);
}

int vox_copy_kv_blocks(void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t slot_bytes,
                       int64_t scale_bytes, const int32_t* entries, int num_entries, void* stream) {
  if (num_entries < 0) return fail(VOX_EINVAL, "copy_kv_blocks: negative count");
  if (num_entries == 0) return VOX_OK;
  if (!entries) return fail(VOX_EINVAL, "copy_kv_blocks: null pointer argument");
  vox::PagesArgs a;
  const int st = pages_setup("copy_kv_blocks", kv, num_planes, num_blocks, block_size, slot_bytes, scale_bytes, &a);
  if (st != VOX_OK) return st;
  return hip_status(vox::launch_copy_entries(a, entries, num_entries, (hipStream_t)stream), "copy_kv_blocks launch");
}

int vox_fork_kv_blocks(void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t slot_bytes,
                       int64_t scale_bytes, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                       const int32_t* context_lens, int batch, const int32_t* parents, const int32_t* new_blocks,
                       int num_forks, int32_t* child_tables, int32_t* child_lens, void* stream) {
  const char* fn = "fork_kv_blocks";
  if (num_forks < 0 || batch < 0) return fail(VOX_EINVAL, "%s: negative count", fn);
  if (num_forks == 0) return VOX_OK;
  if ((batch > 0 && (!block_tables || !context_lens)) || !parents || !new_blocks || !child_tables || !child_lens)
    return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  if (max_blocks <= 0 || bt_stride < max_blocks || (int64_t)max_blocks * block_size > (1 << 30))
    return fail(VOX_EINVAL, "%s: bad block table shape", fn);
  vox::PagesArgs a;
  const int st = pages_setup(fn, kv, num_planes, num_blocks, block_size, slot_bytes, scale_bytes, &a);
  if (st != VOX_OK) return st;
  const vox::ForkArgs f{block_tables, bt_stride, max_blocks, context_lens, batch, parents, new_blocks, num_forks,
                        child_tables, child_lens};
  return hip_status(vox::launch_fork(a, f, (hipStream_t)stream), "fork_kv_blocks launch");
}

int vox_compact_kv_blocks(void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t slot_bytes,
                          int64_t scale_bytes, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                          const int32_t* context_lens, int batch, int32_t* new_tables, int32_t* remap, int32_t* live,
                          int32_t* moves, void* stream) {
  const char* fn = "compact_kv_blocks";
  if (batch < 0) return fail(VOX_EINVAL, "%s: batch < 0", fn);
  if (!remap || !live || !moves || (batch > 0 && (!block_tables || !context_lens || !new_tables)))
    return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  if (batch > 0 && (max_blocks <= 0 || bt_stride < max_blocks || (int64_t)max_blocks * block_size > (1 << 30)))
    return fail(VOX_EINVAL, "%s: bad block table shape", fn);
  vox::PagesArgs a;
  const int st = pages_setup(fn, kv, num_planes, num_blocks, block_size, slot_bytes, scale_bytes, &a);
  if (st != VOX_OK) return st;
  if (num_blocks > (1 << 18))  // its bitmap of the blocks lives in 32 KiB of LDS
    return fail(VOX_EINVAL, "%s: %lld blocks, %d at most", fn, (long long)num_blocks, 1 << 18);
  const vox::CompactArgs c{block_tables, bt_stride, max_blocks > 0 ? max_blocks : 1, context_lens, batch, new_tables, remap, live,
                           moves};
  return hip_status(vox::launch_compact(a, c, (hipStream_t)stream), "compact_kv_blocks launch");
}

}  // extern "C"

// ---- what each key receives, and eviction by it

namespace {
int weights_setup(const char* fn, const float* key_weights, int64_t num_weight_rows, int64_t weight_width, float softmax_scale) {
  if (!key_weights || ((uintptr_t)key_weights & 3u)) return fail(VOX_EINVAL, "%s: null or unaligned key_weights", fn);
  if (num_weight_rows <= 0 || weight_width <= 0) return fail(VOX_EINVAL, "%s: empty key_weights", fn);
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return fail(VOX_EINVAL, "%s: softmax_scale %g must be positive and finite", fn, (double)softmax_scale);
  return VOX_OK;
}
}  // namespace

extern "C" {

size_t vox_decode_scores_bytes(int batch, int max_blocks, int block_size, int num_heads) {
  if (batch <= 0 || max_blocks <= 0 || block_size <= 0 || num_heads <= 0) return 0;
  const int slice = batch < vox::kMaxSeqPerLaunch ? batch : vox::kMaxSeqPerLaunch;
  const size_t steps = ((size_t)max_blocks * block_size + 15) / 16;
  return (size_t)slice * steps * num_heads * 16 * 4;
}

}  // extern "C"

namespace {
int decode_attn_weights(const char* fn, bool fp4, const void* q, int64_t q_row_stride, const void* key, const void* value,
                            int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping, void* k_cache,
                            void* v_cache, int64_t num_blocks, int block_size, const int32_t* block_tables,
                            int64_t bt_stride, int max_blocks, const int32_t* context_lens, int batch, int num_heads,
                            int num_kv_heads, int head_dim, float softmax_scale, float* key_weights,
                            const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width, void* scores,
                            size_t scores_bytes, int plan, void* workspace, size_t workspace_bytes, void* out,
                            void* stream) {
  if (batch < 0) return fail(VOX_EINVAL, "%s: batch < 0", fn);
  if (plan != VOX_PLAN_NONE && plan != VOX_PLAN_RECORD && plan != VOX_PLAN_REUSE)
    return fail(VOX_EINVAL, "%s: plan mode %d", fn, plan);
  if (batch == 0) return VOX_OK;
  int st = weights_setup(fn, key_weights, num_weight_rows, weight_width, softmax_scale);
  if (st == VOX_OK && fp4) st = fp4_cache(fn, k_cache, v_cache, num_blocks, block_size, num_kv_heads, head_dim);
  if (st == VOX_OK && fp4) st = fp4_softmax(fn, softmax_scale);
  if (st != VOX_OK) return st;
  if ((key == nullptr) != (value == nullptr) || (key == nullptr) != (slot_mapping == nullptr))
    return fail(VOX_EINVAL, "%s: key, value and slot_mapping go together", fn);
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key && (key_row_stride < row || value_row_stride < row || key_row_stride % 8 || value_row_stride % 8 ||
              !aligned16(key) || !aligned16(value)))
    return fail(VOX_EINVAL, "%s: key / value rows must be 16-byte aligned, strides multiples of 8 elements and at least "
                            "num_kv_heads * head_dim", fn);
  vox::DecodeArgs a;
  st = decode_setup(q, q_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride, max_blocks,
                    context_lens, batch, num_heads, num_kv_heads, head_dim, softmax_scale, workspace, workspace_bytes, out,
                    &a);
  if (st != VOX_OK) return st;
  const size_t need = vox_decode_scores_bytes(batch, max_blocks, block_size, num_heads);
  if (!scores || !aligned16(scores) || scores_bytes < need)
    return fail(VOX_EINVAL, "%s: scores of %zu bytes (16-byte aligned), %zu needed", fn, scores_bytes, need);
  if (key) {
    a.slot_mapping = slot_mapping;
    a.new_k = (const uint16_t*)key;
    a.new_v = (const uint16_t*)value;
    a.new_k_stride = key_row_stride;
    a.new_v_stride = value_row_stride;
  }
  a.scores = (float*)scores;
  a.weights = key_weights;
  a.weight_rows = weight_rows;
  a.weight_row_count = num_weight_rows;
  a.weight_width = weight_width;
  a.weight_reach = weight_width;
  return launch_decode_slices(a, batch, num_kv_heads, plan, workspace, (hipStream_t)stream,
                              fp4 ? vox::launch_decode_weights_fp4 : vox::launch_decode_weights);
}
}  // namespace

extern "C" {

int vox_decode_attn_weights(const void* q, int64_t q_row_stride, const void* key, const void* value,
                            int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping, void* k_cache,
                            void* v_cache, int64_t num_blocks, int block_size, const int32_t* block_tables,
                            int64_t bt_stride, int max_blocks, const int32_t* context_lens, int batch, int num_heads,
                            int num_kv_heads, int head_dim, float softmax_scale, float* key_weights,
                            const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width, void* scores,
                            size_t scores_bytes, int plan, void* workspace, size_t workspace_bytes, void* out,
                            void* stream) {
  return decode_attn_weights("decode_attn_weights", false, q, q_row_stride, key, value, key_row_stride, value_row_stride, slot_mapping, k_cache, v_cache,
                             num_blocks, block_size, block_tables, bt_stride, max_blocks, context_lens, batch, num_heads,
                             num_kv_heads, head_dim, softmax_scale, key_weights, weight_rows, num_weight_rows, weight_width,
                             scores, scores_bytes, plan, workspace, workspace_bytes, out, stream);
}

int vox_decode_attn_weights_fp4(const void* q, int64_t q_row_stride, const void* key, const void* value,
                            int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping, void* k_cache,
                            void* v_cache, int64_t num_blocks, int block_size, const int32_t* block_tables,
                            int64_t bt_stride, int max_blocks, const int32_t* context_lens, int batch, int num_heads,
                            int num_kv_heads, int head_dim, float softmax_scale, float* key_weights,
                            const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width, void* scores,
                            size_t scores_bytes, int plan, void* workspace, size_t workspace_bytes, void* out,
                            void* stream) {
  return decode_attn_weights("decode_attn_weights_fp4", true, q, q_row_stride, key, value, key_row_stride, value_row_stride, slot_mapping, k_cache, v_cache,
                             num_blocks, block_size, block_tables, bt_stride, max_blocks, context_lens, batch, num_heads,
                             num_kv_heads, head_dim, softmax_scale, key_weights, weight_rows, num_weight_rows, weight_width,
                             scores, scores_bytes, plan, workspace, workspace_bytes, out, stream);
}

namespace {
// Scratch of a varlen call that adds to key weights, each part 256-byte aligned: lse [num_tokens, num_heads], then the sums of
// the sequences that have several parts [places, num_kv_heads, max_k], at most twice as many places as parts fit the call's rows
struct WeightsScratch {
  int part_rows, parts;
  size_t partials, total;
};
WeightsScratch weights_scratch(int64_t num_tokens, int max_q, int max_k, int num_heads, int num_kv_heads) {
  WeightsScratch s;
  const int group = num_heads / num_kv_heads;
  s.part_rows = vox::key_weights_part_rows(num_tokens, max_q, max_k, group, num_kv_heads);
  s.parts = (int)(((int64_t)max_q * group + s.part_rows - 1) / s.part_rows);
  s.partials = round256((size_t)num_tokens * num_heads * 4);
  const size_t places = 2 * (size_t)(num_tokens * group / s.part_rows);
  s.total = s.partials + (s.parts > 1 ? round256(places * num_kv_heads * (size_t)max_k * 4) : 0);
  return s;
}
}  // namespace

size_t vox_prefill_weights_bytes(int64_t num_tokens, int batch, int max_seqlen_q, int max_seqlen_k, int num_heads,
                                 int num_kv_heads) {
  if (num_tokens <= 0 || batch <= 0 || max_seqlen_q <= 0 || max_seqlen_k < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads)
    return 0;
  return weights_scratch(num_tokens, max_seqlen_q, max_seqlen_k, num_heads, num_kv_heads).total;
}

}  // extern "C"

namespace {
int prefill_attn_weights(const char* fn, bool fp4, const void* q, int64_t q_row_stride, const void* key, const void* value,
                             int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                             int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                             int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                             int max_seqlen_q, int max_seqlen_k, int64_t num_tokens, int num_heads, int num_kv_heads,
                             int head_dim, float softmax_scale, float* key_weights, const int32_t* weight_rows,
                             int64_t num_weight_rows, int64_t weight_width, void* scratch,
                             size_t scratch_bytes, void* scores, size_t scores_bytes, int plan, void* workspace,
                             size_t workspace_bytes, void* out, int64_t out_row_stride, void* stream) {
  if (batch < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 || num_tokens < 0)
    return fail(VOX_EINVAL, "%s: negative batch, max_seqlen_q, max_seqlen_k or num_tokens", fn);
  if (batch == 0 || max_seqlen_q == 0 || num_tokens == 0) return VOX_OK;
  if (!cu_seqlens_q || !cu_seqlens_k || !out) return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  int st = weights_setup(fn, key_weights, num_weight_rows, weight_width, softmax_scale);
  if (st != VOX_OK) return st;
  if (out_row_stride < (int64_t)num_heads * head_dim || out_row_stride % 4 || ((uintptr_t)out & 7u))
    return fail(VOX_EINVAL, "%s: bad out row stride or alignment", fn);
  if (batch > 65535 || num_kv_heads > 65535) return fail(VOX_EINVAL, "%s: more than 65535 sequences or kv heads", fn);
  if (q_row_stride >= (1 << 24)) return fail(VOX_EINVAL, "%s: q row stride must be below 2^24 elements", fn);
  if (block_tables && (block_size <= 0 || block_size % 64))
    return fail(VOX_EINVAL, "%s: block_size %d must be a positive multiple of 64", fn, block_size);
  if (block_tables && (int64_t)max_blocks * block_size > (1 << 30))
    return fail(VOX_EINVAL, "%s: block table too wide", fn);
  if (fp4) {
    if (!block_tables) return fail(VOX_EINVAL, "%s: null pointer argument", fn);
    st = fp4_cache(fn, k_cache, v_cache, num_blocks, block_size, num_kv_heads, head_dim);
    if (st == VOX_OK) st = fp4_softmax(fn, softmax_scale);
    if (st != VOX_OK) return st;
  }
  vox::KeyWeightsArgs k{};
  st = prefill_setup(fn, q, q_row_stride, key, value, key_row_stride, value_row_stride, k_cache, v_cache, num_blocks,
                     block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q, 0, 0,
                     num_heads, num_kv_heads, head_dim, softmax_scale, 1, &k.a);
  if (st != VOX_OK) return st;
  k.a.out = (uint16_t*)out;
  k.a.out_row_stride = out_row_stride;
  k.a.row_limit = num_tokens;
  // (rows, keys and work items are counted in 32 bits)
  const int64_t slice = batch < vox::kMaxSeqPerLaunch ? batch : vox::kMaxSeqPerLaunch;
  if ((int64_t)max_seqlen_q * k.a.group > (1 << 30) || max_seqlen_k > (1 << 30) ||
      ((int64_t)max_seqlen_k / 128 + 1) * 16 * num_kv_heads * slice > INT32_MAX)
    return fail(VOX_EINVAL, "%s: max_seqlen_q %d or max_seqlen_k %d too large", fn, max_seqlen_q, max_seqlen_k);
  const WeightsScratch ws = weights_scratch(num_tokens, max_seqlen_q, max_seqlen_k, num_heads, num_kv_heads);
  if (!scratch || !aligned16(scratch) || scratch_bytes < ws.total)
    return fail(VOX_EINVAL, "%s: scratch of %zu bytes (16-byte aligned), %zu needed", fn, scratch_bytes, ws.total);
  k.fp4 = fp4;
  k.a.lse = (float*)scratch;
  k.weights = key_weights;
  k.rows = weight_rows;
  k.row_count = num_weight_rows;
  k.width = weight_width;
  k.max_q = max_seqlen_q;
  k.max_k = max_seqlen_k;
  k.part_rows = ws.part_rows;
  k.max_parts = ws.parts;
  k.partials = (float*)((char*)scratch + ws.partials);
  // with the workspace the one-query sequences run on the decode kernels, which spread a long context over every CU
  const bool decodes = varlen_decode_rows(k.a, workspace, num_kv_heads);
  vox::DecodeArgs d{};
  if (decodes) {
    st = check_varlen_workspace(fn, batch, plan, workspace, workspace_bytes);
    if (st != VOX_OK) return st;
    const size_t need = vox_decode_scores_bytes(batch, max_blocks, block_size, num_heads);
    if (!scores || !aligned16(scores) || scores_bytes < need)
      return fail(VOX_EINVAL, "%s: scores of %zu bytes (16-byte aligned), %zu needed", fn, scores_bytes, need);
    k.a.skip_single = 1;
    d = varlen_decode_args(k.a, q_row_stride, num_blocks, num_heads, num_kv_heads);
    d.scores = (float*)scores;
    d.weights = key_weights;
    d.weight_rows = weight_rows;
    d.weight_row_count = num_weight_rows;
    d.weight_width = weight_width;
    d.weight_reach = weight_width < max_seqlen_k ? weight_width : max_seqlen_k;  // (as the chunk's kernels leave them out)
  }
  const hipStream_t s = (hipStream_t)stream;
  if (!decodes || max_seqlen_q > 1) {
    st = hip_status((fp4 ? vox::launch_prefill_lse_fp4 : vox::launch_prefill_lse)(k.a, max_seqlen_q, s),
                    "prefill_attn_weights launch");
    if (st == VOX_OK) st = hip_status(vox::launch_key_weights(k, s), "prefill_attn_weights sums launch");
    if (st != VOX_OK) return st;
  }
  return decodes ? launch_decode_slices(d, batch, num_kv_heads, plan, workspace, s,
                                        fp4 ? vox::launch_decode_weights_fp4 : vox::launch_decode_weights)
                 : VOX_OK;
}
}  // namespace

extern "C" {

int vox_prefill_attn_weights(const void* q, int64_t q_row_stride, const void* key, const void* value,
                             int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                             int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                             int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                             int max_seqlen_q, int max_seqlen_k, int64_t num_tokens, int num_heads, int num_kv_heads,
                             int head_dim, float softmax_scale, float* key_weights, const int32_t* weight_rows,
                             int64_t num_weight_rows, int64_t weight_width, void* scratch,
                             size_t scratch_bytes, void* scores, size_t scores_bytes, int plan, void* workspace,
                             size_t workspace_bytes, void* out, int64_t out_row_stride, void* stream) {
  return prefill_attn_weights("prefill_attn_weights", false, q, q_row_stride, key, value, key_row_stride,
                              value_row_stride, k_cache, v_cache, num_blocks, block_size, block_tables, bt_stride,
                              max_blocks, cu_seqlens_q, cu_seqlens_k, batch, max_seqlen_q, max_seqlen_k, num_tokens,
                              num_heads, num_kv_heads, head_dim, softmax_scale, key_weights, weight_rows,
                              num_weight_rows, weight_width, scratch, scratch_bytes, scores, scores_bytes, plan,
                              workspace, workspace_bytes, out, out_row_stride, stream);
}

int vox_prefill_attn_weights_fp4(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                 int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                                 int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                                 int max_seqlen_q, int max_seqlen_k, int64_t num_tokens, int num_heads,
                                 int num_kv_heads, int head_dim, float softmax_scale, float* key_weights,
                                 const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width,
                                 void* scratch, size_t scratch_bytes, void* scores, size_t scores_bytes, int plan,
                                 void* workspace, size_t workspace_bytes, void* out, int64_t out_row_stride,
                                 void* stream) {
  return prefill_attn_weights("prefill_attn_weights_fp4", true, q, q_row_stride, nullptr, nullptr, 0, 0, k_cache,
                              v_cache, num_blocks, block_size, block_tables, bt_stride, max_blocks, cu_seqlens_q,
                              cu_seqlens_k, batch, max_seqlen_q, max_seqlen_k, num_tokens, num_heads, num_kv_heads,
                              head_dim, softmax_scale, key_weights, weight_rows, num_weight_rows, weight_width,
                              scratch, scratch_bytes, scores, scores_bytes, plan, workspace, workspace_bytes, out,
                              out_row_stride, stream);
}

int vox_clear_key_weights(float* key_weights, const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width,
                          int num_kv_heads, const int32_t* cu_seqlens_new, const int32_t* cu_seqlens_k, int batch,
                          int max_keys, int max_tokens, void* stream) {
  const char* fn = "clear_key_weights";
  if (batch < 0 || max_keys < 0 || max_tokens < 0) return fail(VOX_EINVAL, "%s: negative batch, max_keys or max_tokens", fn);
  if (batch == 0 || max_keys == 0 || max_tokens == 0) return VOX_OK;
  if (!key_weights || ((uintptr_t)key_weights & 3u)) return fail(VOX_EINVAL, "%s: null or unaligned key_weights", fn);
  if (num_weight_rows <= 0 || weight_width <= 0) return fail(VOX_EINVAL, "%s: empty key_weights", fn);
  if (!cu_seqlens_new || !cu_seqlens_k) return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  if (num_kv_heads <= 0 || num_kv_heads > 65535 || batch > 65535)
    return fail(VOX_EINVAL, "%s: at most 65535 sequences and kv heads", fn);
  vox::ClearWeightsArgs a{};
  a.weights = key_weights;
  a.rows = weight_rows;
  a.row_count = num_weight_rows;
  a.width = weight_width;
  a.num_heads = num_kv_heads;
  a.cu_new = cu_seqlens_new;
  a.cu_k = cu_seqlens_k;
  a.batch = batch;
  a.max_keys = max_keys;
  a.max_tokens = max_tokens;
  return hip_status(vox::launch_clear_new_weights(a, (hipStream_t)stream), "clear_key_weights launch");
}

int vox_evict_kv_tokens(void* kv, int64_t num_layers, int64_t num_blocks, int block_size, int num_kv_heads, int head_bytes,
                        int scale_bytes, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                        const int32_t* context_lens, int batch, float* key_weights, const int32_t* weight_rows,
                        int64_t num_weight_rows, int64_t weight_width, int budget, int sinks, int recent,
                        const int32_t* into, int64_t into_stride, int32_t* moves, int32_t* new_tables, int32_t* new_lens,
                        void* stream) {
  const char* fn = "evict_kv_tokens";
  if (batch < 0 || num_layers < 0) return fail(VOX_EINVAL, "%s: negative count", fn);
  if (batch == 0 || num_layers == 0) return VOX_OK;
  if (!kv || !block_tables || !context_lens || !key_weights || !moves || !new_tables || !new_lens)
    return fail(VOX_EINVAL, "%s: null pointer argument", fn);
  if (block_size <= 0 || num_blocks <= 0 || num_blocks > INT32_MAX / block_size)
    return fail(VOX_EINVAL, "%s: cache of %lld blocks of %d tokens", fn, (long long)num_blocks, block_size);
  if (num_kv_heads <= 0 || head_bytes <= 0 || head_bytes % 16 || head_bytes > 16 * 256 ||
      (scale_bytes != 0 && scale_bytes != 4))
    return fail(VOX_EINVAL, "%s: %d kv heads of %d and %d bytes (multiples of 16 up to 4096, and 0 or 4)", fn, num_kv_heads,
                head_bytes, scale_bytes);
  const int64_t block_bytes = (int64_t)block_size * num_kv_heads * (head_bytes + scale_bytes);
  if (!aligned16(kv) || block_bytes % 16 || ((uintptr_t)moves & 7u))
    return fail(VOX_EINVAL, "%s: kv and its blocks must be 16-byte aligned, moves 8-byte aligned", fn);
  if (max_blocks <= 0 || bt_stride < max_blocks || (int64_t)max_blocks * block_size > (1 << 30))
    return fail(VOX_EINVAL, "%s: bad block table shape", fn);
  if (into && into_stride < max_blocks) return fail(VOX_EINVAL, "%s: bad shape of the new blocks' table", fn);
  if (num_weight_rows <= 0 || weight_width < (int64_t)max_blocks * block_size)
    return fail(VOX_EINVAL, "%s: key_weights of %lld rows of %lld, the tables reach %lld tokens", fn,
                (long long)num_weight_rows, (long long)weight_width, (long long)max_blocks * block_size);
  if (budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return fail(VOX_EINVAL, "%s: budget %d must be positive and hold sinks %d and recent %d", fn, budget, sinks, recent);
  if (batch > 65535 || num_kv_heads > 65535 || num_layers > 32767)
    return fail(VOX_EINVAL, "%s: at most 65535 sequences and kv heads and 32767 layers", fn);
  const int64_t reach = (int64_t)max_blocks * block_size;
  vox::EvictArgs a{};
  a.kv = (uint8_t*)kv;
  a.layers = (int)num_layers;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.num_heads = num_kv_heads;
  a.head_bytes = head_bytes;
  a.scale_bytes = scale_bytes;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks;
  a.context_lens = context_lens;
  a.batch = batch;
  a.weights = key_weights;
  a.rows = weight_rows;
  a.row_count = num_weight_rows;
  a.width = weight_width;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.into = into;
  a.into_stride = into_stride;
  a.moves = (int2*)moves;
  a.kept = budget < reach ? budget : reach;
  a.new_tables = new_tables;
  a.new_lens = new_lens;
  return hip_status(vox::launch_evict(a, (hipStream_t)stream), "evict_kv_tokens launch");
}

}  // extern "C"
