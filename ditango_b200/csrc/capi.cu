// C ABI of the library (declared in include/ditango_b200.h): argument checking, TMA tensor-map
// construction and kernel launches.  No entry point allocates device memory.
#include "../../include/ditango_b200.h"

#include "flash_fwd_sm100.cuh"
#include "flash_paged.cuh"
#include "flash_window.cuh"
#include "drift_stats.cuh"
#include "errors.cuh"
#include "merge_rows.cuh"
#include "merge_states.cuh"
#include "norm_mod.cuh"
#include "norm_rope.cuh"
#include "norm_rope_grid.cuh"
#include "pages.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <mutex>

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

// Device status word written by kernels whose bounded waits ran out.
__device__ int g_status_word;

// First code wins, as for codes reported by the kernels themselves.
__global__ void post_status_kernel(int* word, int code) { atomicCAS(word, 0, code); }

struct DeviceInfo {
  bool probed = false;
  int cc_major = 0;
  int sm_count = 0;
  int* status_ptr = nullptr;
};
DeviceInfo g_dev[64];
std::mutex g_mu;

int device_info(DeviceInfo** out) {
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= 64) return fail(DTB_ERR_CUDA, "cudaGetDevice failed: %s", cudaGetErrorString(e));
  std::lock_guard<std::mutex> lk(g_mu);
  DeviceInfo& d = g_dev[dev];
  if (!d.probed) {
    e = cudaDeviceGetAttribute(&d.cc_major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "device query failed: %s", cudaGetErrorString(e));
    if (d.cc_major == 10) {
      void* p = nullptr;
      e = cudaGetSymbolAddress(&p, g_status_word);
      if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "cudaGetSymbolAddress failed: %s", cudaGetErrorString(e));
      d.status_ptr = static_cast<int*>(p);
    }
    d.probed = true;
  }
  if (d.cc_major != 10) return fail(DTB_ERR_DEVICE, "device %d has compute capability %d.x; sm_100a kernels need 10.x", dev, d.cc_major);
  *out = &d;
  return DTB_OK;
}

}  // namespace

namespace dtb {

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int require_sm100() {
  DeviceInfo* d = nullptr;
  return device_info(&d);
}

}  // namespace dtb

namespace {

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

int load_encoder() {
  static std::once_flag once;
  static cudaError_t err = cudaSuccess;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    err = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
    if (err == cudaSuccess && qres == cudaDriverEntryPointSuccess) g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (g_encode == nullptr) return fail(DTB_ERR_CUDA, "cuTensorMapEncodeTiled not available: %s", cudaGetErrorString(err));
  return DTB_OK;
}

// 2-D bf16 view [rows, width] with a row pitch of tok_stride elements; boxes of 64 x box_rows elements
// (128 bytes x box_rows rows) written to shared memory with the 128-byte swizzle.
int make_tile_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t width, int64_t tok_stride, int box_rows,
                  const char* what) {
  cuuint64_t gdim[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
  cuuint64_t gstride[1] = {static_cast<cuuint64_t>(tok_stride) * 2};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = g_encode(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DTB_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", what, static_cast<int>(r));
  return DTB_OK;
}

// 3-D bf16 view of tokens x batch rows of `width` channels for boxes of 64 channels x 128 tokens, the outer axis of the smaller
// stride first; *batch_first says which one that is.
int make_token_map(CUtensorMap* tm, const void* base, int64_t width, int64_t tokens, int64_t tok_stride, int64_t batch, int64_t batch_stride,
                   int* batch_first, const char* what) {
  const bool swap = batch > 1 && batch_stride < tok_stride;
  const int64_t inner = swap ? batch : tokens, outer = swap ? tokens : batch;
  const int64_t inner_stride = swap ? batch_stride : tok_stride, outer_stride = swap ? tok_stride : batch > 1 ? batch_stride : tok_stride;
  cuuint64_t gdim[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  cuuint64_t gstride[2] = {static_cast<cuuint64_t>(inner_stride) * 2, static_cast<cuuint64_t>(outer_stride) * 2};
  cuuint32_t box[3] = {64, swap ? 1u : 128u, swap ? 128u : 1u};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = g_encode(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  *batch_first = swap ? 1 : 0;
  if (r != CUDA_SUCCESS) return fail(DTB_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", what, static_cast<int>(r));
  return DTB_OK;
}

// 4-D bf16 view of a pool of pages [channel, token, head, page] for boxes of 64 channels x box_rows tokens, of token and head the one with the
// smaller stride first; *head_first says which one that is.
int make_page_map(CUtensorMap* tm, const void* base, int64_t head_dim, int64_t page_size, int64_t tok_stride, int64_t heads, int64_t head_stride,
                  int64_t pages, int64_t page_stride, int box_rows, int* head_first, const char* what) {
  const bool swap = head_stride < tok_stride;
  const int64_t inner = swap ? heads : page_size, outer = swap ? page_size : heads;
  cuuint64_t gdim[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer), static_cast<cuuint64_t>(pages)};
  cuuint64_t gstride[3] = {static_cast<cuuint64_t>(swap ? head_stride : tok_stride) * 2, static_cast<cuuint64_t>(swap ? tok_stride : head_stride) * 2,
                           static_cast<cuuint64_t>(page_stride) * 2};
  cuuint32_t box[4] = {64, swap ? 1u : static_cast<cuuint32_t>(box_rows), swap ? static_cast<cuuint32_t>(box_rows) : 1u, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = g_encode(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  *head_first = swap ? 1 : 0;
  if (r != CUDA_SUCCESS) return fail(DTB_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", what, static_cast<int>(r));
  return DTB_OK;
}

// 4-D bf16 view of queries [channel, head, token, batch], a token's heads dense, for boxes of 64 channels x `pack` heads x 128 / pack tokens.
int make_query_map(CUtensorMap* tm, const void* base, int64_t head_dim, int64_t heads, int64_t tokens, int64_t tok_stride, int64_t batch, int64_t batch_stride,
                   int pack, int* batch_first) {
  const bool swap = batch > 1 && batch_stride < tok_stride;
  const int64_t inner = swap ? batch : tokens, outer = swap ? tokens : batch;
  const int64_t inner_stride = swap ? batch_stride : tok_stride, outer_stride = swap ? tok_stride : batch > 1 ? batch_stride : tok_stride;
  cuuint64_t gdim[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  cuuint64_t gstride[3] = {static_cast<cuuint64_t>(head_dim) * 2, static_cast<cuuint64_t>(inner_stride) * 2, static_cast<cuuint64_t>(outer_stride) * 2};
  const cuuint32_t rows = 128 / static_cast<cuuint32_t>(pack);
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(pack), swap ? 1u : rows, swap ? rows : 1u};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = g_encode(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  *batch_first = swap ? 1 : 0;
  if (r != CUDA_SUCCESS) return fail(DTB_ERR_CUDA, "cuTensorMapEncodeTiled(q) failed with CUresult %d", static_cast<int>(r));
  return DTB_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Encoded tensor maps, kept per (base pointer, rows, width, pitch, box rows).  The attention path calls
// with the same few buffers over and over (persistent receive buffers, a layer's q / k / v of a fixed shape),
// so most launches find their three maps here instead of going through the driver's encoder.
struct MapKey {
  const void* base;
  int64_t rows, width, tok_stride;
  int box_rows;
  bool operator==(const MapKey& o) const {
    return base == o.base && rows == o.rows && width == o.width && tok_stride == o.tok_stride && box_rows == o.box_rows;
  }
};
constexpr int kMapCacheSize = 64;
struct MapEntry {
  MapKey key;
  CUtensorMap map;
  bool used = false;
};
MapEntry g_maps[kMapCacheSize];
std::mutex g_map_mu;

int cached_tile_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t width, int64_t tok_stride, int box_rows,
                    const char* what) {
  const MapKey key{base, rows, width, tok_stride, box_rows};
  const size_t h = (reinterpret_cast<uintptr_t>(base) >> 8) * 0x9E3779B97F4A7C15ull + static_cast<size_t>(rows) * 31 +
                   static_cast<size_t>(box_rows);
  const int slot = static_cast<int>((h >> 20) % kMapCacheSize);
  {
    std::lock_guard<std::mutex> lk(g_map_mu);
    if (g_maps[slot].used && g_maps[slot].key == key) {
      *tm = g_maps[slot].map;
      return DTB_OK;
    }
  }
  int rc = make_tile_map(tm, base, rows, width, tok_stride, box_rows, what);
  if (rc != DTB_OK) return rc;
  std::lock_guard<std::mutex> lk(g_map_mu);
  g_maps[slot].key = key;
  g_maps[slot].map = *tm;
  g_maps[slot].used = true;
  return DTB_OK;
}

}  // namespace

extern "C" {

DTB_API int dtb_version(void) { return 100; }

DTB_API const char* dtb_last_error(void) { return g_err; }

DTB_API int dtb_device_supported(void) {
  DeviceInfo* d = nullptr;
  return device_info(&d);
}

DTB_API int dtb_read_status(void* stream) {
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int host = 0;
  cudaError_t e = cudaMemcpyAsync(&host, d->status_ptr, sizeof(int), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "status read failed: %s", cudaGetErrorString(e));
  if (host != 0) {
    e = cudaMemsetAsync(d->status_ptr, 0, sizeof(int), s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "status clear failed: %s", cudaGetErrorString(e));
    fail(host, "a kernel gave up on a bounded wait (code %d)", host);
  }
  return host;
}

DTB_API int dtb_peek_status_async(int* host_word, void* stream) {
  if (!host_word) return fail(DTB_ERR_ARG, "dtb_peek_status_async: null destination");
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  cudaError_t e = cudaMemcpyAsync(host_word, d->status_ptr, sizeof(int), cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "status copy failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_post_status(int code, void* stream) {
  if (code <= 0) return fail(DTB_ERR_ARG, "dtb_post_status: code must be positive, got %d", code);
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  post_status_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(d->status_ptr, code);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "status write failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_ipc_export_mem(const void* dev_ptr, void* handle64, int64_t* offset) {
  if (!dev_ptr || !handle64 || !offset) return fail(DTB_ERR_ARG, "dtb_ipc_export_mem: null argument");
  static PFN_cuMemGetAddressRange_v3020 get_range = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &fn, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      get_range = reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(fn);
  });
  if (get_range == nullptr) return fail(DTB_ERR_CUDA, "dtb_ipc_export_mem: cuMemGetAddressRange not available");
  CUdeviceptr base = 0;
  size_t size = 0;
  CUresult r = get_range(&base, &size, reinterpret_cast<CUdeviceptr>(dev_ptr));
  if (r != CUDA_SUCCESS) return fail(DTB_ERR_CUDA, "dtb_ipc_export_mem: address range query failed with CUresult %d", static_cast<int>(r));
  cudaIpcMemHandle_t h;
  cudaError_t e = cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "cudaIpcGetMemHandle failed: %s", cudaGetErrorString(e));
  static_assert(sizeof(h) == 64, "handle size");
  memcpy(handle64, &h, sizeof(h));
  *offset = static_cast<int64_t>(reinterpret_cast<CUdeviceptr>(dev_ptr) - base);
  return DTB_OK;
}

DTB_API int dtb_ipc_open_mem(const void* handle64, void** base_ptr) {
  if (!handle64 || !base_ptr) return fail(DTB_ERR_ARG, "dtb_ipc_open_mem: null argument");
  cudaIpcMemHandle_t h;
  memcpy(&h, handle64, sizeof(h));
  cudaError_t e = cudaIpcOpenMemHandle(base_ptr, h, cudaIpcMemLazyEnablePeerAccess);
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "cudaIpcOpenMemHandle failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_ipc_close_mem(void* base_ptr) {
  if (!base_ptr) return DTB_OK;
  cudaError_t e = cudaIpcCloseMemHandle(base_ptr);
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "cudaIpcCloseMemHandle failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_peer_copy_async(void* dst, const void* src, int64_t bytes, void* stream) {
  if (bytes < 0 || (bytes > 0 && (!dst || !src))) return fail(DTB_ERR_ARG, "dtb_peer_copy_async: bad argument");
  if (bytes == 0) return DTB_OK;
  cudaError_t e = cudaMemcpyAsync(dst, src, static_cast<size_t>(bytes), cudaMemcpyDefault, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "peer copy failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

// Which launches take the kernel whose CTAs stay (D = 64).  It saves what a CTA spends in front of its key loop and behind it, which
// shows as soon as some SM gets a second block.  us, a CTA per block -> CTAs that stay, for an fp32 result / a bf16 result:
//    74 heads x 512 x 2222 (148 blocks)    32.9 / 32.4 -> 34.8 / 33.0      48 x 2 x 2222 x 2222     179 / 189 -> 162 / 170
//   100 heads x 512 x 2222 (200)           61.2 / 60.0 -> 59.0 / 57.5      48 x 2 x 8888 x 8888    2470 / 2430 -> 2396 / 2381
//   150 heads x 512 x 128  (300)           20.6 / 18.6 -> 17.5 / 15.2      24 x 17776 x 17776      2411 / 2478 -> 2390 / 2460
//   150 heads x 512 x 2222                 90.8 / 92.3 -> 84.1 / 85.0      24 x 24000 x 24000      4353 / 4342 -> 4341 / 4337
//   150 heads x 512 x 8192                  312 / 301 -> 293 / 293         24 x 35552 x 35552      9380 / 9336 -> 9362 / 9360
// and from about 24000 keys on the two are level, hence kStayMaxKeys.
// A launch that overlaps the one before it needs more blocks: its first CTAs, on the SMs that fall free early, claim blocks while
// that launch still runs, and up to kWork = 4 of them where an item is short (the ring for K and V holds four key tiles, so that
// longer ones hold a CTA back), blocks that the SMs which fall free later then miss.  us, folded into a state, overlapping:
//   512 queries x  128 keys, 300 / 480 / 592 / 700 blocks     22.7 / 35.1 / 40.6 / 54.2 -> 37.0 / 41.2 / 40.3 / 46.3
//            (without a state, 400 / 480 / 592                17.8 / 22.4 / 27.1 -> 22.7 / 22.4 / 23.2)
//                  256 keys, 300 / 400 / 480 / 592            25.5 / 32.7 / 38.4 / 47.5 -> 37.5 / 37.4 / 35.6 / 43.1
//                  384 keys, 300 / 400 / 480                  28.3 / 35.8 / 45.5 -> 35.4 / 36.4 / 38.4
//                  512 keys, 288 / 300 / 400                  26.5 / 30.8 / 38.6 -> 28.0 / 28.2 / 30.8
//                 2222 keys, 190 / 250 / 300 / 444            41.2 / 60.1 / 73.1 / 115 -> 43.7 / 57.9 / 66.5 / 104
//                 8192 keys, 190 / 250 / 350 / 444             145 / 194 / 259 / 333 -> 149 / 190 / 254 / 325
// Folding a single key tile into a state without overlap is bound by the state's way through the CTA, which eight warps do faster
// than four: 4 to 9 % slower at 160 to 296 blocks of 64 and 128 keys, between 6 % slower and 5 % faster at 300 to 1776.
// `blocks` counts what holds queries: the grid of a packed launch has ceil(max_seqlen_q / 256) blocks for each sequence.  The lengths
// are only known on the device; one sequence is taken to have the maximum, and the last block of each other to be half full.
// (Blocks without queries cost less to claim than to launch: 16 x 256 queries and keys with max_seqlen_q = 4096, 24 heads,
// 59.5 -> 40.8 us.)
constexpr int kStayMaxKeys = 24576;

static bool takes_staying_kernel(int head_dim, bool packed, int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int num_heads,
                                 bool accumulate, bool overlap, int sm_count) {
  if (head_dim != 64 || seqlen_k > kStayMaxKeys) return false;
  int64_t blocks = (static_cast<int64_t>(seqlen_q) + 255) / 256 * nseg * num_heads;
  if (packed) {
    const int64_t longest = std::min<int64_t>(seqlen_q, total_q);
    const int64_t rows = (longest + 255) / 256 * 256 + (total_q - longest) + 128 * static_cast<int64_t>(nseg - 1);
    blocks = std::min(blocks, rows * num_heads / 256);
  }
  const int key_tiles = (seqlen_k + 127) / 128;
  if (overlap) return blocks > sm_count * static_cast<int64_t>(key_tiles <= 1 && accumulate ? 4 : key_tiles <= 3 ? 3 : 2);
  return blocks > sm_count && !(accumulate && key_tiles <= 1);
}

static int flash_fwd_impl(const void* q, const void* k, const void* v,
                          int64_t q_tok_stride, int64_t k_tok_stride, int64_t v_tok_stride,
                          void* out, int out_dtype, int64_t out_tok_stride,
                          float* lse, int lse_layout, int accumulate,
                          const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                          int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int64_t total_k,
                          int num_heads, int head_dim, float softmax_scale, int launch_flags, void* stream) {
  if (launch_flags & ~DTB_LAUNCH_OVERLAP_PREVIOUS) return fail(DTB_ERR_ARG, "dtb_flash_fwd: unknown launch flag 0x%x", launch_flags);
  if (!q || !k || !v || !out || !lse) return fail(DTB_ERR_ARG, "dtb_flash_fwd: null tensor pointer");
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "dtb_flash_fwd: head_dim %d not in {64, 128}", head_dim);
  if (num_heads < 1 || num_heads > 65535) return fail(DTB_ERR_ARG, "dtb_flash_fwd: num_heads %d out of range", num_heads);
  if (nseg < 1 || nseg > 65535) return fail(DTB_ERR_ARG, "dtb_flash_fwd: nseg %d out of range", nseg);
  if (seqlen_q < 0 || seqlen_k < 0 || total_q < 0 || total_k < 0) return fail(DTB_ERR_ARG, "dtb_flash_fwd: negative length");
  if (total_q >= (1ll << 31) || total_k >= (1ll << 31)) return fail(DTB_ERR_ARG, "dtb_flash_fwd: more than 2^31 tokens");
  if ((cu_seqlens_q == nullptr) != (cu_seqlens_k == nullptr)) return fail(DTB_ERR_ARG, "dtb_flash_fwd: cu_seqlens_q and cu_seqlens_k must both be given or both be null");
  if (cu_seqlens_q == nullptr && (static_cast<int64_t>(nseg) * seqlen_q > total_q || static_cast<int64_t>(nseg) * seqlen_k > total_k))
    return fail(DTB_ERR_ARG, "dtb_flash_fwd: nseg*seqlen exceeds total tokens");
  const int64_t width = static_cast<int64_t>(num_heads) * head_dim;
  if (q_tok_stride < width || k_tok_stride < width || v_tok_stride < width || out_tok_stride < width)
    return fail(DTB_ERR_ARG, "dtb_flash_fwd: token stride smaller than num_heads*head_dim");
  if ((q_tok_stride | k_tok_stride | v_tok_stride | out_tok_stride) & 7) return fail(DTB_ERR_ARG, "dtb_flash_fwd: token strides must be multiples of 8 elements");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return fail(DTB_ERR_ARG, "dtb_flash_fwd: tensor pointers must be 16-byte aligned");
  if (out_dtype != DTB_F32 && out_dtype != DTB_BF16) return fail(DTB_ERR_ARG, "dtb_flash_fwd: bad out_dtype %d", out_dtype);
  if (lse_layout != DTB_LSE_BHS && lse_layout != DTB_LSE_BSH) return fail(DTB_ERR_ARG, "dtb_flash_fwd: bad lse_layout %d", lse_layout);
  if (accumulate && out_dtype != DTB_F32) return fail(DTB_ERR_ARG, "dtb_flash_fwd: accumulate needs an fp32 state");
  if (!(softmax_scale > 0.f)) return fail(DTB_ERR_ARG, "dtb_flash_fwd: softmax_scale must be positive");
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  if (seqlen_q == 0 || total_q == 0) return DTB_OK;
  rc = load_encoder();
  if (rc != DTB_OK) return rc;

  CUtensorMap tq, tk, tv;
  // A tensor map needs at least one row; an empty key chunk never issues a load.
  const int64_t rows_k = total_k > 0 ? total_k : 1;
  const int kv_rows = dtb::flash_kv_box_rows();
  if ((rc = cached_tile_map(&tq, q, total_q, width, q_tok_stride, 128, "q")) != DTB_OK) return rc;
  if ((rc = cached_tile_map(&tk, k, rows_k, width, k_tok_stride, kv_rows, "k")) != DTB_OK) return rc;
  if ((rc = cached_tile_map(&tv, v, rows_k, width, v_tok_stride, kv_rows, "v")) != DTB_OK) return rc;

  dtb::FlashParams p;
  p.out = out;
  p.lse = lse;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.status = d->status_ptr;
  p.out_tok_stride = out_tok_stride;
  p.total_q = total_q;
  p.nseg = nseg;
  p.seqlen_q = seqlen_q;
  p.seqlen_k = seqlen_k;
  p.num_heads = num_heads;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out_dtype = out_dtype;
  p.lse_layout = lse_layout;
  p.accumulate = accumulate ? 1 : 0;
  p.overlap_previous = (launch_flags & DTB_LAUNCH_OVERLAP_PREVIOUS) ? 1 : 0;
  const bool stay = takes_staying_kernel(head_dim, cu_seqlens_q != nullptr, nseg, seqlen_q, seqlen_k, total_q, num_heads,
                                         p.accumulate != 0, p.overlap_previous != 0, d->sm_count);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = stay              ? dtb::launch_flash_persistent(tq, tk, tv, p, s)
                        : head_dim == 64  ? dtb::launch_flash<64>(tq, tk, tv, p, s)
                                          : dtb::launch_flash<128>(tq, tk, tv, p, s);
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_flash_fwd launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_flash_fwd(const void* q, const void* k, const void* v,
                  int64_t q_tok_stride, int64_t k_tok_stride, int64_t v_tok_stride,
                  void* out, int out_dtype, int64_t out_tok_stride,
                  float* lse, int lse_layout, int accumulate,
                  const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                  int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int64_t total_k,
                  int num_heads, int head_dim, float softmax_scale, void* stream) {
  return flash_fwd_impl(q, k, v, q_tok_stride, k_tok_stride, v_tok_stride, out, out_dtype, out_tok_stride, lse, lse_layout,
                        accumulate, cu_seqlens_q, cu_seqlens_k, nseg, seqlen_q, seqlen_k, total_q, total_k, num_heads,
                        head_dim, softmax_scale, 0, stream);
}

DTB_API int dtb_flash_fwd_ex(const void* q, const void* k, const void* v,
                     int64_t q_tok_stride, int64_t k_tok_stride, int64_t v_tok_stride,
                     void* out, int out_dtype, int64_t out_tok_stride,
                     float* lse, int lse_layout, int accumulate,
                     const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                     int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int64_t total_k,
                     int num_heads, int head_dim, float softmax_scale, int launch_flags, void* stream) {
  return flash_fwd_impl(q, k, v, q_tok_stride, k_tok_stride, v_tok_stride, out, out_dtype, out_tok_stride, lse, lse_layout,
                        accumulate, cu_seqlens_q, cu_seqlens_k, nseg, seqlen_q, seqlen_k, total_q, total_k, num_heads,
                        head_dim, softmax_scale, launch_flags, stream);
}

// Which kernel a launch takes, and the parts that the tiles of 128 split their keys into: what is expected to finish first.  Tiles of 128
// need a walk over the keys of a block of 256 rows for each round of blocks over the SMs, however few there are; parts shorten it where
// blocks leave SMs idle, for a merge behind them and states in fp32 (all parts run at once: with 34 tiles of keys more than a part per
// idle SM gained nothing, e.g. 24 heads of 64 with 1024 rows 57.1 us whole, 56.6 in three; longer walks were not measured so).
// Tiles of 16 rows x 16 keys are taken to be spread over all SMs, which 8 CTAs to a block of 16 rows cannot do for few key heads.
// Packed batches are not split: rows behind the last sequence have no state that a merge could leave alone.
// us in tiles of 16 / of 128 whole / in the best number of parts, each forced:
//   queries                            32                 64                 256                512                 1024
//   24 heads of 128, window 4096  22.0/66.1/26.3(6)  35.9/66.1/26.3(6)   106/67.7/31(6)      189/68.3/54(2)        -/68.9/-
//   24 heads of 128, window 512    9.9/18.8/17.0(4)  12.2/19.1/17.5(4)  27.1/20.5/22.7(4)  46.3/21.4/27.1(2)  84.3/22.1/42.1(2)
//   24 heads of 64, window 4096   14.3/54.4/22.4(6)  22.7/54.3/22.8(6)  56.4/55.4/25.5(6)   105/56.6/34.4(3)   185/57.1/56.6(3)
//   2 x 48 of 64, window 2700     29.4/41.0/39.9(3)  40.9/41.2/41.3(3)   130/45.0/50.7(3)   241/80.4/86.0(3)   473/118/157(2)
//   32 over 8 of 128, window 4096 22.2/68.6/30.6(4)  36.4/68.9/31.0(4)   127/70.6/36.5(4)   226/71.1/54.2(2)   436/72.4/95.6(2)
//   4 x 32 over 8 of 64, 1000     15.0/23.1/31.6(2)  25.0/23.2/32.6(2)  75.5/24.5/41.9(2)   146/41.5/70.3(2)   285/73.2/119(2)
//   8 over 1 of 128, window 8192  21.7/ 124/30.2(8)  22.3/ 124/30.3(8)  63.2/ 126/33.9(8)   120/ 126/36.1(8)   236/132/50.6(4)
//   4 heads of 64, window 700      5.7/16.9/13.9(8)   6.4/16.7/14.5(8)   7.4/19.7/18.3(4)   9.0/19.9/18.4(4)  12.6/19.9/18.9(4)
//   4 heads of 128, window 2000    8.6/37.3/18.3(6)  11.3/39.4/18.9(8)  15.2/41.2/24.1(6)  22.3/41.3/24.0(6)  37.3/41.7/25.6(6)
struct WindowPlan {
  int splits;               // 0: tiles of 16 rows; else tiles of 128 over the keys in that many parts
  int64_t scratch_bytes;    // for more than one part
};
static WindowPlan plan_window(int64_t nseg, int64_t seqlen_q, int64_t seqlen_k, int64_t num_heads, int64_t kv_heads, int head_dim,
                              int64_t left, int64_t right, int64_t sinks, int sm_count, bool may_split) {
  const int64_t group = num_heads / kv_heads, span = std::min(seqlen_k, left + right + sinks);
  const double small_tiles = static_cast<double>((seqlen_q * group + 15) / 16 * kv_heads * nseg) * ((span + 31) / 16);
  double best = 5. + small_tiles / (sm_count * (head_dim == 64 ? 12.8 : 7.2));
  WindowPlan plan = {0, 0};
  const int64_t blocks = (seqlen_q + 255) / 256 * num_heads * nseg, rows = nseg * seqlen_q * num_heads;
  const int64_t steps = (std::min(seqlen_k, span + std::min<int64_t>(seqlen_q, 128)) + 127) / 128;
  const double start = head_dim == 64 ? 6. : 4., block = head_dim == 64 ? 5. : 4., step = head_dim == 64 ? 1.32 : 1.8;
  for (int64_t s = 1; s < dtb::kMergeMaxStates; ++s) {
    double us = start + static_cast<double>((blocks * s + sm_count - 1) / sm_count) * (block + (steps + s - 1) / s * step);
    if (s > 1) {
      if (!may_split || seqlen_q <= 16 || s > steps || blocks * s > sm_count || nseg * s > 65535 || s * nseg * seqlen_q >= (1ll << 31)) break;
      us += 5. + 4. * std::min<int64_t>(seqlen_q, 256) / 256. + static_cast<double>(s * rows * head_dim) * 4. / 5e6;
    }
    if (us < best) {
      best = us;
      plan.splits = static_cast<int>(s);
      plan.scratch_bytes = s > 1 ? s * rows * (head_dim + 1) * 4 : 0;
    }
  }
  return plan;
}

DTB_API int64_t dtb_flash_window_scratch_bytes(int nseg, int seqlen_q, int seqlen_k, int num_heads, int num_kv_heads, int head_dim,
                                               int left, int right, int sinks) {
  if (nseg < 1 || seqlen_q < 0 || seqlen_k < 0 || num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads || (head_dim != 64 && head_dim != 128))
    return fail(DTB_ERR_ARG, "dtb_flash_window_scratch_bytes: bad shape");
  if (left < -1 || right < -1 || sinks < 0) return fail(DTB_ERR_ARG, "dtb_flash_window_scratch_bytes: window (%d, %d) or sinks %d out of range", left, right, sinks);
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  return plan_window(nseg, seqlen_q, seqlen_k, num_heads, num_kv_heads, head_dim, left < 0 ? seqlen_k : left, right < 0 ? seqlen_k : right, sinks,
                     d->sm_count, true).scratch_bytes;
}

DTB_API int dtb_flash_window(const void* q, const void* k, const void* v,
                     int64_t q_tok_stride, int64_t q_batch_stride, int64_t k_tok_stride, int64_t k_batch_stride,
                     int64_t v_tok_stride, int64_t v_batch_stride,
                     void* out, int out_dtype, float* lse, int lse_layout, int accumulate,
                     const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, const int32_t* seqlens_k,
                     int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int64_t total_k,
                     int num_heads, int num_kv_heads, int head_dim, float softmax_scale,
                     int left, int right, int sinks, int q_start, int k_start,
                     void* scratch, int64_t scratch_bytes, void* stream) {
  constexpr int kFar = 1 << 30;
  static_assert(DTB_QUERIES_LAST == dtb::kQueriesLast, "q_start");
  if (!q || !k || !v || !out || !lse) return fail(DTB_ERR_ARG, "dtb_flash_window: null tensor pointer");
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "dtb_flash_window: head_dim %d not in {64, 128}", head_dim);
  if (num_heads < 1 || num_heads > 65535 || num_kv_heads < 1 || num_heads % num_kv_heads)
    return fail(DTB_ERR_ARG, "dtb_flash_window: %d query heads over %d key heads", num_heads, num_kv_heads);
  if (nseg < 1 || nseg > 65535) return fail(DTB_ERR_ARG, "dtb_flash_window: nseg %d out of range", nseg);
  if (seqlen_q < 0 || seqlen_k < 0 || total_q < 0 || total_k < 0) return fail(DTB_ERR_ARG, "dtb_flash_window: negative length");
  if (seqlen_q >= kFar || seqlen_k >= kFar || total_q >= (1ll << 31) || total_k >= (1ll << 31)) return fail(DTB_ERR_ARG, "dtb_flash_window: too many tokens");
  if ((cu_seqlens_q == nullptr) != (cu_seqlens_k == nullptr)) return fail(DTB_ERR_ARG, "dtb_flash_window: cu_seqlens_q and cu_seqlens_k must both be given or both be null");
  if (cu_seqlens_q != nullptr && seqlens_k != nullptr) return fail(DTB_ERR_ARG, "dtb_flash_window: seqlens_k is for dense batches");
  if (cu_seqlens_q == nullptr && (static_cast<int64_t>(nseg) * seqlen_q != total_q || static_cast<int64_t>(nseg) * seqlen_k != total_k))
    return fail(DTB_ERR_ARG, "dtb_flash_window: total tokens are not nseg*seqlen");
  if (left < -1 || right < -1 || sinks < 0 || left > kFar || right > kFar || sinks > kFar) return fail(DTB_ERR_ARG, "dtb_flash_window: window (%d, %d) or sinks %d out of range", left, right, sinks);
  if ((q_start != DTB_QUERIES_LAST && (q_start < -kFar || q_start > kFar)) || k_start < -kFar || k_start > kFar)
    return fail(DTB_ERR_ARG, "dtb_flash_window: position out of range");
  const int64_t q_width = static_cast<int64_t>(num_heads) * head_dim, k_width = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (q_tok_stride < q_width || k_tok_stride < k_width || v_tok_stride < k_width) return fail(DTB_ERR_ARG, "dtb_flash_window: token stride smaller than the heads");
  if (cu_seqlens_q == nullptr && nseg > 1 && (q_batch_stride < q_width || k_batch_stride < k_width || v_batch_stride < k_width))
    return fail(DTB_ERR_ARG, "dtb_flash_window: batch stride smaller than the heads");
  if ((q_tok_stride | q_batch_stride | k_tok_stride | k_batch_stride | v_tok_stride | v_batch_stride) & 7) return fail(DTB_ERR_ARG, "dtb_flash_window: strides must be multiples of 8 elements");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return fail(DTB_ERR_ARG, "dtb_flash_window: tensor pointers must be 16-byte aligned");
  if (!aligned16(scratch)) return fail(DTB_ERR_ARG, "dtb_flash_window: scratch must be 16-byte aligned");
  if (out_dtype != DTB_F32 && out_dtype != DTB_BF16) return fail(DTB_ERR_ARG, "dtb_flash_window: bad out_dtype %d", out_dtype);
  if (lse_layout != DTB_LSE_BHS && lse_layout != DTB_LSE_BSH) return fail(DTB_ERR_ARG, "dtb_flash_window: bad lse_layout %d", lse_layout);
  if (accumulate && out_dtype != DTB_F32) return fail(DTB_ERR_ARG, "dtb_flash_window: accumulate needs an fp32 state");
  if (!(softmax_scale > 0.f)) return fail(DTB_ERR_ARG, "dtb_flash_window: softmax_scale must be positive");
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  if (seqlen_q == 0 || total_q == 0) return DTB_OK;

  dtb::WindowParams p;
  memset(&p, 0, sizeof(p));
  p.f.out = out;
  p.f.lse = lse;
  p.f.cu_q = cu_seqlens_q;
  p.f.cu_k = cu_seqlens_k;
  p.f.status = d->status_ptr;
  p.f.out_tok_stride = q_width;
  p.f.total_q = total_q;
  p.f.nseg = nseg;
  p.f.seqlen_q = seqlen_q;
  p.f.seqlen_k = seqlen_k;
  p.f.num_heads = num_heads;
  p.f.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.f.out_dtype = out_dtype;
  p.f.lse_layout = lse_layout;
  p.f.accumulate = accumulate ? 1 : 0;
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_tok = q_tok_stride;
  p.q_batch = q_batch_stride;
  p.k_tok = k_tok_stride;
  p.k_batch = k_batch_stride;
  p.v_tok = v_tok_stride;
  p.v_batch = v_batch_stride;
  p.seqlens_k = seqlens_k;
  p.kv_heads = num_kv_heads;
  p.left = left;
  p.right = right;
  p.sinks = sinks;
  p.q_start = q_start;
  p.k_start = k_start;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  const WindowPlan plan = plan_window(nseg, seqlen_q, seqlen_k, num_heads, num_kv_heads, head_dim, left < 0 ? seqlen_k : left,
                                      right < 0 ? seqlen_k : right, sinks, d->sm_count, scratch != nullptr && cu_seqlens_q == nullptr);
  if (scratch_bytes < plan.scratch_bytes)
    return fail(DTB_ERR_ARG, "dtb_flash_window: scratch of %lld bytes is smaller than the %lld needed", static_cast<long long>(scratch_bytes),
                static_cast<long long>(plan.scratch_bytes));
  if (plan.splits > 0) {
    dtb::MergeParams m;
    if (plan.splits > 1) {
      // the parts' states in scratch, merged with the state that is there into the result
      const int64_t rows = total_q * num_heads;
      float* parts = static_cast<float*>(scratch);
      memset(&m, 0, sizeof(m));
      auto add = [&](const void* o, const float* l, int layout) {
        m.outs[m.nstates] = o;
        m.lse[m.nstates] = l;
        m.out_dtype[m.nstates] = DTB_F32;
        m.lse_layout[m.nstates++] = layout;
      };
      if (accumulate) add(out, lse, lse_layout);
      for (int i = 0; i < plan.splits; ++i) add(parts + i * rows * head_dim, parts + plan.splits * rows * head_dim + i * rows, DTB_LSE_BSH);
      m.out = out_dtype == DTB_F32 ? static_cast<float*>(out) : nullptr;
      m.out_bf16 = out_dtype == DTB_BF16 ? static_cast<uint16_t*>(out) : nullptr;
      m.lse_out = lse;
      m.lse_out_layout = lse_layout;
      m.rows = rows;
      m.H = num_heads;
      m.S = seqlen_q;
      m.status = d->status_ptr;
      p.f.out = parts;
      p.f.lse = parts + plan.splits * rows * head_dim;
      p.f.out_dtype = DTB_F32;
      p.f.lse_layout = DTB_LSE_BSH;
      p.f.accumulate = 0;
    }
    p.splits = plan.splits;
    if ((rc = load_encoder()) != DTB_OK) return rc;
    const bool packed = cu_seqlens_q != nullptr;
    const int64_t q_tokens = packed ? total_q : seqlen_q, k_tokens = packed ? total_k : seqlen_k, batch = packed ? 1 : nseg;
    CUtensorMap tq, tk, tv;
    // (a tensor map needs a row; without keys none is loaded)
    if ((rc = make_token_map(&tq, q, q_width, q_tokens, q_tok_stride, batch, q_batch_stride, &p.q_batch_first, "q")) != DTB_OK ||
        (rc = make_token_map(&tk, k, k_width, std::max<int64_t>(k_tokens, 1), k_tok_stride, batch, k_batch_stride, &p.k_batch_first, "k")) != DTB_OK ||
        (rc = make_token_map(&tv, v, k_width, std::max<int64_t>(k_tokens, 1), v_tok_stride, batch, v_batch_stride, &p.v_batch_first, "v")) != DTB_OK)
      return rc;
    e = head_dim == 64 ? dtb::launch_window_tiles<64>(tq, tk, tv, p, s) : dtb::launch_window_tiles<128>(tq, tk, tv, p, s);
    if (e == cudaSuccess && plan.splits > 1) e = dtb::launch_merge(m, head_dim, d->sm_count, s);
  } else {
    e = head_dim == 64 ? dtb::launch_window_rows<64>(p, d->sm_count, s) : dtb::launch_window_rows<128>(p, d->sm_count, s);
  }
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_flash_window launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

// Pages hold a power of two of tokens, 16 at least; returns the exponent, or -1.
static int page_shift_of(int page_size) {
  if (page_size < 16 || page_size > (1 << 20) || (page_size & (page_size - 1))) return -1;
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  return shift;
}

// What the table's rows and the pool may be: [streams, columns] and pages of 1 << shift tokens, all numbers of tokens in 31 bits.
static int check_table(const char* what, int streams, int columns, int pages, int shift) {
  if (streams < 1 || columns < 1 || pages < 1) return fail(DTB_ERR_ARG, "%s: a table of %d x %d and %d pages", what, streams, columns, pages);
  if (shift < 0) return fail(DTB_ERR_ARG, "%s: a page size is a power of two from 16 to 2^20", what);
  if ((static_cast<int64_t>(columns) << shift) >= (1ll << 30) || (static_cast<int64_t>(pages) << shift) >= (1ll << 31))
    return fail(DTB_ERR_ARG, "%s: too many tokens in a row of the table or in the pool", what);
  return DTB_OK;
}

DTB_API int dtb_extend_pages(int32_t* table, const int32_t* seqlens, const int32_t* new_lens, const int32_t* free_pages, const int32_t* free_count,
                             int streams, int columns, int pages, int page_size, int32_t* slots, int64_t tokens, int32_t* cu_seqlens,
                             int32_t* seqlens_out, int32_t* free_count_out, int32_t* missing, void* stream) {
  const int shift = page_shift_of(page_size);
  int rc = check_table("dtb_extend_pages", streams, columns, pages, shift);
  if (rc != DTB_OK) return rc;
  if (streams > dtb::kMostStreams) return fail(DTB_ERR_ARG, "dtb_extend_pages: more than %d streams", dtb::kMostStreams);
  if (!table || !seqlens || !new_lens || !free_pages || !free_count || !cu_seqlens || !seqlens_out || !free_count_out || !missing || (!slots && tokens))
    return fail(DTB_ERR_ARG, "dtb_extend_pages: null pointer");
  if (tokens < 0 || tokens >= (1ll << 31) - 4) return fail(DTB_ERR_ARG, "dtb_extend_pages: %lld tokens", static_cast<long long>(tokens));
  if (!aligned16(slots)) return fail(DTB_ERR_ARG, "dtb_extend_pages: slots must be 16-byte aligned");
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  const dtb::ExtendParams p = {table, seqlens, new_lens, free_pages, free_count, slots, cu_seqlens, seqlens_out, free_count_out, missing,
                               streams, columns, pages, shift, static_cast<int>(tokens)};
  const cudaError_t e = dtb::launch_extend_pages(p, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_extend_pages launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_release_pages(const int32_t* table, int32_t* table_out, const int32_t* seqlens, const int32_t* begin, const int32_t* end,
                              int32_t* free_pages, const int32_t* free_count, int streams, int columns, int pages, int page_size,
                              int32_t* seqlens_out, int32_t* free_count_out, void* stream) {
  const int shift = page_shift_of(page_size);
  int rc = check_table("dtb_release_pages", streams, columns, pages, shift);
  if (rc != DTB_OK) return rc;
  if (!table || !table_out || !seqlens || !begin || !end || !free_pages || !free_count || !seqlens_out || !free_count_out)
    return fail(DTB_ERR_ARG, "dtb_release_pages: null pointer");
  const int64_t items = static_cast<int64_t>(streams) * ((columns + dtb::kReleaseColumns - 1) / dtb::kReleaseColumns);
  if (items > static_cast<int64_t>(dtb::kReleaseItems) * dtb::kReleaseCtas)
    return fail(DTB_ERR_ARG, "dtb_release_pages: a table of %d x %d is too large", streams, columns);
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  const dtb::ReleaseParams p = {table, table_out, seqlens, begin, end, free_pages, free_count, seqlens_out, free_count_out, streams, columns, pages, shift};
  const cudaError_t e = dtb::launch_release_pages(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_release_pages launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

// Strides of a pool [pages, P, heads, head_dim]: multiples of 16 bytes, and none below what lies inside.
static int check_pool(const char* what, const char* name, const void* base, int pages, int page_size, int heads, int head_dim, int64_t page_stride,
                      int64_t tok_stride, int64_t head_stride) {
  if (!base) return fail(DTB_ERR_ARG, "%s: null tensor pointer", what);
  if (!aligned16(base) || ((page_stride | tok_stride | head_stride) & 7)) return fail(DTB_ERR_ARG, "%s: %s must be 16-byte aligned, strides multiples of 8 elements", what, name);
  if (tok_stride < head_dim || head_stride < head_dim || page_stride < head_dim || std::max(page_stride, std::max(tok_stride, head_stride)) >= (1ll << 38))
    return fail(DTB_ERR_ARG, "%s: %s has a stride below a row's %d elements or beyond 2^38", what, name, head_dim);
  // (of each two axes that are stepped along, one lies within a step of the other)
  auto apart = [](int64_t na, int64_t sa, int64_t nb, int64_t sb) { return na == 1 || nb == 1 || sa >= nb * sb || sb >= na * sa; };
  if (!apart(page_size, tok_stride, heads, head_stride) || !apart(pages, page_stride, page_size, tok_stride) || !apart(pages, page_stride, heads, head_stride))
    return fail(DTB_ERR_ARG, "%s: %s has strides by which elements lie over one another", what, name);
  return DTB_OK;
}

DTB_API int dtb_write_pages(const void* k, const void* v, int64_t k_tok_stride, int64_t v_tok_stride, int64_t tokens, const int32_t* slots,
                            void* k_pages, int64_t k_page_stride, int64_t k_page_tok_stride, int64_t k_head_stride,
                            void* v_pages, int64_t v_page_stride, int64_t v_page_tok_stride, int64_t v_head_stride,
                            int pages, int page_size, int num_kv_heads, int head_dim, void* stream) {
  const int shift = page_shift_of(page_size);
  int rc = check_table("dtb_write_pages", 1, 1, pages, shift);
  if (rc != DTB_OK) return rc;
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "dtb_write_pages: head_dim %d not in {64, 128}", head_dim);
  if (num_kv_heads < 1 || num_kv_heads > 65535) return fail(DTB_ERR_ARG, "dtb_write_pages: %d key heads", num_kv_heads);
  if (tokens < 0 || tokens >= (1ll << 31)) return fail(DTB_ERR_ARG, "dtb_write_pages: %lld tokens", static_cast<long long>(tokens));
  if (!k || !v || !slots) return fail(DTB_ERR_ARG, "dtb_write_pages: null tensor pointer");
  const int64_t width = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (k_tok_stride < width || v_tok_stride < width || ((k_tok_stride | v_tok_stride) & 7) || !aligned16(k) || !aligned16(v))
    return fail(DTB_ERR_ARG, "dtb_write_pages: tokens must be 16-byte aligned, their strides multiples of 8 elements and not below the heads");
  if ((rc = check_pool("dtb_write_pages", "k_pages", k_pages, pages, page_size, num_kv_heads, head_dim, k_page_stride, k_page_tok_stride, k_head_stride)) != DTB_OK ||
      (rc = check_pool("dtb_write_pages", "v_pages", v_pages, pages, page_size, num_kv_heads, head_dim, v_page_stride, v_page_tok_stride, v_head_stride)) != DTB_OK)
    return rc;
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  if (tokens == 0) return DTB_OK;
  dtb::WriteParams p = {};
  p.src[0] = static_cast<const uint16_t*>(k);
  p.src[1] = static_cast<const uint16_t*>(v);
  p.src_tok[0] = k_tok_stride;
  p.src_tok[1] = v_tok_stride;
  p.dst[0] = static_cast<uint16_t*>(k_pages);
  p.dst[1] = static_cast<uint16_t*>(v_pages);
  p.dst_page[0] = k_page_stride;
  p.dst_page[1] = v_page_stride;
  p.dst_tok[0] = k_page_tok_stride;
  p.dst_tok[1] = v_page_tok_stride;
  p.dst_head[0] = k_head_stride;
  p.dst_head[1] = v_head_stride;
  p.slots = slots;
  p.tokens = static_cast<int>(tokens);
  p.heads = num_kv_heads;
  p.head_shift = head_dim == 64 ? 6 : 7;
  p.page_shift = shift;
  p.capacity = static_cast<int64_t>(pages) << shift;
  const cudaError_t e = dtb::launch_write_pages(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_write_pages launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

// Which kernels a launch over pages takes.
struct PagedPlan {
  int few_rows;                  // sequences with at most this many queries go to the kernel of few rows
  bool tiles;                    // there may be others
  int pack_shift;                // that many heads of a key head (their logarithm) share the tiles of 128 rows
  dtb::PagedRowsPlan rows;
  int states;                    // of parts, at most; 0: the kernel of tiles splits no keys
  int64_t tile_bytes;            // of scratch, in front of that of the kernel of few rows
  int64_t scratch_bytes;
};
static PagedPlan plan_paged(int64_t nseg, int64_t seqlen_q, int64_t seqlen_k, int64_t total_q, int64_t num_heads, int64_t kv_heads, int head_dim, int sm_count) {
  PagedPlan plan = {};
  const int64_t group = num_heads / kv_heads;
  // Up to 64 rows of a key head are a block of the kernel of few rows, which reads keys at the rate of HBM; for more, tiles of 256 rows take as long for a key
  // as one of its blocks.  Batches some of whose sequences have up to twice that stay in one launch.  (us: 10 queries of 16 heads each against 4236 keys of
  // three sequences 69 in that kernel, 29 in tiles; 15 queries and 1 of two sequences, 8 heads, 11396 keys of 128 43, and 57 in both kernels.)
  const bool few = seqlen_q * group <= 128 && total_q != nseg * seqlen_q;
  plan.few_rows = static_cast<int>(std::max<int64_t>((few ? 128 : 64) / group, 1));
  while (plan.pack_shift < 7 && group % (2ll << plan.pack_shift) == 0) ++plan.pack_shift;
  plan.tiles = seqlen_q > plan.few_rows;
  plan.rows = dtb::plan_paged_rows(std::min<int64_t>(seqlen_q, plan.few_rows) * group, seqlen_k, kv_heads, nseg, head_dim, sm_count);
  if (plan.tiles) {
    // Of sequences of one number of queries the blocks are known: with a round of them for each sequence the one that walks furthest has no more
    // than its share, and with a last round that is nearly full nothing is split.  (The launch that joins takes 5 us.)
    const int64_t blocks = ((seqlen_q << plan.pack_shift) + 255) / 256 * (num_heads >> plan.pack_shift) * nseg, rounds = (blocks + sm_count - 1) / sm_count;
    const bool may = total_q != nseg * seqlen_q || blocks <= sm_count * nseg || static_cast<double>(rounds * sm_count) > 1.15 * static_cast<double>(blocks);
    plan.states = may && seqlen_k > 256 ? 2 * sm_count : 0;
    plan.tile_bytes = plan.states * (256ll * (head_dim + 1) * 4) + plan.states / 2 * static_cast<int64_t>(sizeof(dtb::TileJoin));
  }
  plan.scratch_bytes = plan.tile_bytes + plan.rows.scratch_bytes;
  return plan;
}

static int check_paged_shape(const char* what, int nseg, int seqlen_q, int seqlen_k, int num_heads, int num_kv_heads, int head_dim) {
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "%s: head_dim %d not in {64, 128}", what, head_dim);
  if (num_heads < 1 || num_heads > 65535 || num_kv_heads < 1 || num_heads % num_kv_heads) return fail(DTB_ERR_ARG, "%s: %d query heads over %d key heads", what, num_heads, num_kv_heads);
  if (nseg < 1 || nseg > 65535) return fail(DTB_ERR_ARG, "%s: nseg %d out of range", what, nseg);
  if (seqlen_q < 0 || seqlen_k < 0 || seqlen_q >= (1 << 30) || seqlen_k >= (1 << 30)) return fail(DTB_ERR_ARG, "%s: length out of range", what);
  if (static_cast<int64_t>(seqlen_q) * num_heads >= (1ll << 31)) return fail(DTB_ERR_ARG, "%s: too many rows in a sequence", what);
  return DTB_OK;
}

DTB_API int64_t dtb_flash_paged_scratch_bytes(int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int num_heads, int num_kv_heads, int head_dim) {
  int rc = check_paged_shape("dtb_flash_paged_scratch_bytes", nseg, seqlen_q, seqlen_k, num_heads, num_kv_heads, head_dim);
  if (rc != DTB_OK) return rc;
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  return plan_paged(nseg, seqlen_q, seqlen_k, total_q, num_heads, num_kv_heads, head_dim, d->sm_count).scratch_bytes;
}

// Sequences of few and of many queries in one batch take a launch each.  (With rows for more than that, none of them has few, unless there are
// rows behind the last one; the kernel of many then takes it.)
static bool paged_mixed(const PagedPlan& plan, bool packed, int64_t nseg, int64_t seqlen_q, int64_t total_q) {
  return plan.tiles && packed && total_q <= (nseg - 1) * seqlen_q + plan.few_rows;
}
// Blocks of 256 rows, as many as fit the rows that there are.
static int64_t paged_blocks(const PagedPlan& plan, int64_t nseg, int64_t total_q, int64_t num_heads) {
  return ((total_q << plan.pack_shift) / 256 + nseg) * (num_heads >> plan.pack_shift);
}
static bool paged_planned(const PagedPlan& plan, int64_t nseg, int64_t total_q, int64_t num_heads) {
  return nseg <= dtb::kPlanSeqs && paged_blocks(plan, nseg, total_q, num_heads) < dtb::kPlanBlocks;
}

DTB_API int dtb_flash_paged_launches(int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int packed, int num_heads, int num_kv_heads, int head_dim) {
  int rc = check_paged_shape("dtb_flash_paged_launches", nseg, seqlen_q, seqlen_k, num_heads, num_kv_heads, head_dim);
  if (rc != DTB_OK) return rc;
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  if (seqlen_q == 0 || total_q == 0) return 0;
  const PagedPlan plan = plan_paged(nseg, seqlen_q, seqlen_k, total_q, num_heads, num_kv_heads, head_dim, d->sm_count);
  int n = 0;
  if (plan.tiles) n += plan.states > 0 && paged_planned(plan, nseg, total_q, num_heads) ? 2 : 1;
  if (!plan.tiles || paged_mixed(plan, packed != 0, nseg, seqlen_q, total_q)) n += plan.rows.cluster > 0 ? 1 : 2;
  return n;
}

DTB_API int dtb_flash_paged(const void* q, int64_t q_tok_stride, int64_t q_batch_stride,
                            const void* k_pages, int64_t k_page_stride, int64_t k_tok_stride, int64_t k_head_stride,
                            const void* v_pages, int64_t v_page_stride, int64_t v_tok_stride, int64_t v_head_stride,
                            int pages, int page_size, const int32_t* table, int columns, const int32_t* seqlens_k, const int32_t* cu_seqlens_q,
                            void* out, int out_dtype, float* lse, int lse_layout, int accumulate,
                            int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int num_heads, int num_kv_heads, int head_dim, float softmax_scale,
                            int left, int right, int sinks, void* scratch, int64_t scratch_bytes, void* stream) {
  constexpr const char* kWhat = "dtb_flash_paged";
  int rc = check_paged_shape(kWhat, nseg, seqlen_q, seqlen_k, num_heads, num_kv_heads, head_dim);
  if (rc != DTB_OK) return rc;
  const int shift = page_shift_of(page_size);
  if ((rc = check_table(kWhat, nseg, columns, pages, shift)) != DTB_OK) return rc;
  if ((static_cast<int64_t>(nseg) * columns << shift) >= (1ll << 31)) return fail(DTB_ERR_ARG, "%s: the table's %d rows have room for 2^31 tokens or more", kWhat, nseg);
  if (!q || !out || !lse || !table || !seqlens_k) return fail(DTB_ERR_ARG, "%s: null tensor pointer", kWhat);
  if (total_q < 0 || total_q >= (1ll << 31) || total_q * num_heads >= (1ll << 31)) return fail(DTB_ERR_ARG, "%s: too many tokens", kWhat);
  if (cu_seqlens_q == nullptr && static_cast<int64_t>(nseg) * seqlen_q != total_q) return fail(DTB_ERR_ARG, "%s: total tokens are not nseg*seqlen", kWhat);
  constexpr int kFar = 1 << 30;
  if (left < -1 || right < -1 || sinks < 0 || left > kFar || right > kFar || sinks > kFar) return fail(DTB_ERR_ARG, "%s: window (%d, %d) or sinks %d out of range", kWhat, left, right, sinks);
  const int64_t q_width = static_cast<int64_t>(num_heads) * head_dim;
  if (q_tok_stride < q_width || (cu_seqlens_q == nullptr && nseg > 1 && q_batch_stride < q_width)) return fail(DTB_ERR_ARG, "%s: q's stride smaller than the heads", kWhat);
  if ((q_tok_stride | q_batch_stride) & 7) return fail(DTB_ERR_ARG, "%s: strides must be multiples of 8 elements", kWhat);
  if (!aligned16(q) || !aligned16(out)) return fail(DTB_ERR_ARG, "%s: tensor pointers must be 16-byte aligned", kWhat);
  if ((rc = check_pool(kWhat, "k_pages", k_pages, pages, page_size, num_kv_heads, head_dim, k_page_stride, k_tok_stride, k_head_stride)) != DTB_OK ||
      (rc = check_pool(kWhat, "v_pages", v_pages, pages, page_size, num_kv_heads, head_dim, v_page_stride, v_tok_stride, v_head_stride)) != DTB_OK)
    return rc;
  if (out_dtype != DTB_F32 && out_dtype != DTB_BF16) return fail(DTB_ERR_ARG, "%s: bad out_dtype %d", kWhat, out_dtype);
  if (lse_layout != DTB_LSE_BHS && lse_layout != DTB_LSE_BSH) return fail(DTB_ERR_ARG, "%s: bad lse_layout %d", kWhat, lse_layout);
  if (accumulate && out_dtype != DTB_F32) return fail(DTB_ERR_ARG, "%s: accumulate needs an fp32 state", kWhat);
  if (!(softmax_scale > 0.f)) return fail(DTB_ERR_ARG, "%s: softmax_scale must be positive", kWhat);
  if (!aligned16(scratch)) return fail(DTB_ERR_ARG, "%s: scratch must be 16-byte aligned", kWhat);
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  if (seqlen_q == 0 || total_q == 0) return DTB_OK;
  const PagedPlan plan = plan_paged(nseg, seqlen_q, seqlen_k, total_q, num_heads, num_kv_heads, head_dim, d->sm_count);
  if (scratch_bytes < plan.scratch_bytes || (!scratch && plan.scratch_bytes))
    return fail(DTB_ERR_ARG, "%s: scratch of %lld bytes is smaller than the %lld needed", kWhat, static_cast<long long>(scratch_bytes),
                static_cast<long long>(plan.scratch_bytes));

  dtb::PagedParams p;
  memset(&p, 0, sizeof(p));
  p.f.out = out;
  p.f.lse = lse;
  p.f.cu_q = cu_seqlens_q;
  p.f.status = d->status_ptr;
  p.f.out_tok_stride = q_width;
  p.f.total_q = total_q;
  p.f.nseg = nseg;
  p.f.seqlen_q = seqlen_q;
  p.f.seqlen_k = seqlen_k;
  p.f.num_heads = num_heads;
  p.f.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.f.out_dtype = out_dtype;
  p.f.lse_layout = lse_layout;
  p.f.accumulate = accumulate ? 1 : 0;
  p.q = static_cast<const uint16_t*>(q);
  p.q_tok = q_tok_stride;
  p.q_batch = q_batch_stride;
  p.seqlens_k = seqlens_k;
  p.kv_heads = num_kv_heads;
  p.left = left;
  p.right = right;
  p.sinks = left < 0 ? 0 : sinks;             // (all are seen as it is)
  p.q_start = DTB_QUERIES_LAST;
  p.splits = 1;
  p.table = table;
  p.columns = columns;
  p.pages = pages;
  p.page_shift = shift;
  const bool mixed = paged_mixed(plan, cu_seqlens_q != nullptr, nseg, seqlen_q, total_q);
  p.few_rows = plan.tiles && !mixed ? -1 : plan.few_rows;
  p.real = p.f;
  if ((rc = load_encoder()) != DTB_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  dtb::PagedMap mk, mv;
  auto make_maps = [&](int box_rows) {
    mk.dim_shift = mv.dim_shift = head_dim == 64 ? 6 : 7;
    p.box_rows = p.key_align = box_rows;
    const int r = make_page_map(&mk.map, k_pages, head_dim, page_size, k_tok_stride, num_kv_heads, k_head_stride, pages, k_page_stride, box_rows, &p.k_batch_first, "k_pages");
    return r != DTB_OK ? r : make_page_map(&mv.map, v_pages, head_dim, page_size, v_tok_stride, num_kv_heads, v_head_stride, pages, v_page_stride, box_rows, &p.v_batch_first, "v_pages");
  };
  cudaError_t e = cudaSuccess;
  if (plan.tiles) {
    // (with a limit to the left runs begin anywhere, and fewer than 16 keys in front of them are cleared)
    if ((rc = make_maps(left < 0 ? std::min(page_size, 128) : 16)) != DTB_OK) return rc;
    const bool packed = cu_seqlens_q != nullptr;
    dtb::PagedParams t = p;
    dtb::QueryMap tq;
    tq.dim_shift = mk.dim_shift;
    tq.pack_shift = t.pack_shift = plan.pack_shift;
    if ((rc = make_query_map(&tq.map, q, head_dim, num_heads, packed ? total_q : seqlen_q, q_tok_stride, packed ? 1 : nseg, q_batch_stride, 1 << plan.pack_shift,
                             &t.q_batch_first)) != DTB_OK) return rc;
    t.f.num_heads = num_heads >> plan.pack_shift;
    t.f.seqlen_q = seqlen_q << plan.pack_shift;
    t.f.total_q = total_q << plan.pack_shift;
    // the grid: places for the blocks and for the parts, or CTAs that share the blocks out
    t.planned = paged_planned(plan, nseg, total_q, num_heads);
    const int64_t per_seq = (static_cast<int64_t>(t.f.seqlen_q) + 255) / 256 * nseg * t.f.num_heads;
    const int64_t blocks = std::min(per_seq, paged_blocks(plan, nseg, total_q, num_heads));
    t.blocks = static_cast<int>(t.planned ? blocks + plan.states : std::min<int64_t>(blocks, d->sm_count));
    t.ctas = d->sm_count;
    t.most_states = t.planned ? plan.states : 0;
    t.parts.out = scratch;
    t.parts.lse = static_cast<float*>(scratch) + plan.states * 256ll * head_dim;
    t.joins = reinterpret_cast<dtb::TileJoin*>(t.parts.lse + plan.states * 256ll);
    e = head_dim == 64 ? dtb::launch_paged_tiles<64>(tq, mk, mv, t, s) : dtb::launch_paged_tiles<128>(tq, mk, mv, t, s);
    if (e == cudaSuccess && t.most_states > 0) {
      t.f = t.real;
      e = head_dim == 64 ? dtb::launch_tile_join<64>(t, s) : dtb::launch_tile_join<128>(t, s);
    }
  }
  if (e == cudaSuccess && (!plan.tiles || mixed)) {
    if ((rc = make_maps(std::min(page_size, 64))) != DTB_OK) return rc;
    void* rows_scratch = static_cast<uint8_t*>(scratch) + plan.tile_bytes;
    e = head_dim == 64 ? dtb::launch_paged_rows<64>(mk, mv, p, plan.rows, rows_scratch, s) : dtb::launch_paged_rows<128>(mk, mv, p, plan.rows, rows_scratch, s);
  }
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "%s launch failed: %s", kWhat, cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_merge_states(int nstates, const void* const* outs, const int* out_dtypes,
                     const float* const* lses, const int* lse_layouts,
                     float* out, float* lse_out, int lse_out_layout, void* out_bf16,
                     int batch, int seq, int num_heads, int head_dim, void* stream) {
  if (nstates < 1 || nstates > DTB_MERGE_MAX_STATES) return fail(DTB_ERR_ARG, "dtb_merge_states: nstates %d not in [1, %d]", nstates, DTB_MERGE_MAX_STATES);
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "dtb_merge_states: head_dim %d not in {64, 128}", head_dim);
  if (!outs || !out_dtypes || !lses || !lse_layouts) return fail(DTB_ERR_ARG, "dtb_merge_states: null argument");
  if (!out && !out_bf16) return fail(DTB_ERR_ARG, "dtb_merge_states: neither an fp32 nor a bf16 result buffer was given");
  if (batch < 0 || seq < 0 || num_heads < 1) return fail(DTB_ERR_ARG, "dtb_merge_states: bad shape");
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  dtb::MergeParams p;
  memset(&p, 0, sizeof(p));
  for (int i = 0; i < nstates; ++i) {
    if (!outs[i] || !lses[i]) return fail(DTB_ERR_ARG, "dtb_merge_states: state %d has a null pointer", i);
    if (!aligned16(outs[i])) return fail(DTB_ERR_ARG, "dtb_merge_states: state %d is not 16-byte aligned", i);
    if (out_dtypes[i] != DTB_F32 && out_dtypes[i] != DTB_BF16) return fail(DTB_ERR_ARG, "dtb_merge_states: bad dtype for state %d", i);
    if (lse_layouts[i] != DTB_LSE_BHS && lse_layouts[i] != DTB_LSE_BSH) return fail(DTB_ERR_ARG, "dtb_merge_states: bad lse layout for state %d", i);
    if (i > 0 && ((out && outs[i] == out) || (lse_out && lses[i] == lse_out))) return fail(DTB_ERR_ARG, "dtb_merge_states: the result may alias state 0 only");
    p.outs[i] = outs[i];
    p.lse[i] = lses[i];
    p.out_dtype[i] = out_dtypes[i];
    p.lse_layout[i] = lse_layouts[i];
  }
  if (out && outs[0] == out && out_dtypes[0] != DTB_F32) return fail(DTB_ERR_ARG, "dtb_merge_states: in-place merge needs an fp32 state 0");
  if (lse_out && lses[0] == lse_out && lse_layouts[0] != lse_out_layout) return fail(DTB_ERR_ARG, "dtb_merge_states: in-place lse needs matching layouts");
  if ((out && !aligned16(out)) || (out_bf16 && !aligned16(out_bf16))) return fail(DTB_ERR_ARG, "dtb_merge_states: result not 16-byte aligned");
  p.out = out;
  p.lse_out = lse_out;
  p.out_bf16 = static_cast<uint16_t*>(out_bf16);
  p.rows = static_cast<int64_t>(batch) * seq * num_heads;
  p.lse_out_layout = lse_out_layout;
  p.nstates = nstates;
  p.H = num_heads;
  p.S = seq;
  if (p.rows == 0) return DTB_OK;
  cudaError_t e = dtb::launch_merge(p, head_dim, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_merge_states launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_merge_rows(int nstates, const void* const* outs, const int* out_dtypes, const uint8_t* const* exponents,
                     const float* const* lses, const int* lse_layouts,
                     float* out, float* lse_out, int lse_out_layout, void* out_bf16,
                     void* out_codes, int out_codes_dtype, uint8_t* out_exponents,
                     int batch, int seq, int num_heads, int head_dim, void* stream) {
  static_assert(DTB_F32 == dtb::kRowsF32 && DTB_BF16 == dtb::kRowsBf16 && DTB_I8 == dtb::kRowsI8 && DTB_E4M3 == dtb::kRowsE4m3, "types");
  static_assert(DTB_MERGE_MAX_STATES == dtb::kMergeRowsMaxStates, "states");
  if (nstates < 1 || nstates > DTB_MERGE_MAX_STATES) return fail(DTB_ERR_ARG, "dtb_merge_rows: nstates %d not in [1, %d]", nstates, DTB_MERGE_MAX_STATES);
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "dtb_merge_rows: head_dim %d not in {64, 128}", head_dim);
  if (!outs || !out_dtypes || !exponents || !lses || !lse_layouts) return fail(DTB_ERR_ARG, "dtb_merge_rows: null argument");
  if (!out && !out_bf16 && !out_codes) return fail(DTB_ERR_ARG, "dtb_merge_rows: no result buffer was given");
  if (out_codes && out_codes_dtype != DTB_I8 && out_codes_dtype != DTB_E4M3) return fail(DTB_ERR_ARG, "dtb_merge_rows: bad type %d of the 8-bit result", out_codes_dtype);
  if (out_codes && !out_exponents) return fail(DTB_ERR_ARG, "dtb_merge_rows: an 8-bit result needs a buffer of exponents");
  if (lse_out && lse_out_layout != DTB_LSE_BHS && lse_out_layout != DTB_LSE_BSH) return fail(DTB_ERR_ARG, "dtb_merge_rows: bad lse_out_layout %d", lse_out_layout);
  if (batch < 0 || seq < 0 || num_heads < 1) return fail(DTB_ERR_ARG, "dtb_merge_rows: bad shape");
  const int64_t rows = static_cast<int64_t>(batch) * seq;
  if (rows >= (1ll << 31) || rows * num_heads >= (1ll << 31)) return fail(DTB_ERR_ARG, "dtb_merge_rows: more than 2^31 rows");
  if (!aligned16(out) || !aligned16(out_bf16) || !aligned16(out_codes)) return fail(DTB_ERR_ARG, "dtb_merge_rows: result not 16-byte aligned");
  dtb::MergeRowsParams p;
  memset(&p, 0, sizeof(p));
  int at = 0;
  for (int pass = 0; pass < 2; ++pass) {           // the states in 8 bits, then the others
    for (int i = 0; i < nstates; ++i) {
      const int t = out_dtypes[i];
      if (t != DTB_F32 && t != DTB_BF16 && t != DTB_I8 && t != DTB_E4M3) return fail(DTB_ERR_ARG, "dtb_merge_rows: bad dtype for state %d", i);
      const bool narrow = t == DTB_I8 || t == DTB_E4M3;
      if (narrow != (pass == 0)) continue;
      if (!outs[i] || (narrow && !exponents[i])) return fail(DTB_ERR_ARG, "dtb_merge_rows: state %d has a null pointer", i);
      if (!lses[i]) return fail(DTB_ERR_ARG, "dtb_merge_rows: state %d has no lse", i);
      if (!aligned16(outs[i])) return fail(DTB_ERR_ARG, "dtb_merge_rows: state %d is not 16-byte aligned", i);
      if (lse_layouts[i] != DTB_LSE_BHS && lse_layouts[i] != DTB_LSE_BSH) return fail(DTB_ERR_ARG, "dtb_merge_rows: bad lse layout for state %d", i);
      if ((outs[i] == out_bf16 && t != DTB_BF16) || (outs[i] == out_codes) || (outs[i] == out && t != DTB_F32))
        return fail(DTB_ERR_ARG, "dtb_merge_rows: a result may take the place of a state of its own type only, an 8-bit one of none");
      if (out_codes && narrow && exponents[i] == out_exponents) return fail(DTB_ERR_ARG, "dtb_merge_rows: the exponents of an 8-bit result are those of state %d", i);
      if (lse_out && lses[i] == lse_out && lse_layouts[i] != lse_out_layout) return fail(DTB_ERR_ARG, "dtb_merge_rows: in-place lse needs matching layouts");
      p.values[at] = outs[i];
      p.exponents[at] = exponents[i];
      p.lse[at] = lses[i];
      p.dtype[at] = t;
      p.lse_layout[at] = lse_layouts[i];
      ++at;
    }
    if (pass == 0) p.narrow = at;
  }
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  p.nstates = nstates;
  p.out = out;
  p.out_bf16 = static_cast<uint16_t*>(out_bf16);
  p.out_codes = static_cast<uint8_t*>(out_codes);
  p.out_exponents = out_exponents;
  p.out_codes_dtype = out_codes_dtype;
  p.lse_out = lse_out;
  p.lse_out_layout = lse_out_layout;
  p.rows = rows * num_heads;
  p.H = num_heads;
  p.S = seq;
  if (p.rows == 0) return DTB_OK;
  cudaError_t e = dtb::launch_merge_rows(p, head_dim, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_merge_rows launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

// `wide` values (fp32 or bf16) and their rows in 8 bits
static int check_rows(const char* what, const void* wide, int dtype, const void* codes, int codes_dtype, const uint8_t* exponents, int64_t rows, int head_dim) {
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "%s: head_dim %d not in {64, 128}", what, head_dim);
  if (dtype != DTB_F32 && dtype != DTB_BF16) return fail(DTB_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (codes_dtype != DTB_I8 && codes_dtype != DTB_E4M3) return fail(DTB_ERR_ARG, "%s: bad type %d of the codes", what, codes_dtype);
  if (rows < 0 || rows >= (1ll << 31)) return fail(DTB_ERR_ARG, "%s: %lld rows", what, static_cast<long long>(rows));
  if (!wide || !codes || !exponents) return fail(DTB_ERR_ARG, "%s: null tensor pointer", what);
  if (!aligned16(wide) || !aligned16(codes)) return fail(DTB_ERR_ARG, "%s: pointers must be 16-byte aligned", what);
  return DTB_OK;
}

DTB_API int dtb_quantize_rows(const void* values, int dtype, void* codes, int codes_dtype, uint8_t* exponents, int64_t rows, int head_dim, void* stream) {
  int rc = check_rows("dtb_quantize_rows", values, dtype, codes, codes_dtype, exponents, rows, head_dim);
  DeviceInfo* d = nullptr;
  if (rc != DTB_OK || (rc = device_info(&d)) != DTB_OK || rows == 0) return rc;
  cudaError_t e = dtb::launch_quantize_rows(values, dtype == DTB_BF16, static_cast<uint8_t*>(codes), exponents, codes_dtype, rows, head_dim, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_quantize_rows launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_dequantize_rows(const void* codes, int codes_dtype, const uint8_t* exponents, void* out, int out_dtype, int64_t rows, int head_dim, void* stream) {
  int rc = check_rows("dtb_dequantize_rows", out, out_dtype, codes, codes_dtype, exponents, rows, head_dim);
  DeviceInfo* d = nullptr;
  if (rc != DTB_OK || (rc = device_info(&d)) != DTB_OK || rows == 0) return rc;
  cudaError_t e = dtb::launch_dequantize_rows(static_cast<const uint8_t*>(codes), exponents, codes_dtype, out, out_dtype == DTB_BF16, rows, head_dim, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_dequantize_rows launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_copy_chunks(int npairs, const void* const* srcs, void* const* dsts, int64_t chunk_bytes,
                    int64_t n0, int64_t n1, int64_t n2,
                    int64_t ss0, int64_t ss1, int64_t ss2,
                    int64_t ds0, int64_t ds1, int64_t ds2, void* stream) {
  if (npairs < 1 || npairs > 4) return fail(DTB_ERR_ARG, "dtb_copy_chunks: npairs %d not in [1, 4]", npairs);
  if (!srcs || !dsts) return fail(DTB_ERR_ARG, "dtb_copy_chunks: null argument");
  if (chunk_bytes <= 0 || (chunk_bytes & 15)) return fail(DTB_ERR_ARG, "dtb_copy_chunks: chunk_bytes must be a positive multiple of 16");
  if ((ss0 | ss1 | ss2 | ds0 | ds1 | ds2) & 15) return fail(DTB_ERR_ARG, "dtb_copy_chunks: strides must be multiples of 16 bytes");
  if (n0 < 0 || n1 < 0 || n2 < 0) return fail(DTB_ERR_ARG, "dtb_copy_chunks: negative extent");
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  dtb::CopyParams p;
  memset(&p, 0, sizeof(p));
  for (int i = 0; i < npairs; ++i) {
    if (!srcs[i] || !dsts[i] || !aligned16(srcs[i]) || !aligned16(dsts[i])) return fail(DTB_ERR_ARG, "dtb_copy_chunks: pair %d null or misaligned", i);
    p.src[i] = srcs[i];
    p.dst[i] = dsts[i];
  }
  p.chunk_bytes = chunk_bytes;
  p.n0 = n0; p.n1 = n1; p.n2 = n2;
  p.ss0 = ss0; p.ss1 = ss1; p.ss2 = ss2;
  p.ds0 = ds0; p.ds1 = ds1; p.ds2 = ds2;
  if (n0 * n1 * n2 == 0) return DTB_OK;
  cudaError_t e = dtb::launch_copy_chunks(p, npairs, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_copy_chunks launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_norm_rope(const void* q, void* q_out, const void* q_weight, const void* q_bias, float q_eps,
                          const void* k, void* k_out, const void* k_weight, const void* k_bias, float k_eps,
                          const float* cos, const float* sin,
                          int batch, int seq, int text_len, int num_heads, int head_dim, void* stream) {
  if (!q || !q_out || !q_weight || !q_bias || !k || !k_out || !k_weight || !k_bias) return fail(DTB_ERR_ARG, "dtb_norm_rope: null tensor pointer");
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "dtb_norm_rope: head_dim %d not in {64, 128}", head_dim);
  if (batch < 0 || seq < 0 || num_heads < 1 || text_len < 0 || text_len > seq) return fail(DTB_ERR_ARG, "dtb_norm_rope: bad shape");
  if (text_len < seq && (!cos || !sin)) return fail(DTB_ERR_ARG, "dtb_norm_rope: null rotary table");
  const void* all[10] = {q, q_out, q_weight, q_bias, k, k_out, k_weight, k_bias, cos, sin};
  for (const void* x : all)
    if (!aligned16(x)) return fail(DTB_ERR_ARG, "dtb_norm_rope: pointers must be 16-byte aligned");
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  dtb::NormRopeParams p;
  p.src[0] = static_cast<const uint16_t*>(q);
  p.src[1] = static_cast<const uint16_t*>(k);
  p.dst[0] = static_cast<uint16_t*>(q_out);
  p.dst[1] = static_cast<uint16_t*>(k_out);
  p.weight[0] = static_cast<const uint16_t*>(q_weight);
  p.weight[1] = static_cast<const uint16_t*>(k_weight);
  p.bias[0] = static_cast<const uint16_t*>(q_bias);
  p.bias[1] = static_cast<const uint16_t*>(k_bias);
  p.cos = cos;
  p.sin = sin;
  p.eps[0] = q_eps;
  p.eps[1] = k_eps;
  p.tokens = static_cast<int64_t>(batch) * seq;
  p.seq = seq;
  p.text_len = text_len;
  p.num_heads = num_heads;
  if (p.tokens == 0) return DTB_OK;
  cudaError_t e = dtb::launch_norm_rope(p, head_dim, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_norm_rope launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

// What the forward and the backward pass are given alike.
static int grid_rope_params(const char* what, dtb::NormRopeGridParams* p, const void* const x[2], const int64_t strides[4], void* const dst[2],
                            const void* const weight[2], const void* const bias[2], const float eps[2], int dtype,
                            const int* grid, const int* axes, const double* place, int64_t first, int shards,
                            int batch, int seq, int text_len, int video_len, int q_heads, int k_heads, int head_dim) {
  if (!grid || !axes || !place) return fail(DTB_ERR_ARG, "%s: null argument", what);
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "%s: head_dim %d not in {64, 128}", what, head_dim);
  if (dtype != DTB_F32 && dtype != DTB_BF16) return fail(DTB_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || seq < 0 || q_heads < 1 || k_heads < 1) return fail(DTB_ERR_ARG, "%s: bad shape", what);
  if (text_len < 0 || video_len < 0 || video_len > seq || text_len > seq - video_len) return fail(DTB_ERR_ARG, "%s: %d text and %d video tokens of %d", what, text_len, video_len, seq);
  int64_t places = 1;
  for (int i = 0; i < 3; ++i) {
    if (grid[i] < 0) return fail(DTB_ERR_ARG, "%s: negative grid", what);
    places *= grid[i];
    if (places >= (1ll << 31)) return fail(DTB_ERR_ARG, "%s: grid of 2^31 places or more", what);
  }
  int channels = 0;
  for (int i = 0; i < 3; ++i) {
    if (axes[i] < 0 || axes[i] > head_dim || axes[i] % 2) return fail(DTB_ERR_ARG, "%s: an axis has %d channels", what, axes[i]);
    channels += axes[i];
  }
  if (channels != head_dim) return fail(DTB_ERR_ARG, "%s: the axes have %d channels, a head %d", what, channels, head_dim);
  if (first < 0 || first > (1ll << 62) || shards < 1) return fail(DTB_ERR_ARG, "%s: first token %lld of %d shards", what, static_cast<long long>(first), shards);
  const int64_t shard_len = places / shards + (places % shards ? 1 : 0);
  if (shard_len * shards >= (1ll << 31)) return fail(DTB_ERR_ARG, "%s: %d shards of %lld tokens", what, shards, static_cast<long long>(shard_len));
  if (!(place[0] > 0.) || !std::isfinite(place[0])) return fail(DTB_ERR_ARG, "%s: base must be positive", what);
  for (int i = 1; i < 7; ++i)
    if (!std::isfinite(place[i])) return fail(DTB_ERR_ARG, "%s: origin and step must be finite", what);
  const int width = dtype == DTB_F32 ? 4 : 8;                     // values in 16 bytes
  const int heads[2] = {q_heads, k_heads};
  for (int i = 0; i < 2; ++i) {
    if (!x[i] || !dst[i] || !weight[i]) return fail(DTB_ERR_ARG, "%s: null tensor pointer", what);
    if (!aligned16(x[i]) || !aligned16(dst[i]) || !aligned16(weight[i]) || !aligned16(bias[i])) return fail(DTB_ERR_ARG, "%s: pointers must be 16-byte aligned", what);
    // (the kernels count smaller numbers as 0, and 0 has no inverse root)
    if (!(eps[i] >= FLT_MIN)) return fail(DTB_ERR_ARG, "%s: eps must be positive, and not below the smallest normal float", what);
    if (strides[2 * i] % width || strides[2 * i + 1] % width) return fail(DTB_ERR_ARG, "%s: strides must be multiples of 16 bytes", what);
    p->src[i] = x[i];
    p->tok_stride[i] = strides[2 * i];
    p->batch_stride[i] = strides[2 * i + 1];
    p->dst[i] = dst[i];
    p->weight[i] = weight[i];
    p->bias[i] = bias[i];
    p->eps[i] = eps[i];
    p->heads[i] = heads[i];
  }
  p->tokens = static_cast<int64_t>(batch) * seq;
  p->seq = seq;
  p->text_len = text_len;
  p->video_len = video_len;
  p->first = first;
  p->shards = shards;
  p->shard_len = static_cast<int>(shard_len);
  p->shard_places = static_cast<int>(places / shards);
  p->shard_rest = static_cast<int>(places % shards);
  p->size_y = grid[1];
  p->size_x = grid[2];
  for (int a = 0; a < 3; ++a) {
    p->origin[a] = place[1 + a];
    p->step[a] = place[4 + a];
    p->ratio[a] = axes[a] > 0 ? std::pow(place[0], -2. / axes[a]) : 1.;
    p->pairs_end[a] = (a == 0 ? 0 : p->pairs_end[a - 1]) + axes[a] / 2;
  }
  return DTB_OK;
}

DTB_API int dtb_norm_rope_grid(const void* q, int64_t q_tok_stride, int64_t q_batch_stride, void* q_out, const void* q_weight, const void* q_bias, float q_eps,
                               const void* k, int64_t k_tok_stride, int64_t k_batch_stride, void* k_out, const void* k_weight, const void* k_bias, float k_eps,
                               int dtype, int rms, const int* grid, const int* axes, const double* place, int64_t first, int shards,
                               int batch, int seq, int text_len, int video_len, int q_heads, int k_heads, int head_dim, void* stream) {
  dtb::NormRopeGridParams p;
  memset(&p, 0, sizeof(p));
  const void* x[2] = {q, k};
  const int64_t strides[4] = {q_tok_stride, q_batch_stride, k_tok_stride, k_batch_stride};
  void* dst[2] = {q_out, k_out};
  const void* w[2] = {q_weight, k_weight};
  const void* b[2] = {q_bias, k_bias};
  const float eps[2] = {q_eps, k_eps};
  int rc = grid_rope_params("dtb_norm_rope_grid", &p, x, strides, dst, w, b, eps, dtype, grid, axes, place, first, shards, batch, seq, text_len,
                            video_len, q_heads, k_heads, head_dim);
  if (rc != DTB_OK) return rc;
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  if (p.tokens == 0) return DTB_OK;
  cudaError_t e = dtb::launch_norm_rope_grid(p, head_dim, dtype == DTB_BF16, rms != 0, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_norm_rope_grid launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int64_t dtb_norm_rope_grid_scratch_bytes(int head_dim) {
  DeviceInfo* d = nullptr;
  if (head_dim != 64 && head_dim != 128) return fail(DTB_ERR_ARG, "dtb_norm_rope_grid_scratch_bytes: head_dim %d not in {64, 128}", head_dim);
  int rc = device_info(&d);
  return rc != DTB_OK ? rc : dtb::norm_rope_grid_scratch_bytes(head_dim, d->sm_count);
}

DTB_API int dtb_norm_rope_grid_backward(const void* dq_out, int64_t dq_tok_stride, int64_t dq_batch_stride,
                                        const void* dk_out, int64_t dk_tok_stride, int64_t dk_batch_stride,
                                        const void* q, int64_t q_tok_stride, int64_t q_batch_stride, const void* q_weight, float q_eps,
                                        const void* k, int64_t k_tok_stride, int64_t k_batch_stride, const void* k_weight, float k_eps,
                                        void* dq, void* dk, void* dq_weight, void* dq_bias, void* dk_weight, void* dk_bias,
                                        int dtype, int rms, const int* grid, const int* axes, const double* place, int64_t first, int shards,
                                        int batch, int seq, int text_len, int video_len, int q_heads, int k_heads, int head_dim,
                                        void* scratch, int64_t scratch_bytes, void* stream) {
  dtb::NormRopeGridParams p;
  memset(&p, 0, sizeof(p));
  const void* x[2] = {q, k};
  const int64_t strides[4] = {q_tok_stride, q_batch_stride, k_tok_stride, k_batch_stride};
  void* dst[2] = {dq, dk};
  const void* w[2] = {q_weight, k_weight};
  const void* b[2] = {nullptr, nullptr};
  const float eps[2] = {q_eps, k_eps};
  const char* what = "dtb_norm_rope_grid_backward";
  int rc = grid_rope_params(what, &p, x, strides, dst, w, b, eps, dtype, grid, axes, place, first, shards, batch, seq, text_len, video_len,
                            q_heads, k_heads, head_dim);
  if (rc != DTB_OK) return rc;
  const int width = dtype == DTB_F32 ? 4 : 8;
  if (!dq_out || !dk_out || !scratch) return fail(DTB_ERR_ARG, "%s: null tensor pointer", what);
  if (!aligned16(dq_out) || !aligned16(dk_out) || !aligned16(scratch)) return fail(DTB_ERR_ARG, "%s: pointers must be 16-byte aligned", what);
  if (dq_tok_stride % width || dq_batch_stride % width || dk_tok_stride % width || dk_batch_stride % width) return fail(DTB_ERR_ARG, "%s: strides must be multiples of 16 bytes", what);
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  const int64_t need = dtb::norm_rope_grid_scratch_bytes(head_dim, d->sm_count);
  if (scratch_bytes < need)
    return fail(DTB_ERR_ARG, "%s: scratch of %lld bytes is smaller than the %lld needed", what, static_cast<long long>(scratch_bytes), static_cast<long long>(need));
  p.grad[0] = dq_out;
  p.grad[1] = dk_out;
  p.grad_tok_stride[0] = dq_tok_stride;
  p.grad_tok_stride[1] = dk_tok_stride;
  p.grad_batch_stride[0] = dq_batch_stride;
  p.grad_batch_stride[1] = dk_batch_stride;
  const dtb::NormRopeGridSums sums = {{dq_weight, dk_weight}, {dq_bias, dk_bias}};
  p.partial = static_cast<float*>(scratch);
  cudaError_t e = dtb::launch_norm_rope_grid_backward(p, sums, head_dim, dtype == DTB_BF16, rms != 0, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
  return DTB_OK;
}

static int check_streams(const char* what, std::initializer_list<const void*> ptrs, int batch, int video_len, int text_len, int dim) {
  for (const void* x : ptrs) {
    if (!x) return fail(DTB_ERR_ARG, "%s: null tensor pointer", what);
    if (!aligned16(x)) return fail(DTB_ERR_ARG, "%s: pointers must be 16-byte aligned", what);
  }
  if (batch < 0 || batch > 65535 || video_len < 0 || text_len < 0) return fail(DTB_ERR_ARG, "%s: bad shape", what);
  if (dim < 256 || dim > dtb::kModMaxDim || dim % 256) return fail(DTB_ERR_ARG, "%s: dim %d is not a multiple of 256 up to %d", what, dim, dtb::kModMaxDim);
  return DTB_OK;
}

DTB_API int dtb_ln_modulate(const void* video, const void* text, const void* weight, const void* bias, float eps,
                            const void* mod, void* out, int batch, int video_len, int text_len, int dim, void* stream) {
  int rc = check_streams("dtb_ln_modulate", {video, text, weight, bias, mod, out}, batch, video_len, text_len, dim);
  if (rc != DTB_OK) return rc;
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  if (batch == 0 || (video_len == 0 && text_len == 0)) return DTB_OK;
  dtb::LnModulateParams p;
  p.video = static_cast<const uint16_t*>(video);
  p.text = static_cast<const uint16_t*>(text);
  p.weight = static_cast<const uint16_t*>(weight);
  p.bias = static_cast<const uint16_t*>(bias);
  p.mod = static_cast<const uint16_t*>(mod);
  p.out = static_cast<uint16_t*>(out);
  p.mod_stride = 6ll * dim;
  p.eps = eps;
  p.video_len = video_len;
  p.text_len = text_len;
  p.dim = dim;
  cudaError_t e = dtb::launch_ln_modulate(p, batch, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_ln_modulate launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int dtb_gate_add(const void* video, const void* text, const void* a, const void* mod, void* video_out, void* text_out,
                         int batch, int video_len, int text_len, int dim, void* stream) {
  int rc = check_streams("dtb_gate_add", {video, text, a, mod, video_out, text_out}, batch, video_len, text_len, dim);
  if (rc != DTB_OK) return rc;
  DeviceInfo* d = nullptr;
  if ((rc = device_info(&d)) != DTB_OK) return rc;
  if (batch == 0 || (video_len == 0 && text_len == 0)) return DTB_OK;
  dtb::GateAddParams p;
  p.video = static_cast<const uint16_t*>(video);
  p.text = static_cast<const uint16_t*>(text);
  p.a = static_cast<const uint16_t*>(a);
  p.mod = static_cast<const uint16_t*>(mod);
  p.video_out = static_cast<uint16_t*>(video_out);
  p.text_out = static_cast<uint16_t*>(text_out);
  p.mod_stride = 6ll * dim;
  p.video_len = video_len;
  p.text_len = text_len;
  p.dim = dim;
  cudaError_t e = dtb::launch_gate_add(p, batch, d->sm_count, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_gate_add launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

DTB_API int64_t dtb_drift_scratch_bytes(int64_t n) { return dtb::drift_scratch_bytes(n < 0 ? 0 : n); }

DTB_API int dtb_drift_accumulate(const float* cur, const float* prev, int64_t n, float* accum,
                                 void* scratch, int64_t scratch_bytes, void* stream) {
  if (n < 0) return fail(DTB_ERR_ARG, "dtb_drift_accumulate: negative length");
  if (!accum || !scratch || (n > 0 && (!cur || !prev))) return fail(DTB_ERR_ARG, "dtb_drift_accumulate: null pointer");
  if (reinterpret_cast<uintptr_t>(scratch) & 255) return fail(DTB_ERR_ARG, "dtb_drift_accumulate: scratch must be 256-byte aligned");
  if (scratch_bytes < dtb::drift_scratch_bytes(n))
    return fail(DTB_ERR_ARG, "dtb_drift_accumulate: scratch of %lld bytes is smaller than the %lld needed for n = %lld",
                static_cast<long long>(scratch_bytes), static_cast<long long>(dtb::drift_scratch_bytes(n)), static_cast<long long>(n));
  if (dtb::drift_blocks(n) >= (1ll << 31)) return fail(DTB_ERR_ARG, "dtb_drift_accumulate: n too large");
  DeviceInfo* d = nullptr;
  int rc = device_info(&d);
  if (rc != DTB_OK) return rc;
  cudaError_t e = dtb::launch_drift_stats(cur, prev, n, accum, static_cast<unsigned char*>(scratch), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(DTB_ERR_CUDA, "dtb_drift_accumulate launch failed: %s", cudaGetErrorString(e));
  return DTB_OK;
}

}  // extern "C"
