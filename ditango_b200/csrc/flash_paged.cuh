// Attention over keys and values that lie in pages: what the kernels are given (flash_paged_rows.cu for few query rows, flash_window_sm100.cu
// for many), and how a sequence's keys are found.
//
// Page n of a pool holds P tokens (a power of two, at least 16); key j of sequence b is token j % P of page table[b][j / P].  A page number
// outside the pool stands for keys and values of 0.
#pragma once
#include "flash_common.cuh"
#include "flash_window.cuh"

namespace dtb {

struct PagedParams : WindowParams {    // (k, v, their strides, cu_k and k_start are not used; seqlens_k is given always)
  const int32_t* table;                // [sequences, columns]
  int columns, pages, page_shift;
  int box_rows;                        // tokens of a tile that one load fetches; divides a page, so that no load crosses one
  int key_align;                       // runs of keys are walked from a multiple of this
  int few_rows;                        // the kernel of few rows takes the sequences with at most this many queries, that of many the others
};

// A tensor map of the pool [channel, token, head, page] (head before token where heads are nearer to one another), with what its loads go by.
struct alignas(64) PagedMap {
  CUtensorMap map;
  int dim_shift;           // head_dim = 1 << dim_shift
};

// Runs of keys begin where the loads of a tile can: at a multiple of 16 tokens, or of whole tiles where no window moves them.
__device__ __forceinline__ int key_align(const PagedParams& p) { return p.key_align; }

__device__ __forceinline__ int paged_keys(const PagedParams& p, int seg) { return max(min(p.seqlens_k[seg], p.columns << p.page_shift), 0); }

// The tile kernel's view of a sequence.  Its keys are numbered through all sequences, seg * columns * P + j.
__device__ __forceinline__ WindowSeq paged_seq(const PagedParams& p, int seg) {
  WindowSeq s;
  s.q_begin = p.f.cu_q != nullptr ? p.f.cu_q[seg] : 0;
  s.q_len = p.f.cu_q != nullptr ? p.f.cu_q[seg + 1] - s.q_begin : p.f.seqlen_q;
  s.q_len = max(min(s.q_len, p.f.seqlen_q), 0);
  s.k_begin = seg * (p.columns << p.page_shift);
  s.k_len = paged_keys(p, seg);
  const int64_t x = static_cast<int64_t>(s.k_len) - s.q_len;
  s.from = p.left < 0 ? -kFar : clamp_position(x - p.left);
  s.to = p.right < 0 ? kFar : clamp_position(x + p.right + 1);
  s.sinks = max(min(p.sinks, s.k_len), 0);
  return s;
}
__device__ __forceinline__ WindowSeq window_seq(const PagedParams& p, int seg) {
  WindowSeq s = paged_seq(p, seg);
  if (s.q_len <= p.few_rows) s.q_len = 0;
  return s;
}

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, int a, int b, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(a), "r"(b), "r"(page)
      : "memory");
}

__device__ __forceinline__ void prefetch_tmap(const PagedMap* m) { prefetch_tmap(&m->map); }

// Loads of tiles over pages.  The thread that walks a block's tiles asks for them, and two warps that have no other role look the pages up and
// issue the loads, a lane to each 64 channels of a box.  (One thread that does all of it is what bounds a launch: 16 loads of 2 KB and 8
// look-ups for a tile at D = 128 and pages of 16, which a step of 1.6 us takes two of.)  A request's place in the queue is taken again only
// when the tile's slot in the ring is, that is, after its loads have landed: there are more places than loads in the ring, and nothing to wait for.
constexpr int kLoadPlaces = 16;
constexpr int kLoadWarps = 2;            // they take requests in turn
struct LoadRequest {
  const PagedMap* map;                   // null: no more
  uint64_t* bar;
  uint8_t* dst;
  int token, head, head_first;
};
struct LoadQueue {
  LoadRequest at[kLoadPlaces];
  uint64_t posted[kLoadPlaces];          // barriers: a request is there
  uint32_t n;                            // requests so far, of the thread that asks
};
__device__ __forceinline__ LoadQueue& load_queue() {
  __shared__ LoadQueue queue;
  return queue;
}
__device__ __forceinline__ void post_load(const LoadRequest& r) {
  LoadQueue& q = load_queue();
  const uint32_t i = q.n++ % kLoadPlaces;
  q.at[i] = r;
  mbar_arrive(&q.posted[i]);
}

// The first 64 channels' call asks for all of a tile: 128 tokens from `token` (counted through all sequences, a multiple of the box).
__device__ __forceinline__ void tma_load_token(void* smem_dst, const PagedMap* m, uint64_t* bar, int x, int token, int /*batch*/, int head_first) {
  if ((x & ((1 << m->dim_shift) - 1)) == 0) post_load(LoadRequest{m, bar, static_cast<uint8_t*>(smem_dst), token, x >> m->dim_shift, head_first});
}

// What the kernel of tiles does for its loads beside its loader: nothing where keys are dense.
__device__ __forceinline__ void init_loads(const WindowParams&) {}
__device__ __forceinline__ void end_loads(const WindowParams&) {}
template <int D>
__device__ __forceinline__ void serve_loads(const WindowParams&, int) {}

__device__ __forceinline__ void init_loads(const PagedParams&) {         // by one thread
  LoadQueue& q = load_queue();
  q.n = 0;
  for (int i = 0; i < kLoadPlaces; ++i) mbar_init(&q.posted[i], 1);
}
__device__ __forceinline__ void end_loads(const PagedParams&) {          // by the thread that asks
  for (int i = 0; i < kLoadWarps; ++i) post_load(LoadRequest{nullptr, nullptr, nullptr, 0, 0, 0});
}
// By a whole warp, the `which`th of them.  What lies behind the table's last column, or in a page outside the pool, is filled with zeros by the
// load (its page number is one past the last).
template <int D>
__device__ __forceinline__ void serve_loads(const PagedParams& p, int which) {
  constexpr int kSlabs = D / 64;
  LoadQueue& q = load_queue();
  const int lane = threadIdx.x & 31, slab = lane % kSlabs, at = lane / kSlabs * p.box_rows;       // this lane's box begins at that token
  const int span = p.columns << p.page_shift;
  for (uint32_t n = which;; n += kLoadWarps) {
    const uint32_t i = n % kLoadPlaces;
    if (!flash::warp_wait_or_abort(&q.posted[i], (n / kLoadPlaces) & 1, p.f.status, 16)) break;
    const LoadRequest r = q.at[i];
    if (r.map == nullptr) break;
    if (at < 128) {
      const int seq = r.token / span, pos = r.token - seq * span + at, j = pos >> p.page_shift;
      int page = -1;
      if (j < p.columns) page = p.table[static_cast<int64_t>(seq) * p.columns + j];
      if (page < 0 || page >= p.pages) page = p.pages;
      const int in_page = pos & ((1 << p.page_shift) - 1);
      tma_load_4d(r.dst + slab * (128 * 128) + at * 128, &r.map->map, r.bar, slab * 64, r.head_first ? r.head : in_page, r.head_first ? in_page : r.head, page);
    }
    __syncwarp();
  }
}

// Tiles of 128: q [heads * D, tokens, batch] as for the dense kernel.
template <int D>
cudaError_t launch_paged_tiles(const CUtensorMap& tm_q, const PagedMap& tm_k, const PagedMap& tm_v, const PagedParams& p, cudaStream_t stream);

// Few rows: blocks of 16, 32 or 64.  Scratch holds the states of sequences that more than one CTA works on.
struct PagedRowsPlan {
  int rows;                // of a block
  int ctas;                // at most
  int64_t scratch_bytes;
};
// (rows of a key head's longest sequence; `keys` of the longest sequence, about: more CTAs than that needs would not be used)
PagedRowsPlan plan_paged_rows(int64_t rows_of_a_head, int64_t keys, int64_t kv_heads, int64_t nseg, int head_dim, int sm_count);
template <int D>
cudaError_t launch_paged_rows(const PagedMap& tm_k, const PagedMap& tm_v, const PagedParams& p, const PagedRowsPlan& plan, void* scratch, cudaStream_t stream);

}  // namespace dtb
