// Attention over keys and values that lie in pages: what the kernels are given (flash_paged_rows.cu for few query rows, flash_window_sm100.cu
// for many), and how a sequence's keys are found.
//
// Page n of a pool holds P tokens (a power of two, at least 16); key j of sequence b is token j % P of page table[b][j / P].  A page number
// outside the pool stands for keys and values of 0.
#pragma once
#include "flash_window.cuh"
#include "ptx_sm100.cuh"

namespace dtb {

struct PagedParams : WindowParams {    // (k, v, their strides, cu_k and k_start are not used; seqlens_k is given always)
  const int32_t* table;                // [sequences, columns]
  int columns, pages, page_shift;
  int box_rows;                        // tokens of a tile that one load fetches; divides a page, so that no load crosses one
  int key_align;                       // runs of keys are walked from a multiple of this
  int few_rows;                        // the kernel of few rows takes the sequences with at most this many queries, that of many the others
};

// A tensor map of the pool [channel, token, head, page] (head before token where heads are nearer to one another), with what its loads need.
struct alignas(64) PagedMap {
  CUtensorMap map;
  const int32_t* table;
  int columns, pages, page_shift, box_rows, dim_shift;
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

// 64 channels of 128 tokens from `token` (counted through all sequences, a multiple of the box), page by page; what lies behind the
// table's last column, or in a page outside the pool, is filled with zeros by the load (its page number is one past the last).
__device__ __forceinline__ void tma_load_token(void* smem_dst, const PagedMap* m, uint64_t* bar, int x, int token, int /*batch*/, int head_first) {
  const int span = m->columns << m->page_shift, seq = token / span, pos = token - seq * span;
  const int32_t* row = m->table + static_cast<int64_t>(seq) * m->columns;
  const int head = x >> m->dim_shift, ch = x & ((1 << m->dim_shift) - 1), box = m->box_rows;
  int page[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    page[i] = -1;
    const int j = (pos + i * box) >> m->page_shift;
    if (i * box < 128 && j < m->columns) page[i] = row[j];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i * box < 128) {
      const int n = page[i] >= 0 && page[i] < m->pages ? page[i] : m->pages, in_page = (pos + i * box) & ((1 << m->page_shift) - 1);
      tma_load_4d(static_cast<uint8_t*>(smem_dst) + i * box * 128, &m->map, bar, ch, head_first ? head : in_page, head_first ? in_page : head, n);
    }
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
PagedRowsPlan plan_paged_rows(int rows_of_a_head, int head_dim, int sm_count);
template <int D>
cudaError_t launch_paged_rows(const PagedMap& tm_k, const PagedMap& tm_v, const PagedParams& p, const PagedRowsPlan& plan, void* scratch, cudaStream_t stream);

}  // namespace dtb
