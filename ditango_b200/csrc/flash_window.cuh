// Parameters and launchers of the windowed attention kernels (flash_window_rows.cu for few query rows, flash_window_sm100.cu for
// many), and which keys a row sees.
#pragma once
#include "flash_fwd_sm100.cuh"

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace dtb {

constexpr int kQueriesLast = INT32_MIN;      // q_start: the queries are the last positions of their sequence

struct WindowParams {
  FlashParams f;                 // (scale, results, lengths; out is contiguous)
  const uint16_t* q;             // token t of sequence b, head h: q + b * q_batch + t * q_tok + h * D
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_tok, q_batch, k_tok, k_batch, v_tok, v_batch;      // elements; packed: no batch strides
  const int32_t* seqlens_k;      // keys of each sequence of a dense batch, or null: all seqlen_k
  int kv_heads;                  // divides f.num_heads
  int left, right, sinks;        // each within [0, 2^30]; left, right -1: no limit
  int q_start, k_start;          // positions of the first query (or kQueriesLast) and the first key
  // the order of a tensor map's outer axes, the one with the smaller stride first: 1 batch then token, 0 token then batch
  int q_batch_first, k_batch_first, v_batch_first;
  // Parts that the keys of a block of 256 rows are split into, each attended like a block of its own.  With more than one, f.out and
  // f.lse (fp32, [B,S,H]) hold the parts' states one after another, f.total_q tokens each, for a merge.
  int splits;
};

// A sequence: where its queries and keys begin among the tokens, how many there are, and which keys its first query sees: [0, sinks) as
// far as it sees them, and from `from` up to `to`, which move on by one with every query.
struct WindowSeq {
  int q_begin, q_len, k_begin, k_len;
  int from, to, sinks;
};

constexpr int kFar = 1 << 30;                       // beyond all keys, and a query's number can still be added
__device__ __forceinline__ int clamp_position(int64_t x) {
  return static_cast<int>(x < -kFar ? -kFar : x > kFar ? kFar : x);
}

__device__ __forceinline__ WindowSeq window_seq(const WindowParams& p, int seg) {
  WindowSeq s;
  if (p.f.cu_q != nullptr) {
    s.q_begin = p.f.cu_q[seg];
    s.q_len = p.f.cu_q[seg + 1] - s.q_begin;
    s.k_begin = p.f.cu_k[seg];
    s.k_len = p.f.cu_k[seg + 1] - s.k_begin;
  } else {
    s.q_begin = s.k_begin = 0;
    s.q_len = p.f.seqlen_q;
    s.k_len = p.f.seqlen_k;
    if (p.seqlens_k != nullptr) s.k_len = min(p.seqlens_k[seg], s.k_len);
  }
  s.q_len = max(min(s.q_len, p.f.seqlen_q), 0);
  s.k_len = max(min(s.k_len, p.f.seqlen_k), 0);
  // the first query's position, counted from the first key
  const int64_t x = p.q_start == kQueriesLast ? static_cast<int64_t>(s.k_len) - s.q_len : static_cast<int64_t>(p.q_start) - p.k_start;
  s.from = p.left < 0 ? -kFar : clamp_position(x - p.left);
  s.to = p.right < 0 ? kFar : clamp_position(x + p.right + 1);
  s.sinks = max(min(clamp_position(static_cast<int64_t>(p.sinks) - p.k_start), s.k_len), 0);
  return s;
}

// Of what number of keys a run that is walked begins at a multiple.  (Dense keys: anywhere.)
__device__ __forceinline__ constexpr int key_align(const WindowParams&) { return 1; }
template <class Walk>
__device__ __forceinline__ constexpr int front_of(const WindowParams&, const Walk&) { return 0; }
// Which block a CTA's place in the grid stands for: row block, head, sequence x parts, and the parts that its keys are split into.
__device__ __forceinline__ void place_block(const WindowParams&, int&, int&, int&, int&, int&) {}
// Whether a CTA that is done with a block claims one of the grid's that has not started; else next_place says which place is its next, if any.
__device__ __forceinline__ constexpr bool claims_blocks(const WindowParams&) { return true; }
__device__ __forceinline__ constexpr bool next_place(const WindowParams&, int&) { return false; }
// Rows are queries (here: times 1 << 0 heads), and where a block's results go, whichever part of its keys it has.
__device__ __forceinline__ constexpr int row_shift(const WindowParams&) { return 0; }
template <class Item>
__device__ __forceinline__ void place_results(const WindowParams&, Item&, int) {}
template <class Item>
__device__ __forceinline__ const FlashParams& results_at(const WindowParams& p, const Item&) { return p.f; }

// Keys that query i sees: [0, first) and [lo, hi), first <= lo <= hi.  A key at position j is seen from position x when
// j <= x + right and (j >= x - left or j < sinks).
struct WindowSpan {
  int first, lo, hi;
};

// `k_end`: no key from there on; `k_floor`: the window holds no key before it (sinks, or more where a block's keys are split).
__device__ __forceinline__ WindowSpan window_span(int from, int to, int sinks, int k_end, int k_floor, int i) {
  WindowSpan w;
  w.hi = min(max(to + i, 0), k_end);
  w.first = min(sinks, w.hi);
  w.lo = max(min(max(from + i, k_floor), w.hi), w.first);
  return w;
}
__device__ __forceinline__ WindowSpan window_span(const WindowSeq& s, int i) { return window_span(s.from, s.to, s.sinks, s.k_len, s.sinks, i); }

// Element offset of a sequence's token in a q / k / v tensor (dense: token inside its sequence; packed: of the whole tensor).
__device__ __forceinline__ int64_t window_offset(const WindowParams& p, int seg, int64_t tok, int64_t tok_stride, int64_t batch_stride) {
  return (p.f.cu_q != nullptr ? 0 : seg * batch_stride) + tok * tok_stride;
}

// Tensor maps of q, k and v: [heads * D, tokens, batch] (or batch and tokens changed over), boxes of 64 channels x 128 tokens.
template <int D>
cudaError_t launch_window_tiles(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowParams& p, cudaStream_t stream);
template <int D>
cudaError_t launch_window_rows(const WindowParams& p, int sm_count, cudaStream_t stream);

}  // namespace dtb
