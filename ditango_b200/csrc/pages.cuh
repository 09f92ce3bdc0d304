// Pages of keys and values: tables of them made longer and shorter, and tokens written into them (pages.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dtb {

constexpr int kMostStreams = 16384;      // of a table that is made longer (12 bytes of shared memory each)

struct ExtendParams {
  int32_t* table;                        // [streams, columns]
  const int32_t* seqlens;                // [streams]
  const int32_t* new_lens;               // [streams]
  const int32_t* free_pages;             // [pages]: the first *free_count are free, the last of those is taken first
  const int32_t* free_count;
  int32_t* slots;                        // [tokens]
  int32_t* cu_seqlens;                   // [streams + 1]
  int32_t* seqlens_out;
  int32_t* count_out;
  int32_t* missing;
  int streams, columns, pages, page_shift, tokens;
};

struct ReleaseParams {
  const int32_t* table;
  int32_t* table_out;                    // may be table
  const int32_t* seqlens;
  const int32_t* begin;
  const int32_t* end;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* seqlens_out;
  int32_t* count_out;
  int streams, columns, pages, page_shift;
};
constexpr int kReleaseColumns = 256;     // entries of a stream that a warp looks at together
constexpr int kReleaseCtas = 8;          // of the cluster, at most
constexpr int kReleaseItems = 32768;     // of such pieces to a CTA, at most

struct WriteParams {
  const uint16_t* src[2];                // keys and values of the new tokens
  int64_t src_tok[2];                    // elements
  uint16_t* dst[2];
  int64_t dst_page[2], dst_tok[2], dst_head[2];
  const int32_t* slots;
  int tokens, heads, head_shift;         // head_dim = 1 << head_shift
  int page_shift;
  int64_t capacity;                      // slots of the pool
};

cudaError_t launch_extend_pages(const ExtendParams& p, int sm_count, cudaStream_t stream);
cudaError_t launch_release_pages(const ReleaseParams& p, cudaStream_t stream);
cudaError_t launch_write_pages(const WriteParams& p, cudaStream_t stream);

}  // namespace dtb
