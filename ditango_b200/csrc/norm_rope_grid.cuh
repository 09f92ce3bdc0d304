// Parameters and launchers of the query / key norm with rotary positions on three axes, and of its gradients (norm_rope_grid.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dtb {

struct NormRopeGridParams {
  const void* src[2];            // query and key projections: token s of sequence b, head h at b * batch_stride + s * tok_stride + h * D
  int64_t tok_stride[2];
  int64_t batch_stride[2];
  const void* grad[2];           // backward: gradients of the results, strides of their own
  int64_t grad_tok_stride[2];
  int64_t grad_batch_stride[2];
  void* dst[2];                  // results, or gradients of src: [batch, seq, heads, D] contiguous
  const void* weight[2];         // [D]
  const void* bias[2];           // [D] or null
  float* partial;                // backward: scratch, a row of 2 D sums for each CTA
  float eps[2];
  int heads[2];
  int64_t tokens;                // batch * seq
  int seq;
  int text_len;                  // tokens in front of the grid's
  int video_len;                 // tokens of the grid (and padding); what follows is text again
  int64_t first;                 // number of the token behind the text among those of the grid and its padding
  // the grid's T Y X places lie in `shards` pieces of shard_len tokens: shard_rest of them with shard_places + 1 places, the
  // others with shard_places, the rest of a piece padding
  int shards, shard_len, shard_places, shard_rest;
  int size_y, size_x;
  double origin[3], step[3];
  // the i'th pair of an axis with d channels turns by base^(-2 i / d) = ratio^i; axis a has the pairs up to pairs_end[a]
  double ratio[3];
  int pairs_end[3];
};

cudaError_t launch_norm_rope_grid(const NormRopeGridParams& p, int head_dim, bool bf16, bool rms, int sm_count, cudaStream_t stream);
// Bytes behind p.partial that the backward pass needs.
int64_t norm_rope_grid_scratch_bytes(int head_dim, int sm_count);
// What the sums become: [D] each, or null.
struct NormRopeGridSums {
  void* weight_grad[2];
  void* bias_grad[2];
};
cudaError_t launch_norm_rope_grid_backward(const NormRopeGridParams& p, const NormRopeGridSums& sums, int head_dim, bool bf16, bool rms, int sm_count, cudaStream_t stream);

}  // namespace dtb
