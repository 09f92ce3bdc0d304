// Parameters and launcher of the merge of partial states some of which are held in 8 bits (merge_rows.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dtb {

constexpr int kMergeRowsMaxStates = 16;

// Types of a state's values, as DTB_F32 ... DTB_E4M3 of the C interface.
constexpr int kRowsF32 = 0, kRowsBf16 = 1, kRowsI8 = 2, kRowsE4m3 = 3;

struct MergeRowsParams {
  const void* values[kMergeRowsMaxStates];       // [rows, D]; the states in 8 bits come first
  const uint8_t* exponents[kMergeRowsMaxStates]; // [rows], of the states in 8 bits
  const float* lse[kMergeRowsMaxStates];
  int dtype[kMergeRowsMaxStates];
  int lse_layout[kMergeRowsMaxStates];           // 0 [B,H,S], 1 [B,S,H]
  int narrow;                                    // states in 8 bits
  int nstates;
  float* out;                                    // fp32 result, or null
  uint16_t* out_bf16;                            // bf16 result, or null
  uint8_t* out_codes;                            // 8-bit result, or null
  uint8_t* out_exponents;
  int out_codes_dtype;
  float* lse_out;                                // may be null
  int lse_out_layout;
  int64_t rows;                                  // B*S*H, below 2^31
  int H;
  int S;
};

// A single state's values in 8 bits, and back: `rows` (below 2^31) rows of head_dim.
cudaError_t launch_quantize_rows(const void* values, bool bf16, uint8_t* codes, uint8_t* exponents, int codes_dtype, int64_t rows, int head_dim,
                                 cudaStream_t stream);
cudaError_t launch_dequantize_rows(const uint8_t* codes, const uint8_t* exponents, int codes_dtype, void* out, bool bf16, int64_t rows, int head_dim,
                                   cudaStream_t stream);
cudaError_t launch_merge_rows(const MergeRowsParams& p, int head_dim, int sm_count, cudaStream_t stream);

}  // namespace dtb
