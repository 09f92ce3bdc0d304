// Merge of partial softmax-attention states of which some are held in 8 bits, and states written in 8 bits, in one pass.
//
//   out = sum_i w_i v_i,  w_i = exp(lse_i - lse),  lse = log sum_i exp(lse_i)
//   in 8 bits  v = code * 2^(b - 127):  b is the smallest exponent byte (at least 8) with max|v| <= M 2^(b - 127), M the largest
//              code (127 of int8, 448 of e4m3), code = v 2^(127 - b) rounded to nearest, ties to even
// A row is one (token, head) pair and has one b.  A power of two, and not max|v| / M: then v 2^(127 - b) is exact, so that the
// code's rounding is the only one, the value it stands for is a bf16 number (at most 7 bits behind the leading one), and the
// factor is one byte and goes into the weight.  It costs int8 up to one bit of its 7, and e4m3 (a floating type) nothing.
// A row with an infinity or a NaN gets b = 255: its codes are 0, and 0 * 2^128 reads back as NaN.
//
// Bound by HBM.  In the merge D / 16 lanes own a row, 16 values each: 16 bytes of a state in 8 bits.  The 8-bit states come first in the
// parameters and are fetched kNarrow at a time, all of those loads and the first wide state's in flight before the weights (which
// wait for the lse) are formed.  All sums are fp32.
#include "merge_rows.cuh"

#include "row_access.cuh"

#include <cuda_fp8.h>
#include <math.h>

namespace dtb {

namespace {

constexpr int kThreads = 128;
constexpr int kMinExponent = 8;      // 2^(127 - b) stays finite; below 2^-111 of a row's maximum nothing is lost that matters

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 2^(b - 127); 0 for b = 0, infinity for b = 255
__device__ __forceinline__ float power_of(uint32_t b) { return __uint_as_float(b << 23); }

// 16 values of a wide state as loaded: fp32 in all four, bf16 in the first two.
struct Wide {
  uint4 q[4];
};

__device__ __forceinline__ void load_wide(Wide& w, const void* values, int dtype, int64_t off) {
  if (dtype == kRowsF32) {
    const float* src = static_cast<const float*>(values) + off;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.q[i] = ld_stream(src + 4 * i);
  } else {
    const uint16_t* src = static_cast<const uint16_t*>(values) + off;
    w.q[0] = ld_stream(src);
    w.q[1] = ld_stream(src + 8);
  }
}
__device__ __forceinline__ void add_wide(float (&acc)[16], float w, const Wide& v, int dtype) {
  if (dtype == kRowsF32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[4 * i] = fmaf(w, __uint_as_float(v.q[i].x), acc[4 * i]);
      acc[4 * i + 1] = fmaf(w, __uint_as_float(v.q[i].y), acc[4 * i + 1]);
      acc[4 * i + 2] = fmaf(w, __uint_as_float(v.q[i].z), acc[4 * i + 2]);
      acc[4 * i + 3] = fmaf(w, __uint_as_float(v.q[i].w), acc[4 * i + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a[4] = {v.q[i].x, v.q[i].y, v.q[i].z, v.q[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        acc[8 * i + 2 * k] = fmaf(w, __uint_as_float(a[k] << 16), acc[8 * i + 2 * k]);
        acc[8 * i + 2 * k + 1] = fmaf(w, __uint_as_float(a[k] & 0xffff0000u), acc[8 * i + 2 * k + 1]);
      }
    }
  }
}
// The four codes of a word as floats.
__device__ __forceinline__ void decode4(uint32_t a, int dtype, float (&f)[4]) {
  if (dtype == kRowsI8) {
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = static_cast<float>(static_cast<int8_t>(a >> (8 * k)));
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(a >> (16 * k)), __NV_E4M3);
      const float2 x = __half22float2(h);
      f[2 * k] = x.x;
      f[2 * k + 1] = x.y;
    }
  }
}
__device__ __forceinline__ void add_codes(float (&acc)[16], float w, uint4 v, int dtype) {
  const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
    decode4(a[i], dtype, f);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[4 * i + k] = fmaf(w, f[k], acc[4 * i + k]);
  }
}

// The exponent byte of a row whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t exponent_byte(uint32_t top, int dtype) {
  if (top >= 0x7f800000u) return 255u;
  // round the exponent up where the mantissa is above that of the largest code: 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
  const int b = dtype == kRowsI8 ? static_cast<int>((top + (0x7fffffu - 0x7e0000u)) >> 23) - 6
                                 : static_cast<int>((top + (0x7fffffu - 0x600000u)) >> 23) - 8;
  return static_cast<uint32_t>(b < kMinExponent ? kMinExponent : b);
}
// Four values as codes of a row with exponent byte b; f = 2^(127 - b).
__device__ __forceinline__ uint32_t encode4(float x0, float x1, float x2, float x3, uint32_t b, float f, int dtype) {
  if (b == 255u) return 0u;
  x0 *= f;
  x1 *= f;
  x2 *= f;
  x3 *= f;
  if (dtype == kRowsI8)
    return (static_cast<uint32_t>(__float2int_rn(x0)) & 0xffu) | (static_cast<uint32_t>(__float2int_rn(x1)) & 0xffu) << 8 |
           (static_cast<uint32_t>(__float2int_rn(x2)) & 0xffu) << 16 | static_cast<uint32_t>(__float2int_rn(x3)) << 24;
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3)) |
         static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x2, x3), __NV_SATFINITE, __NV_E4M3)) << 16;
}
__device__ __forceinline__ float inverse_of(uint32_t b) { return __uint_as_float((254u - b) << 23); }

}  // namespace

// G = D / 16 lanes per row, U rows per group in flight, 8-bit states fetched kNarrow at a time.
template <int G, int U, int kNarrow>
__global__ void __launch_bounds__(kThreads) merge_rows_kernel(const MergeRowsParams p) {
  constexpr int D = G * 16;
  constexpr int kGroupsPerWarp = 32 / G;
  constexpr int kPerLane = kMergeRowsMaxStates / G;    // states whose lse a lane holds: lane, lane + G, ...
  constexpr unsigned full = 0xffffffffu;
  const int lane = threadIdx.x % G;
  const int64_t warp_id = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / 32;
  const int64_t n_warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  const int group = (threadIdx.x % 32) / G;
  const int n = p.nstates, n8 = p.narrow;

  // (the bound is the same for all lanes of a warp: the shuffles below use the full mask)
  for (int64_t wbase = warp_id * kGroupsPerWarp * U; wbase < p.rows; wbase += n_warps * kGroupsPerWarp * U) {
    // rows of a group are kGroupsPerWarp apart, so that the warp's accesses of one step are to consecutive rows
    const int64_t base = wbase + group;
    auto row_of = [&](int u) { return base + u * kGroupsPerWarp; };
    uint4 code[kNarrow][U];
    Wide wide[U];
    auto load_codes = [&](int c0) {
#pragma unroll
      for (int k = 0; k < kNarrow; ++k)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          code[k][u] = make_uint4(0u, 0u, 0u, 0u);
          if (c0 + k < n8 && row_of(u) < p.rows)
            code[k][u] = ld_stream(static_cast<const uint8_t*>(p.values[c0 + k]) + row_of(u) * D + lane * 16);
        }
    };
    auto load_wides = [&](int st) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (st < n && row_of(u) < p.rows) load_wide(wide[u], p.values[st], p.dtype[st], row_of(u) * D + lane * 16);
    };
    float w[U][kPerLane], lse_out[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) wide[u].q[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < kPerLane; ++t) {
        const int st = lane + t * G;
        w[u][t] = -INFINITY;
        if (row_of(u) < p.rows && st < n)
          w[u][t] = p.lse[st][lse_offset(p.lse_layout[st], static_cast<uint32_t>(row_of(u)), p.H, p.S)];
      }
    uint32_t eb[U][kPerLane];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < kPerLane; ++t) {
        const int st = lane + t * G;
        eb[u][t] = 127u;
        if (row_of(u) < p.rows && st < n8) eb[u][t] = p.exponents[st][row_of(u)];
      }
    load_codes(0);
    load_wides(n8);

#pragma unroll
    for (int u = 0; u < U; ++u) {
      float mx = w[u][0];
#pragma unroll
      for (int t = 1; t < kPerLane; ++t) mx = fmaxf(mx, w[u][t]);
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(full, mx, o, G));
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < kPerLane; ++t) {
        w[u][t] = w[u][t] == -INFINITY ? 0.f : exp2f((w[u][t] - mx) * 1.4426950408889634f);
        sum += w[u][t];
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(full, sum, o, G);
      lse_out[u] = sum > 0.f ? mx + logf(sum) : -INFINITY;
#pragma unroll
      for (int t = 0; t < kPerLane; ++t) w[u][t] = sum > 0.f ? __fdiv_rn(w[u][t], sum) : 0.f;
      // the factor of a state in 8 bits goes into its weight; a weight of 0 stays one
#pragma unroll
      for (int t = 0; t < kPerLane; ++t)
        if (w[u][t] != 0.f && lane + t * G < n8) w[u][t] *= power_of(eb[u][t]);
    }

    float acc[U][16];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[u][i] = 0.f;
    auto weight = [&](int u, int st) {
      float mine = w[u][0];
#pragma unroll
      for (int t = 1; t < kPerLane; ++t) mine = st / G == t ? w[u][t] : mine;
      return __shfl_sync(full, mine, st % G, G);
    };
    for (int c0 = 0; c0 < n8; c0 += kNarrow) {
#pragma unroll
      for (int k = 0; k < kNarrow; ++k)
        if (c0 + k < n8) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const float wi = weight(u, c0 + k);
            // a state of weight 0 may hold anything, a NaN too: it must not reach the sum
            if (wi != 0.f) add_codes(acc[u], wi, code[k][u], p.dtype[c0 + k]);
          }
        }
      if (c0 + kNarrow < n8) load_codes(c0 + kNarrow);
    }
    for (int st = n8; st < n; ++st) {
      const int dtype = p.dtype[st];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float wi = weight(u, st);
        if (wi != 0.f) add_wide(acc[u], wi, wide[u], dtype);
      }
      load_wides(st + 1);
    }

#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row_of(u);
      const int64_t off = row * D + lane * 16;
      if (p.out_codes != nullptr) {
        uint32_t top = 0u;            // magnitudes compare as their bits do, NaNs above all
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(acc[u][i]) & 0x7fffffffu);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(full, top, o, G));
        const uint32_t b = exponent_byte(top, p.out_codes_dtype);
        if (row < p.rows) {
          const float f = inverse_of(b);
          uint32_t r[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            r[i] = encode4(acc[u][4 * i], acc[u][4 * i + 1], acc[u][4 * i + 2], acc[u][4 * i + 3], b, f, p.out_codes_dtype);
          st_stream(p.out_codes + off, make_uint4(r[0], r[1], r[2], r[3]));
          if (lane == 0) p.out_exponents[row] = static_cast<uint8_t>(b);
        }
      }
      if (row < p.rows) {
        if (p.out != nullptr) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            st_stream(p.out + off + i, make_uint4(__float_as_uint(acc[u][i]), __float_as_uint(acc[u][i + 1]),
                                                  __float_as_uint(acc[u][i + 2]), __float_as_uint(acc[u][i + 3])));
        }
        if (p.out_bf16 != nullptr) {
#pragma unroll
          for (int i = 0; i < 16; i += 8)
            st_stream(p.out_bf16 + off + i, make_uint4(pack_bf16(acc[u][i], acc[u][i + 1]), pack_bf16(acc[u][i + 2], acc[u][i + 3]),
                                                       pack_bf16(acc[u][i + 4], acc[u][i + 5]), pack_bf16(acc[u][i + 6], acc[u][i + 7])));
        }
        if (p.lse_out != nullptr && lane == 0)
          p.lse_out[lse_offset(p.lse_out_layout, static_cast<uint32_t>(row), p.H, p.S)] = lse_out[u];
      }
    }
  }
}

// A single state written in 8 bits: D / 8 lanes to a row, 8 values each, kRowsPerThread rows whose loads are in flight together.  (The
// two halves of an fp32 row are loaded one after the other, four values a lane, so that each access is to whole lines.)
constexpr int kCodeThreads = 256;
constexpr int kRowsPerThread = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kCodeThreads) quantize_rows_kernel(const T* values, uint8_t* codes, uint8_t* exponents, int codes_dtype, int64_t rows) {
  constexpr int G = D / 8, U = kRowsPerThread;
  constexpr bool f32 = sizeof(T) == 4;
  const int lane = threadIdx.x % G;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kCodeThreads / G * U) + threadIdx.x / G;
  uint4 raw[U][f32 ? 2 : 1];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = row0 + u * (kCodeThreads / G);
    raw[u][0] = make_uint4(0u, 0u, 0u, 0u);
    if (f32) raw[u][f32 ? 1 : 0] = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows) {
      raw[u][0] = ld_stream(values + row * D + lane * (f32 ? 4 : 8));
      if (f32) raw[u][f32 ? 1 : 0] = ld_stream(values + row * D + D / 2 + lane * 4);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = row0 + u * (kCodeThreads / G);
    float x[8];
    const uint32_t a[4] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w};
    if (f32) {
      const uint4 v = raw[u][f32 ? 1 : 0];
      const uint32_t b[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __uint_as_float(a[i]);
        x[4 + i] = __uint_as_float(b[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(a[i] << 16);
        x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
      }
    }
    uint32_t top = 0u;                // magnitudes compare as their bits do, NaNs above all
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o, G));
    const uint32_t b = exponent_byte(top, codes_dtype);
    const float f = inverse_of(b);
    const uint32_t r0 = encode4(x[0], x[1], x[2], x[3], b, f, codes_dtype), r1 = encode4(x[4], x[5], x[6], x[7], b, f, codes_dtype);
    if (row < rows) {
      if (f32) {
        *reinterpret_cast<uint32_t*>(codes + row * D + lane * 4) = r0;
        *reinterpret_cast<uint32_t*>(codes + row * D + D / 2 + lane * 4) = r1;
      } else {
        *reinterpret_cast<uint2*>(codes + row * D + lane * 8) = make_uint2(r0, r1);
      }
      if (lane == 0) exponents[row] = static_cast<uint8_t>(b);
    }
  }
}

// ... and read back.
template <typename T, int D>
__global__ void __launch_bounds__(kCodeThreads) dequantize_rows_kernel(const uint8_t* codes, const uint8_t* exponents, T* out, int codes_dtype, int64_t rows) {
  constexpr int G = D / 8, U = kRowsPerThread;
  const int lane = threadIdx.x % G;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kCodeThreads / G * U) + threadIdx.x / G;
  uint2 raw[U];
  uint32_t b[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = row0 + u * (kCodeThreads / G);
    raw[u] = make_uint2(0u, 0u);
    b[u] = 0u;
    if (row < rows) {
      raw[u] = __ldcs(reinterpret_cast<const uint2*>(codes + row * D + lane * 8));
      b[u] = exponents[row];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = row0 + u * (kCodeThreads / G);
    if (row >= rows) break;
    const float f = power_of(b[u]);
    float x[4], y[4];
    decode4(raw[u].x, codes_dtype, x);
    decode4(raw[u].y, codes_dtype, y);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] *= f;
      y[i] *= f;
    }
    T* dst = out + row * D + lane * 8;
    if (sizeof(T) == 4) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(y[0], y[1], y[2], y[3]);
    } else {
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    }
  }
}

static unsigned code_blocks(int64_t rows, int head_dim) {
  const int64_t per_block = kCodeThreads / (head_dim / 8) * kRowsPerThread;
  return static_cast<unsigned>((rows + per_block - 1) / per_block);
}

cudaError_t launch_quantize_rows(const void* values, bool bf16, uint8_t* codes, uint8_t* exponents, int codes_dtype, int64_t rows, int head_dim,
                                 cudaStream_t stream) {
  const unsigned blocks = code_blocks(rows, head_dim);
  const uint16_t* h = static_cast<const uint16_t*>(values);
  const float* f = static_cast<const float*>(values);
  if (head_dim == 64) {
    if (bf16) quantize_rows_kernel<uint16_t, 64><<<blocks, kCodeThreads, 0, stream>>>(h, codes, exponents, codes_dtype, rows);
    else quantize_rows_kernel<float, 64><<<blocks, kCodeThreads, 0, stream>>>(f, codes, exponents, codes_dtype, rows);
  } else {
    if (bf16) quantize_rows_kernel<uint16_t, 128><<<blocks, kCodeThreads, 0, stream>>>(h, codes, exponents, codes_dtype, rows);
    else quantize_rows_kernel<float, 128><<<blocks, kCodeThreads, 0, stream>>>(f, codes, exponents, codes_dtype, rows);
  }
  return cudaGetLastError();
}

cudaError_t launch_dequantize_rows(const uint8_t* codes, const uint8_t* exponents, int codes_dtype, void* out, bool bf16, int64_t rows, int head_dim,
                                   cudaStream_t stream) {
  const unsigned blocks = code_blocks(rows, head_dim);
  uint16_t* h = static_cast<uint16_t*>(out);
  float* f = static_cast<float*>(out);
  if (head_dim == 64) {
    if (bf16) dequantize_rows_kernel<uint16_t, 64><<<blocks, kCodeThreads, 0, stream>>>(codes, exponents, h, codes_dtype, rows);
    else dequantize_rows_kernel<float, 64><<<blocks, kCodeThreads, 0, stream>>>(codes, exponents, f, codes_dtype, rows);
  } else {
    if (bf16) dequantize_rows_kernel<uint16_t, 128><<<blocks, kCodeThreads, 0, stream>>>(codes, exponents, h, codes_dtype, rows);
    else dequantize_rows_kernel<float, 128><<<blocks, kCodeThreads, 0, stream>>>(codes, exponents, f, codes_dtype, rows);
  }
  return cudaGetLastError();
}

template <int G, int U, int kNarrow>
static cudaError_t launch_cfg(const MergeRowsParams& p, int sm_count, cudaStream_t stream) {
  int per_sm = 0;
  cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, merge_rows_kernel<G, U, kNarrow>, kThreads, 0);
  if (e != cudaSuccess) return e;
  const int64_t rows_per_block = kThreads / G * U;
  const int64_t need = (p.rows + rows_per_block - 1) / rows_per_block, cap = static_cast<int64_t>(sm_count) * per_sm;
  merge_rows_kernel<G, U, kNarrow><<<static_cast<unsigned>(need < cap ? need : cap), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_merge_rows(const MergeRowsParams& p, int head_dim, int sm_count, cudaStream_t stream) {
  if (p.rows >= (1ll << 31)) return cudaErrorInvalidValue;
  if (head_dim == 64) return launch_cfg<4, 1, 4>(p, sm_count, stream);
  return launch_cfg<8, 1, 4>(p, sm_count, stream);
}

}  // namespace dtb
