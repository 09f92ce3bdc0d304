// Merge of partial softmax-attention states of which some are held in 8 bits, and states written in 8 bits, in one pass.
//
//   out = sum_i w_i v_i,  w_i = exp(lse_i - lse),  lse = log sum_i exp(lse_i)
//   in 8 bits  v = code * 2^(b - 127):  b is the smallest exponent byte (at least 8) with max|v| <= M 2^(b - 127), M the largest
//              code (127 of int8, 448 of e4m3), code = v 2^(127 - b) rounded to nearest, ties to even
// A row is one (token, head) pair and has one b.  A power of two, and not max|v| / M: then v 2^(127 - b) is exact, so that the
// code's rounding is the only one, the value it stands for is a bf16 number (at most 7 bits behind the leading one), and the
// factor is one byte and goes into the weight.  It costs int8 up to one bit of its 7, and e4m3 (a floating type) nothing.
// A row with an infinity or a NaN gets b = 255: its codes are 0, and 0 * 2^128 reads back as NaN.
// With one state and no lse the weight is 1: that writes a state in 8 bits, or reads it back.
//
// Bound by HBM.  D / 16 lanes own a row, 16 values each: 16 bytes of a state in 8 bits.  The 8-bit states come first in the
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
__device__ __forceinline__ void add_codes(float (&acc)[16], float w, uint4 v, int dtype) {
  const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
    if (dtype == kRowsI8) {
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = static_cast<float>(static_cast<int8_t>(a[i] >> (8 * k)));
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(a[i] >> (16 * k)), __NV_E4M3);
        const float2 x = __half22float2(h);
        f[2 * k] = x.x;
        f[2 * k + 1] = x.y;
      }
    }
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
__device__ __forceinline__ uint4 encode(const float (&acc)[16], uint32_t b, int dtype) {
  if (b == 255u) return make_uint4(0u, 0u, 0u, 0u);
  const float f = __uint_as_float((254u - b) << 23);
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x0 = acc[4 * i] * f, x1 = acc[4 * i + 1] * f, x2 = acc[4 * i + 2] * f, x3 = acc[4 * i + 3] * f;
    if (dtype == kRowsI8) {
      r[i] = (static_cast<uint32_t>(__float2int_rn(x0)) & 0xffu) | (static_cast<uint32_t>(__float2int_rn(x1)) & 0xffu) << 8 |
             (static_cast<uint32_t>(__float2int_rn(x2)) & 0xffu) << 16 | static_cast<uint32_t>(__float2int_rn(x3)) << 24;
    } else {
      r[i] = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3)) |
             static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x2, x3), __NV_SATFINITE, __NV_E4M3)) << 16;
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

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
    if (p.lse[0] != nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < kPerLane; ++t) {
          const int st = lane + t * G;
          w[u][t] = -INFINITY;
          if (row_of(u) < p.rows && st < n)
            w[u][t] = p.lse[st][lse_offset(p.lse_layout[st], static_cast<uint32_t>(row_of(u)), p.H, p.S)];
        }
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
      if (p.lse[0] == nullptr) {
        lse_out[u] = 0.f;
#pragma unroll
        for (int t = 0; t < kPerLane; ++t) w[u][t] = 1.f;
      } else {
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
      }
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
          st_stream(p.out_codes + off, encode(acc[u], b, p.out_codes_dtype));
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
