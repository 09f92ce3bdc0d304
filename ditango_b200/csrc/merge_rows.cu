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
// parameters.  All sums are fp32.
#include "merge_rows.cuh"

#include "flash_common.cuh"
#include "row_access.cuh"

#include <cuda_fp8.h>
#include <math.h>

namespace dtb {

namespace {

using namespace flash;               // packed fp32 pairs

constexpr int kThreads = 128;
constexpr int kMinExponent = 8;      // 2^(127 - b) stays finite; below 2^-111 of a row's maximum nothing is lost that matters

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 2^(b - 127); 0 for b = 0, infinity for b = 255
__device__ __forceinline__ float power_of(uint32_t b) { return __uint_as_float(b << 23); }
// a b where a may be smaller than the smallest normal number (which a plain product counts as 0 under the compiler's fast arithmetic)
__device__ __forceinline__ float scaled(float a, float b) {
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(b));
  return a;
}

// The values of a lane are eight pairs of fp32.
// 16 values of a wide state as loaded: fp32 in all four, bf16 in the first two.
struct Wide {
  uint4 q[4];
};
// Codes and exponents, which no result may take the place of, are read as memory that nobody writes meanwhile; wide values and lse,
// whose place a result may take, by ordinary loads (plain ones, which the compiler issues in front of the codes' arithmetic: a load
// that it may not move took a call on one int8 and one fp32 state of 14882 x 24 x 128 from 84 to 94 us).
__device__ __forceinline__ uint4 load_codes16(const void* p) { return __ldg(static_cast<const uint4*>(p)); }
__device__ __forceinline__ void load_wide(Wide& w, const void* values, int dtype, int64_t off) {
  if (dtype == kRowsF32) {
    const float* src = static_cast<const float*>(values) + off;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.q[i] = *reinterpret_cast<const uint4*>(src + 4 * i);
  } else {
    const uint16_t* src = static_cast<const uint16_t*>(values) + off;
    w.q[0] = *reinterpret_cast<const uint4*>(src);
    w.q[1] = *reinterpret_cast<const uint4*>(src + 8);
  }
}
// The values of a lane are eight pairs of fp32.
__device__ __forceinline__ void add_wide(uint64_t (&acc)[8], float w, const Wide& v, int dtype) {
  const uint64_t w2 = pack2(w, w);
  if (dtype == kRowsF32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[2 * i] = fma2(w2, pack2(__uint_as_float(v.q[i].x), __uint_as_float(v.q[i].y)), acc[2 * i]);
      acc[2 * i + 1] = fma2(w2, pack2(__uint_as_float(v.q[i].z), __uint_as_float(v.q[i].w)), acc[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a[4] = {v.q[i].x, v.q[i].y, v.q[i].z, v.q[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        acc[4 * i + k] = fma2(w2, pack2(__uint_as_float(a[k] << 16), __uint_as_float(a[k] & 0xffff0000u)), acc[4 * i + k]);
    }
  }
}
// The four codes of a word as two pairs of floats.  Whole numbers of 8 bits are placed in the low bits of 2^23, which is then taken
// off: the conversion unit has a quarter of the rate of that.
template <bool kWhole>
__device__ __forceinline__ void decode4(uint32_t a, uint64_t& lo, uint64_t& hi) {
  if (kWhole) {
    a ^= 0x80808080u;                 // code + 128
    const uint64_t off = pack2(-8388736.f, -8388736.f);
    lo = add2(pack2(__uint_as_float(__byte_perm(a, 0x4b000000u, 0x7540)), __uint_as_float(__byte_perm(a, 0x4b000000u, 0x7541))), off);
    hi = add2(pack2(__uint_as_float(__byte_perm(a, 0x4b000000u, 0x7542)), __uint_as_float(__byte_perm(a, 0x4b000000u, 0x7543))), off);
  } else {
    const float2 x = __half22float2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(a), __NV_E4M3));
    const float2 y = __half22float2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(a >> 16), __NV_E4M3));
    lo = pack2(x.x, x.y);
    hi = pack2(y.x, y.y);
  }
}
template <bool kWhole>
__device__ __forceinline__ void add_codes(uint64_t (&acc)[8], float w, uint4 v) {
  const uint32_t a[4] = {v.x, v.y, v.z, v.w};
  const uint64_t w2 = pack2(w, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint64_t lo, hi;
    decode4<kWhole>(a[i], lo, hi);
    acc[2 * i] = fma2(w2, lo, acc[2 * i]);
    acc[2 * i + 1] = fma2(w2, hi, acc[2 * i + 1]);
  }
}

// The larger magnitude, a NaN above all.
__device__ __forceinline__ float larger(float a, float b) {
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(fabsf(a)), "f"(fabsf(b)));
  return a;
}

// The exponent byte of a row whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t exponent_byte(uint32_t top, int dtype) {
  if (top >= 0x7f800000u) return 255u;
  // round the exponent up where the mantissa is above that of the largest code: 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
  const int b = dtype == kRowsI8 ? static_cast<int>((top + (0x7fffffu - 0x7e0000u)) >> 23) - 6
                                 : static_cast<int>((top + (0x7fffffu - 0x600000u)) >> 23) - 8;
  return static_cast<uint32_t>(b < kMinExponent ? kMinExponent : b);
}
// Four values as codes of a row with exponent byte b; f = 2^(127 - b).  (x f is exact, so that adding 1.5 * 2^23 is what rounds it.)
template <bool kWholeCodes>
__device__ __forceinline__ uint32_t encode4(float x0, float x1, float x2, float x3, float f) {
  if (kWholeCodes) {
    constexpr float kWhole = 12582912.f;
    const uint32_t t0 = __float_as_uint(fmaf(x0, f, kWhole)), t1 = __float_as_uint(fmaf(x1, f, kWhole));
    const uint32_t t2 = __float_as_uint(fmaf(x2, f, kWhole)), t3 = __float_as_uint(fmaf(x3, f, kWhole));
    return __byte_perm(__byte_perm(t0, t1, 0x0040), __byte_perm(t2, t3, 0x0040), 0x5410);
  }
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(scaled(x0, f), scaled(x1, f)), __NV_SATFINITE, __NV_E4M3)) |
         static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(scaled(x2, f), scaled(x3, f)), __NV_SATFINITE, __NV_E4M3)) << 16;
}
__device__ __forceinline__ float inverse_of(uint32_t b) { return __uint_as_float((254u - b) << 23); }

}  // namespace

// A CTA takes kTile rows.  First a thread has a row and forms its weights (and lse), then G = D / 16 lanes have a row and sum its values,
// kThreads / G rows at a time.  (Weights formed by the lanes of a row, each the same ones, took half of all instructions.)
// Measured, us and TB/s: four int8 blocks of 2 x 2222 x 48 x 64 into one 21.5 (3.4; 30.0 with weights formed by the lanes), of
// 14882 x 24 x 128 54 (4.4; 80); seven e4m3 blocks and a fresh fp32 state of 14882 x 24 x 128 into bf16 108 (5.6; 107), one of each into
// fp32 78 (5.3; 83).  More codes in flight (eight states' 27 and 65 us, 118 for seven and one) cost more by the registers they
// take; copied ahead through shared memory 24 and 70, 110, 97.  The first is bound by instructions: some 300 for 16 values of four blocks.
constexpr int kTile = kThreads;

template <int G>
__global__ void __launch_bounds__(kThreads) merge_rows_kernel(const __grid_constant__ MergeRowsParams p) {
  constexpr int D = G * 16, kNarrow = 4, kRows = kThreads / G;
  __shared__ float s_w[kMergeRowsMaxStates][kTile];
  const int n = p.nstates, n8 = p.narrow;
  const int64_t tile = static_cast<int64_t>(blockIdx.x) * kTile;
  const int lane = threadIdx.x % G;
  uint4 code[kNarrow];
  Wide wide;
  auto load_codes = [&](int c0, int64_t row) {
#pragma unroll
    for (int k = 0; k < kNarrow; ++k)
      if (c0 + k < n8 && row < p.rows) code[k] = load_codes16(static_cast<const uint8_t*>(p.values[c0 + k]) + row * D + lane * 16);
  };
  // (under way while the weights are formed)
  load_codes(0, tile + threadIdx.x / G);
  {
    const int64_t row = tile + threadIdx.x;
    if (row < p.rows) {
      // (eight states' loads are under way together)
      float mx = -INFINITY, sum = 0.f;
      for (int c = 0; c < n; c += 8) {
        float l[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          l[k] = c + k < n ? p.lse[c + k][lse_offset(p.lse_layout[c + k], static_cast<uint32_t>(row), p.H, p.S)] : -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (c + k < n) s_w[c + k][threadIdx.x] = l[k];
          mx = fmaxf(mx, l[k]);
        }
      }
      for (int st = 0; st < n; ++st) {
        const float l = s_w[st][threadIdx.x];
        sum += l == -INFINITY ? 0.f : ex2((l - mx) * 1.4426950408889634f);
      }
      // the factor of a state in 8 bits goes into its weight; a weight of 0 stays one
      const float scale = sum == 0.f ? 0.f : __fdividef(1.f, sum);       // (a NaN among the lse goes on into the result)
      for (int c = 0; c < n; c += 8) {
        uint32_t b[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) b[k] = c + k < n8 ? __ldg(p.exponents[c + k] + row) : 127u;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < n) {
            const float l = s_w[c + k][threadIdx.x];
            const float w = l == -INFINITY ? 0.f : ex2((l - mx) * 1.4426950408889634f) * scale;
            s_w[c + k][threadIdx.x] = w == 0.f ? 0.f : w * power_of(b[k]);        // (power_of may be infinite)
          }
      }
      if (p.lse_out != nullptr)
        p.lse_out[lse_offset(p.lse_out_layout, static_cast<uint32_t>(row), p.H, p.S)] = sum == 0.f ? -INFINITY : mx + logf(sum);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int r = threadIdx.x / G; r < kTile; r += kRows) {
    const int64_t row = tile + r;
    const int64_t off = row * D + lane * 16;
    const bool live = row < p.rows;
    uint64_t sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = pack2(0.f, 0.f);
    for (int c0 = 0; c0 < n8; c0 += kNarrow) {
#pragma unroll
      for (int k = 0; k < kNarrow; ++k)
        if (c0 + k < n8) {
          const float w = s_w[c0 + k][r];
          // a state of weight 0 may hold anything, a NaN too: it must not reach the sum
          if (live && w != 0.f) {
            if (p.dtype[c0 + k] == kRowsI8) add_codes<true>(sum, w, code[k]);
            else add_codes<false>(sum, w, code[k]);
          }
        }
      if (c0 + kNarrow < n8) load_codes(c0 + kNarrow, row);
    }
    load_codes(0, row + kRows);
    if (n8 < n && live) load_wide(wide, p.values[n8], p.dtype[n8], off);
    for (int st = n8; st < n; ++st) {
      const float w = s_w[st][r];
      if (live && w != 0.f) add_wide(sum, w, wide, p.dtype[st]);
      if (st + 1 < n && live) load_wide(wide, p.values[st + 1], p.dtype[st + 1], off);
    }

    float acc[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) unpack2(sum[i], acc[2 * i], acc[2 * i + 1]);
    if (p.out_codes != nullptr) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = larger(top, acc[i]);
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) top = larger(top, __shfl_xor_sync(0xffffffffu, top, o, G));
      const uint32_t b = exponent_byte(__float_as_uint(top), p.out_codes_dtype);
      if (live) {
        const float f = inverse_of(b);
        uint32_t q[4];
        if (p.out_codes_dtype == kRowsI8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = encode4<true>(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3], f);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = encode4<false>(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3], f);
        }
        if (b == 255u) q[0] = q[1] = q[2] = q[3] = 0u;
        st_stream(p.out_codes + off, make_uint4(q[0], q[1], q[2], q[3]));
        if (lane == 0) p.out_exponents[row] = static_cast<uint8_t>(b);
      }
    }
    if (live) {
      if (p.out != nullptr) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          st_stream(p.out + off + i, make_uint4(__float_as_uint(acc[i]), __float_as_uint(acc[i + 1]), __float_as_uint(acc[i + 2]), __float_as_uint(acc[i + 3])));
      }
      if (p.out_bf16 != nullptr) {
#pragma unroll
        for (int i = 0; i < 16; i += 8)
          st_stream(p.out_bf16 + off + i, make_uint4(pack_bf16(acc[i], acc[i + 1]), pack_bf16(acc[i + 2], acc[i + 3]),
                                                     pack_bf16(acc[i + 4], acc[i + 5]), pack_bf16(acc[i + 6], acc[i + 7])));
      }
    }
  }
}

// A single state written in 8 bits: D / 8 lanes to a row, 8 values each, kRowsPerThread rows whose loads are in flight together.  (The
// two halves of an fp32 row are accessed one after the other, four values a lane, so that each access is to whole lines: read back to
// fp32, 14882 x 24 x 128, 50 -> 36 us.)  Measured there: written from fp32 35 us (6.5 TB/s), from bf16 24 (5.7), read back to bf16 23 (6.1).
constexpr int kCodeThreads = 256;
constexpr int kRowsPerThread = 2;

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
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = larger(top, x[i]);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) top = larger(top, __shfl_xor_sync(0xffffffffu, top, o, G));
    const uint32_t b = exponent_byte(__float_as_uint(top), codes_dtype);
    const float f = inverse_of(b);
    uint32_t r0 = 0u, r1 = 0u;
    if (codes_dtype == kRowsI8) {
      r0 = encode4<true>(x[0], x[1], x[2], x[3], f);
      r1 = encode4<true>(x[4], x[5], x[6], x[7], f);
    } else {
      r0 = encode4<false>(x[0], x[1], x[2], x[3], f);
      r1 = encode4<false>(x[4], x[5], x[6], x[7], f);
    }
    if (b == 255u) r0 = r1 = 0u;
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
  constexpr bool f32 = sizeof(T) == 4;
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
      const uint8_t* src = codes + row * D + lane * (f32 ? 4 : 8);
      raw[u] = f32 ? make_uint2(*reinterpret_cast<const uint32_t*>(src), *reinterpret_cast<const uint32_t*>(src + D / 2))
                   : *reinterpret_cast<const uint2*>(src);
      b[u] = exponents[row];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = row0 + u * (kCodeThreads / G);
    if (row >= rows) break;
    const float f = power_of(b[u]);
    uint64_t v[4];
    if (codes_dtype == kRowsI8) {
      decode4<true>(raw[u].x, v[0], v[1]);
      decode4<true>(raw[u].y, v[2], v[3]);
    } else {
      decode4<false>(raw[u].x, v[0], v[1]);
      decode4<false>(raw[u].y, v[2], v[3]);
    }
    float x[4], y[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unpack2(mul2(v[i], pack2(f, f)), x[2 * i], x[2 * i + 1]);
      unpack2(mul2(v[2 + i], pack2(f, f)), y[2 * i], y[2 * i + 1]);
    }
    if (f32) {
      float* dst = reinterpret_cast<float*>(out) + row * D + lane * 4;
      *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(dst + D / 2) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
      *reinterpret_cast<uint4*>(out + row * D + lane * 8) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
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

cudaError_t launch_merge_rows(const MergeRowsParams& p, int head_dim, int sm_count, cudaStream_t stream) {
  if (p.rows >= (1ll << 31)) return cudaErrorInvalidValue;
  const unsigned tiles = static_cast<unsigned>((p.rows + kTile - 1) / kTile);
  if (head_dim == 64) merge_rows_kernel<4><<<tiles, kThreads, 0, stream>>>(p);
  else merge_rows_kernel<8><<<tiles, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace dtb
