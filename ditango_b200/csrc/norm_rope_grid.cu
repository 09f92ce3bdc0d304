// Norm of each head of the query and key projections, then rotary positions on three axes (time, height, width): one pass forward,
// one pass backward.
//
//   forward    y = (x - mean) rstd w + b     (RMS: y = x rstd w + b),      z = R y of the tokens that have a place in the grid
//   backward   dy = R^T dz,  g = dy w,  dx = rstd (g - mean(g) - x^ mean(g x^))   (RMS: without mean(g)),  x^ = (x - mean) rstd
//              dw = sum over rows of dy x^,  db = sum of dy
//   R turns channels (2 i, 2 i + 1) by the angle  (origin + step * index on pair i's axis) * base^(-2 i' / d)
// The angles come from the token's place in the grid and not from tables: in turns, product and reduction to [-1/2, 1/2] in 64 bits
// (far positions keep their precision), cosine and sine of what is left in 32.
//
// Bound by HBM: each value read once and written once.  D / 8 lanes own a head's row, 8 values each, so that pairs lie inside a lane
// and the means are shuffles inside the row's lanes.  A CTA's rows of lanes are dealt to the heads of one token, and to several tokens
// where there are fewer heads; a lane's four angles are formed once for all heads it takes.  All arithmetic is fp32, rounded once.
// The sums for the weights stay in a lane's registers over all its rows, are added up in the CTA and then over CTAs, in a fixed order.
#include "norm_rope_grid.cuh"

#include "ptx_sm100.cuh"

namespace dtb {

namespace {

constexpr int kThreads = 128;
constexpr int kBackwardPerSm = 4;       // CTAs of the backward pass per SM and tensor (what the scratch is sized for)

template <typename T>
struct Raw8;
template <>
struct Raw8<uint16_t> {
  uint4 a;
};
template <>
struct Raw8<float> {
  uint4 a, b;
};
__device__ __forceinline__ void load8(Raw8<uint16_t>& r, const uint16_t* p) { r.a = __ldcs(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ void load8(Raw8<float>& r, const float* p) {
  r.a = __ldcs(reinterpret_cast<const uint4*>(p));
  r.b = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
}
__device__ __forceinline__ void unpack8(const Raw8<uint16_t>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&x)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store1(uint16_t* p, float x) { *p = static_cast<uint16_t>(pack_bf16x2(x, 0.f)); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, kLanes);
  return v;
}

// x becomes x^ = (x - mean) rstd; returns rstd.
template <int D, bool kRms>
__device__ __forceinline__ float standardise(float (&x)[8], float eps) {
  constexpr int kLanes = D / 8;
  if (!kRms) {
    const float mean = row_sum<kLanes>(((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]))) * (1.f / D);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] -= mean;
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sq = fmaf(x[i], x[i], sq);
  const float rstd = rsqrtf(row_sum<kLanes>(sq) * (1.f / D) + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= rstd;
  return rstd;
}

// What happens to a token behind the norm.
enum Place { kText, kTurned, kPadding };

// Frequencies and axes of a lane's four pairs, and the angles of a token.
struct Pairs {
  double turns[4];
  int axis[4];
  __device__ __forceinline__ void load(const NormRopeGridParams& p, int col) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      turns[i] = p.turns[col / 2 + i];
      axis[i] = p.axis[col / 2 + i];
    }
  }
  __device__ __forceinline__ Place place(const NormRopeGridParams& p, int64_t tok, float (&cs)[4], float (&sn)[4]) const {
    const int s = static_cast<int>(tok % p.seq) - p.text_len;
    if (s < 0 || s >= p.video_len) return kText;
    const int64_t n = p.first + s;
    if (n >= static_cast<int64_t>(p.shards) * p.shard_len) return kPadding;
    const uint32_t shard = static_cast<uint32_t>(n) / static_cast<uint32_t>(p.shard_len), in = static_cast<uint32_t>(n) - shard * p.shard_len;
    const uint32_t rest = static_cast<uint32_t>(p.shard_rest);
    if (in >= p.shard_places + (shard < rest ? 1u : 0u)) return kPadding;
    const uint32_t at = shard * p.shard_places + min(shard, rest) + in, row = at / static_cast<uint32_t>(p.size_x);
    const uint32_t t = row / static_cast<uint32_t>(p.size_y);
    const double pos[3] = {p.origin[0] + p.step[0] * t, p.origin[1] + p.step[1] * (row - t * p.size_y),
                           p.origin[2] + p.step[2] * (at - row * p.size_x)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double turn = (axis[i] == 0 ? pos[0] : axis[i] == 1 ? pos[1] : pos[2]) * turns[i];
      sincospif(2.f * static_cast<float>(turn - rint(turn)), &sn[i], &cs[i]);
    }
    return kTurned;
  }
};

// How a CTA's rows of lanes are dealt: `width` of them (a power of two) to a token's heads.
template <int D>
struct Deal {
  static constexpr int kLanes = D / 8;
  static constexpr int kRowsOfLanes = kThreads / kLanes;
  int width, tokens, head0, sub;
  __device__ __forceinline__ explicit Deal(int heads) {
    width = 1;
    while (width < kRowsOfLanes && width < heads) width *= 2;
    tokens = kRowsOfLanes / width;
    const int row = threadIdx.x / kLanes;
    head0 = row % width;
    sub = row / width;
  }
};

}  // namespace

template <typename T, int D, bool kRms>
__global__ void __launch_bounds__(kThreads) norm_rope_grid_kernel(const __grid_constant__ NormRopeGridParams p) {
  constexpr int kLanes = D / 8;
  constexpr int U = 3;                    // heads of each tensor whose loads are in flight together
  const int col = (threadIdx.x % kLanes) * 8;
  const Deal<D> deal(max(p.heads[0], p.heads[1]));
  Pairs pairs;
  pairs.load(p, col);
  float w[2][8], b[2][8];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    Raw8<T> r;
    load8(r, static_cast<const T*>(p.weight[x]) + col);
    unpack8(r, w[x]);
#pragma unroll
    for (int i = 0; i < 8; ++i) b[x][i] = 0.f;
    if (p.bias[x] != nullptr) {
      load8(r, static_cast<const T*>(p.bias[x]) + col);
      unpack8(r, b[x]);
    }
  }
  const int most = max(p.heads[0], p.heads[1]);
  // (the bound is the same for all lanes of a warp: the shuffles use the full mask)
  for (int64_t tok0 = static_cast<int64_t>(blockIdx.x) * deal.tokens; tok0 < p.tokens; tok0 += static_cast<int64_t>(gridDim.x) * deal.tokens) {
    const int64_t tok = tok0 + deal.sub;
    const bool live = tok < p.tokens;
    const int64_t seq_no = tok / p.seq, s = tok - seq_no * p.seq;
    float cs[4], sn[4];
    Place place = kText;
    bool placed = false;
    for (int h0 = 0; h0 < most; h0 += U * deal.width) {
      Raw8<T> raw[2][U];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * deal.width + deal.head0;
          raw[x][u] = Raw8<T>{};
          if (live && h < p.heads[x])
            load8(raw[x][u], static_cast<const T*>(p.src[x]) + seq_no * p.batch_stride[x] + s * p.tok_stride[x] + static_cast<int64_t>(h) * D + col);
        }
      if (!placed) {                       // under the loads
        if (live) place = pairs.place(p, tok, cs, sn);
        placed = true;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * deal.width + deal.head0;
          float v[8];
          unpack8(raw[x][u], v);
          standardise<D, kRms>(v, p.eps[x]);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], w[x][i], b[x][i]);
          if (place == kTurned) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float re = v[2 * i], im = v[2 * i + 1];
              v[2 * i] = re * cs[i] - im * sn[i];
              v[2 * i + 1] = im * cs[i] + re * sn[i];
            }
          } else if (place == kPadding) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
          }
          if (live && h < p.heads[x]) store8(static_cast<T*>(p.dst[x]) + (tok * p.heads[x] + h) * D + col, v);
        }
    }
  }
}

// grid: (CTAs, tensor)
template <typename T, int D, bool kRms>
__global__ void __launch_bounds__(kThreads) norm_rope_grid_backward_kernel(const __grid_constant__ NormRopeGridParams p) {
  constexpr int kLanes = D / 8;
  constexpr int U = 2;
  __shared__ float s_sum[kThreads / kLanes][2 * D];
  const int x = blockIdx.y;
  const int heads = p.heads[x];
  const int col = (threadIdx.x % kLanes) * 8;
  const Deal<D> deal(heads);
  Pairs pairs;
  pairs.load(p, col);
  float w[8], dw[8], db[8];
  {
    Raw8<T> r;
    load8(r, static_cast<const T*>(p.weight[x]) + col);
    unpack8(r, w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = db[i] = 0.f;
  const float eps = p.eps[x];
  const T* src = static_cast<const T*>(p.src[x]) + col;
  const T* grad = static_cast<const T*>(p.grad[x]) + col;
  T* dst = static_cast<T*>(p.dst[x]) + col;
  for (int64_t tok0 = static_cast<int64_t>(blockIdx.x) * deal.tokens; tok0 < p.tokens; tok0 += static_cast<int64_t>(gridDim.x) * deal.tokens) {
    const int64_t tok = tok0 + deal.sub;
    const bool live = tok < p.tokens;
    const int64_t seq_no = tok / p.seq, s = tok - seq_no * p.seq;
    float cs[4], sn[4];
    Place place = kText;
    bool placed = false;
    for (int h0 = 0; h0 < heads; h0 += U * deal.width) {
      Raw8<T> rx[U], rg[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * deal.width + deal.head0;
        rx[u] = rg[u] = Raw8<T>{};
        if (live && h < heads) {
          load8(rx[u], src + seq_no * p.batch_stride[x] + s * p.tok_stride[x] + static_cast<int64_t>(h) * D);
          load8(rg[u], grad + seq_no * p.grad_batch_stride[x] + s * p.grad_tok_stride[x] + static_cast<int64_t>(h) * D);
        }
      }
      if (!placed) {
        if (live) place = pairs.place(p, tok, cs, sn);
        placed = true;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * deal.width + deal.head0;
        float v[8], g[8];
        unpack8(rx[u], v);
        unpack8(rg[u], g);
        if (place == kTurned) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float re = g[2 * i], im = g[2 * i + 1];
            g[2 * i] = re * cs[i] + im * sn[i];
            g[2 * i + 1] = im * cs[i] - re * sn[i];
          }
        } else if (place == kPadding) {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = 0.f;
        }
        const float rstd = standardise<D, kRms>(v, eps);
        float sum_g = 0.f, sum_gx = 0.f;
        const bool counts = live && h < heads && place != kPadding;      // (a row that is cut off may hold anything)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (counts) {
            dw[i] = fmaf(g[i], v[i], dw[i]);
            db[i] += g[i];
          }
          g[i] *= w[i];
          sum_g += g[i];
          sum_gx = fmaf(g[i], v[i], sum_gx);
        }
        const float mean_gx = row_sum<kLanes>(sum_gx) * (1.f / D);
        const float mean_g = kRms ? 0.f : row_sum<kLanes>(sum_g) * (1.f / D);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = place == kPadding ? 0.f : rstd * ((g[i] - mean_g) - v[i] * mean_gx);
        if (live && h < heads) store8(dst + (tok * heads + h) * D, g);
      }
    }
  }
  const int row = threadIdx.x / kLanes;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s_sum[row][col + i] = dw[i];
    s_sum[row][D + col + i] = db[i];
  }
  __syncthreads();
  float* to = p.partial + (static_cast<int64_t>(x) * gridDim.x + blockIdx.x) * (2 * D);
  for (int c = threadIdx.x; c < 2 * D; c += kThreads) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < kThreads / kLanes; ++r) sum += s_sum[r][c];
    to[c] = sum;
  }
}

// Sums of the CTAs' rows.  grid: (2 D / 32, tensor); 32 columns, 32 threads to a column.
template <typename T, int D>
__global__ void __launch_bounds__(1024) norm_rope_grid_sums_kernel(const __grid_constant__ NormRopeGridParams p, int rows) {
  __shared__ float s_sum[32][33];
  grid_dependency_wait();
  const int x = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  const float* from = p.partial + static_cast<int64_t>(x) * rows * (2 * D) + c;
  float sum = 0.f;
#pragma unroll 4
  for (int r = slice; r < rows; r += 32) sum += from[static_cast<int64_t>(r) * (2 * D)];
  s_sum[threadIdx.x & 31][slice] = sum;
  __syncthreads();
  sum = s_sum[slice][threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) {
    const int at = blockIdx.x * 32 + slice;
    void* dst = at < D ? p.weight_grad[x] : p.bias_grad[x];
    if (dst != nullptr) store1(static_cast<T*>(dst) + (at < D ? at : at - D), sum);
  }
}

template <int D>
static int tokens_per_cta(int heads) {
  constexpr int rows = kThreads / (D / 8);
  int width = 1;
  while (width < rows && width < heads) width *= 2;
  return rows / width;
}

template <typename T, int D, bool kRms>
static cudaError_t launch_forward(const NormRopeGridParams& p, int sm_count, cudaStream_t stream) {
  const int per_cta = tokens_per_cta<D>(p.heads[0] > p.heads[1] ? p.heads[0] : p.heads[1]);
  const int64_t need = (p.tokens + per_cta - 1) / per_cta, cap = static_cast<int64_t>(sm_count) * 16;
  norm_rope_grid_kernel<T, D, kRms><<<static_cast<unsigned>(need < cap ? need : cap), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, int D, bool kRms>
static cudaError_t launch_backward(const NormRopeGridParams& p, int sm_count, cudaStream_t stream) {
  const int per_cta = tokens_per_cta<D>(p.heads[0] < p.heads[1] ? p.heads[0] : p.heads[1]);
  const int64_t need = (p.tokens + per_cta - 1) / per_cta, cap = static_cast<int64_t>(sm_count) * kBackwardPerSm;
  // (without tokens one CTA still writes its sums, which are 0)
  const int ctas = static_cast<int>(need < 1 ? 1 : need < cap ? need : cap);
  norm_rope_grid_backward_kernel<T, D, kRms><<<dim3(ctas, 2), kThreads, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  norm_rope_grid_sums_kernel<T, D><<<dim3(2 * D / 32, 2), 1024, 0, stream>>>(p, ctas);
  return cudaGetLastError();
}

cudaError_t launch_norm_rope_grid(const NormRopeGridParams& p, int head_dim, bool bf16, bool rms, int sm_count, cudaStream_t stream) {
  if (head_dim == 64) {
    if (bf16) return rms ? launch_forward<uint16_t, 64, true>(p, sm_count, stream) : launch_forward<uint16_t, 64, false>(p, sm_count, stream);
    return rms ? launch_forward<float, 64, true>(p, sm_count, stream) : launch_forward<float, 64, false>(p, sm_count, stream);
  }
  if (bf16) return rms ? launch_forward<uint16_t, 128, true>(p, sm_count, stream) : launch_forward<uint16_t, 128, false>(p, sm_count, stream);
  return rms ? launch_forward<float, 128, true>(p, sm_count, stream) : launch_forward<float, 128, false>(p, sm_count, stream);
}

int64_t norm_rope_grid_scratch_bytes(int head_dim, int sm_count) { return 2ll * sm_count * kBackwardPerSm * 2 * head_dim * 4; }

cudaError_t launch_norm_rope_grid_backward(const NormRopeGridParams& p, int head_dim, bool bf16, bool rms, int sm_count, cudaStream_t stream) {
  if (head_dim == 64) {
    if (bf16) return rms ? launch_backward<uint16_t, 64, true>(p, sm_count, stream) : launch_backward<uint16_t, 64, false>(p, sm_count, stream);
    return rms ? launch_backward<float, 64, true>(p, sm_count, stream) : launch_backward<float, 64, false>(p, sm_count, stream);
  }
  if (bf16) return rms ? launch_backward<uint16_t, 128, true>(p, sm_count, stream) : launch_backward<uint16_t, 128, false>(p, sm_count, stream);
  return rms ? launch_backward<float, 128, true>(p, sm_count, stream) : launch_backward<float, 128, false>(p, sm_count, stream);
}

}  // namespace dtb
