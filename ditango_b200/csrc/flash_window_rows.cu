// Windowed attention of few query rows: the keys of a row block are split over the warps of a cluster and joined there.
//
// A block of 16 rows, a row being a query and one of the query heads that share a key head, meets the keys that any of its rows sees:
// T = [0, first) and [lo, hi) put side by side.  Warp w of CTA c takes every (4 C)-th tile of 16 of them, through its own ring of
// stages in shared memory (cp.async, no barrier but the warp's own), and keeps a softmax state (m, l, O) of its rows:
//     S = Q K^T,  m' = max(m, max S),  P = 2^(c (S - m')),  l' = l 2^(c (m - m')) + sum P,  O' = O 2^(c (m - m')) + P V
// The states of the four warps are joined in shared memory, those of the cluster's CTAs through distributed shared memory, in a
// fixed order: one launch, no workspace, no atomics.
//
// Bound by HBM for few rows (a key and a value are read once per 16 rows); mma.sync, because 16 rows fill an instruction of it and a
// 128-row tile of tcgen05 would be empty for the most part.  P is rounded to bf16 for the product (by 2^-8 of each weight at
// most, as in the other attention kernels), sums and states are fp32.
// Measured, launches in a graph: a token of 24 heads of 128 against 4352 keys 13.8 us (53 MB, 3.9 TB/s), three tokens of seven sequences, 32
// over 8 heads of 64, against 3013 keys 12.6 us (43 MB, 3.4 TB/s).  With hardly any keys a launch takes 5 us; the rest is at the rate of HBM.
#include "flash_common.cuh"
#include "flash_window.cuh"

#include <cooperative_groups.h>

#include <mutex>

namespace dtb {

namespace {

using namespace flash;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;
constexpr int kKeys = 16;           // keys of a tile
constexpr int kStages = 3;
constexpr int kMostCtas = 8;        // of a cluster

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// d += a b: 16 x 16 (rows x k) by 16 x 8
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// The exponent's reference for a running maximum: 0 while no key has been seen, so that -inf - ref stays -inf.
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

template <int D>
struct Smem {
  static constexpr int kTileBytes = kKeys * D * 2;                    // of K or V
  static constexpr int kRing = kWarps * kStages * 2 * kTileBytes;
  static constexpr int kStates = kWarps * kRows * D * 4;              // O of the warps, over the ring
  static constexpr int kBytes = kRing + (kWarps + 1) * kRows * 8 + kRows * D * 4;     // + (m, l) of the warps and the CTA, O of the CTA
  static_assert(kStates <= kRing, "states take the ring's place");
};

}  // namespace

// grid: (row blocks x C, key heads, sequences); a cluster is the C CTAs of a row block.
template <int D>
__global__ void __launch_bounds__(kThreads) flash_window_rows_kernel(const WindowParams p) {
  namespace cg = cooperative_groups;
  using M = Smem<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  float2* s_ml = reinterpret_cast<float2*>(smem + M::kRing);          // [warp][row]
  float2* s_ml_cta = s_ml + kWarps * kRows;                           // [row]
  float* s_o_cta = reinterpret_cast<float*>(s_ml_cta + kRows);        // [row][D]
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seg = blockIdx.z, kv_head = blockIdx.y;
  const int group = p.f.num_heads / p.kv_heads;
  const WindowSeq s = window_seq(p, seg);
  const int rows = s.q_len * group, row0 = static_cast<int>(blockIdx.x) / C * kRows;       // (the launcher sees to it that they fit)
  if (row0 >= rows) return;                           // all CTAs of the cluster or none
  const int status = *reinterpret_cast<volatile int*>(p.f.status);
  const int n_rows = min(kRows, rows - row0);

  // what the block sees: the first row reaches furthest to the left, the last one to the right
  const WindowSpan w0 = window_span(s, row0 / group);
  const WindowSpan w1 = window_span(s, (row0 + n_rows - 1) / group);
  const int first = w1.first, lo = max(w0.lo, first);
  const int total = first + max(w1.hi - lo, 0);
  const int n_tiles = (total + kKeys - 1) / kKeys;

  // this thread's rows lane / 4 and lane / 4 + 8, counted in the keys put side by side: [0, end) and [from, to)
  int end[2], from[2], to[2];
  uint32_t qf[D / 16][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (lane >> 2) + 8 * h;
    end[h] = from[h] = to[h] = 0;
    const uint16_t* src = nullptr;
    if (r < n_rows) {
      const int i = (row0 + r) / group, g = (row0 + r) % group;
      const WindowSpan w = window_span(s, i);
      end[h] = w.first;
      from[h] = w.lo - lo + first;
      to[h] = w.hi - lo + first;
      src = p.q + window_offset(p, seg, static_cast<int64_t>(s.q_begin) + i, p.q_tok, p.q_batch) + static_cast<int64_t>(kv_head * group + g) * D;
    }
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        qf[k][h + 2 * half] = src != nullptr ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 * half + 2 * (lane & 3)) : 0u;
  }

  uint8_t* ring = smem + warp * (kStages * 2 * M::kTileBytes);
  const uint16_t* k_base = p.k + window_offset(p, seg, s.k_begin, p.k_tok, p.k_batch) + kv_head * D;
  const uint16_t* v_base = p.v + window_offset(p, seg, s.k_begin, p.v_tok, p.v_batch) + kv_head * D;
  constexpr int kPieces = D / 8;                      // 16-byte pieces of a row
  auto load = [&](int tile, int stage) {
    const uint32_t dst = smem_u32(ring + stage * 2 * M::kTileBytes);
#pragma unroll
    for (int x = 0; x < kKeys * kPieces / 32; ++x) {
      const int id = x * 32 + lane, row = id / kPieces, piece = id % kPieces;
      const int t = tile * kKeys + row;
      const bool valid = t < total;
      const int64_t j = !valid ? 0 : t < first ? t : lo + (t - first);
      const uint32_t at = dst + row * (D * 2) + ((piece ^ (row & 7)) << 4);
      cp_async16(at, k_base + j * p.k_tok + piece * 8, valid);
      cp_async16(at + M::kTileBytes, v_base + j * p.v_tok + piece * 8, valid);
    }
  };

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float c = p.f.scale_log2;
  const int tile0 = rank * kWarps + warp, step = C * kWarps;
  // (every step commits a group, an empty one past the last tile, so that the count of groups in flight is always known)
  for (int i = 0; i < kStages - 1; ++i) {
    if (tile0 + i * step < n_tiles) load(tile0 + i * step, i);
    cp_async_commit();
  }
  int stage = 0;
  for (int tile = tile0; tile < n_tiles; tile += step) {
    cp_async_wait<kStages - 2>();
    __syncwarp();                                     // ... and all lanes have read the tile before it, whose slot the next load takes
    const int ahead = tile + (kStages - 1) * step;
    const int slot = stage == 0 ? kStages - 1 : stage - 1;
    if (ahead < n_tiles) load(ahead, slot);
    cp_async_commit();
    const uint32_t ks = smem_u32(ring + stage * 2 * M::kTileBytes), vs = ks + M::kTileBytes;
    float sc[2][4] = {};
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t b[4];
      const int row = ((lane >> 4) << 3) + (lane & 7), piece = 2 * k + ((lane >> 3) & 1);
      ldmatrix4(ks + row * (D * 2) + ((piece ^ (row & 7)) << 4), b);
      mma16816(sc[0], qf[k], b[0], b[1]);
      mma16816(sc[1], qf[k], b[2], b[3]);
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int h = e >> 1, t = tile * kKeys + n * 8 + 2 * (lane & 3) + (e & 1);
        if (!(t < end[h] || (t >= from[h] && t < to[h]))) sc[n][e] = -INFINITY;
        mx[h] = fmaxf(mx[h], sc[n][e]);
      }
    float f[2], ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float mn = fmaxf(m[h], quad_max(mx[h]));
      ref[h] = reference(mn) * c;
      f[h] = ex2(m[h] * c - ref[h]);
      m[h] = mn;
      l[h] *= f[h];
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      o[i][0] *= f[0];
      o[i][1] *= f[0];
      o[i][2] *= f[1];
      o[i][3] *= f[1];
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[n][e] = ex2(fmaf(sc[n][e], c, -ref[e >> 1]));
        l[e >> 1] += sc[n][e];
      }
    const uint32_t a[4] = {pack_bf16x2(sc[0][0], sc[0][1]), pack_bf16x2(sc[0][2], sc[0][3]),
                           pack_bf16x2(sc[1][0], sc[1][1]), pack_bf16x2(sc[1][2], sc[1][3])};
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      uint32_t b[4];
      const int row = (((lane >> 3) & 1) << 3) + (lane & 7), piece = 2 * d + (lane >> 4);
      ldmatrix4_trans(vs + row * (D * 2) + ((piece ^ (row & 7)) << 4), b);
      mma16816(o[2 * d], a, b[0], b[1]);
      mma16816(o[2 * d + 1], a, b[2], b[3]);
    }
    if (++stage == kStages) stage = 0;
  }
  cp_async_wait<0>();
  __syncthreads();                                    // the ring's memory takes the states

  // join the warps
  float* s_o = reinterpret_cast<float*>(smem) + warp * kRows * D;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (lane >> 2) + 8 * h;
    const float sum = quad_sum(l[h]);
    if ((lane & 3) == 0) s_ml[warp * kRows + r] = make_float2(m[h], sum);
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<float2*>(s_o + r * D + 8 * i + 2 * (lane & 3)) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
  }
  __syncthreads();
  for (int u = threadIdx.x; u < n_rows * (D / 4); u += kThreads) {
    const int r = u / (D / 4), col = (u % (D / 4)) * 4;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_ml[w * kRows + r].x);
    const float ref = reference(mx);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = s_ml[w * kRows + r];
      const float f = ex2((ml.x - ref) * c);
      const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + (w * kRows + r) * D + col);
      sum = fmaf(ml.y, f, sum);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z);
      acc.w = fmaf(v.w, f, acc.w);
    }
    *reinterpret_cast<float4*>(s_o_cta + r * D + col) = acc;
    if (col == 0) s_ml_cta[r] = make_float2(mx, sum);
  }
  // ... and the CTAs: four columns of a row per thread, the rows' columns dealt out over the cluster
  cluster.sync();
  // after a failure elsewhere nothing is stored (a CTA that left instead would take its shared memory with it)
  const bool stores = status == 0;
  for (int u = rank * kThreads + threadIdx.x; u < n_rows * (D / 4); u += C * kThreads) {
    const int r = u / (D / 4), col = (u % (D / 4)) * 4;
    // (all reads of the other CTAs' memory are under way before one is used)
    float2 ml[kMostCtas];
    float4 v[kMostCtas];
#pragma unroll
    for (int b = 0; b < kMostCtas; ++b) {
      ml[b] = make_float2(-INFINITY, 0.f);
      v[b] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (b < C) {
        ml[b] = cluster.map_shared_rank(s_ml_cta, b)[r];
        v[b] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(s_o_cta, b) + r * D + col);
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < kMostCtas; ++b) mx = fmaxf(mx, ml[b].x);
    const float ref = reference(mx);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int b = 0; b < kMostCtas; ++b) {
      const float f = ex2((ml[b].x - ref) * c);
      sum = fmaf(ml[b].y, f, sum);
      acc.x = fmaf(v[b].x, f, acc.x);
      acc.y = fmaf(v[b].y, f, acc.y);
      acc.z = fmaf(v[b].z, f, acc.z);
      acc.w = fmaf(v[b].w, f, acc.w);
    }
    const int i = (row0 + r) / group, head = kv_head * group + (row0 + r) % group;
    const int64_t tok = p.f.cu_q != nullptr ? static_cast<int64_t>(s.q_begin) + i : static_cast<int64_t>(seg) * p.f.seqlen_q + i;
    const int64_t li = lse_index(p.f, seg, head, i, tok), oi = tok * p.f.out_tok_stride + static_cast<int64_t>(head) * D + col;
    const bool empty = sum == 0.f;                    // no key seen: nothing to write over a state  (a NaN among the scores is not empty)
    if (stores && !(empty && p.f.accumulate != 0)) {
      const float lse = empty ? -INFINITY : (mx * c + log2f(sum)) * kLn2;
      float w_new = 0.f, w_old = 0.f, lse_out = lse;
      if (!empty) merge_weights(p.f.accumulate != 0, p.f.accumulate ? p.f.lse[li] : -INFINITY, lse, sum, w_new, w_old, lse_out);
      acc.x *= w_new;
      acc.y *= w_new;
      acc.z *= w_new;
      acc.w *= w_new;
      if (p.f.out_dtype == 0) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.f.out) + oi);
        if (w_old != 0.f) {
          const float4 old = *dst;
          acc.x = fmaf(old.x, w_old, acc.x);
          acc.y = fmaf(old.y, w_old, acc.y);
          acc.z = fmaf(old.z, w_old, acc.z);
          acc.w = fmaf(old.w, w_old, acc.w);
        }
        *dst = acc;
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.f.out) + oi) = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
      }
      // the threads of a row, D / 4 lanes of one warp, have read its lse before one of them writes it
      __syncwarp(D == 128 ? 0xffffffffu : 0xffffu << (lane & 16));
      if (col == 0) p.f.lse[li] = lse_out;
    }
  }
  cluster.sync();                                     // nobody leaves while its shared memory is read
}

template <int D>
cudaError_t launch_window_rows(const WindowParams& p, int sm_count, cudaStream_t stream) {
  using M = Smem<D>;
  static bool configured[64] = {};
  static std::mutex mu;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!configured[dev & 63]) {
      e = cudaFuncSetAttribute(flash_window_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, M::kBytes);
      if (e != cudaSuccess) return e;
      configured[dev & 63] = true;
    }
  }
  const int group = p.f.num_heads / p.kv_heads;
  const int64_t row_blocks = (static_cast<int64_t>(p.f.seqlen_q) * group + kRows - 1) / kRows;
  const int64_t blocks = row_blocks * p.kv_heads * p.f.nseg;
  // as many CTAs to a row block as give every SM one, each with two tiles for every warp (56 blocks of 188 tiles at D = 64: 13.0 us
  // with 4, 14.0 with 8; 24 blocks of 272 tiles at D = 128, 8 CTAs either way: 14.5)
  int64_t span = static_cast<int64_t>(p.left) + p.right + p.sinks + kRows;
  if (p.left < 0 || p.right < 0 || span > p.f.seqlen_k) span = p.f.seqlen_k;
  const int64_t tiles = (span + kKeys - 1) / kKeys;
  int C = 1;
  while (C < kMostCtas && blocks * C < sm_count && tiles > 2 * kWarps * C) C *= 2;
  if ((row_blocks * C + 1) * kRows > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(row_blocks * C), p.kv_heads, p.f.nseg);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = M::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, flash_window_rows_kernel<D>, p);
}

template cudaError_t launch_window_rows<64>(const WindowParams&, int, cudaStream_t);
template cudaError_t launch_window_rows<128>(const WindowParams&, int, cudaStream_t);

}  // namespace dtb
