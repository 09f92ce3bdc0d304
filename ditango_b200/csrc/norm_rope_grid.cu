// Norm of each head of the query and key projections, then rotary positions on three axes (time, height, width): one pass forward,
// one pass backward.
//
//   forward    y = (x - mean) rstd w + b     (RMS: y = x rstd w + b),      z = R y of the tokens that have a place in the grid
//   backward   dy = R^T dz,  g = dy w,  dx = rstd (g - mean(g) - x^ mean(g x^))   (RMS: without mean(g)),  x^ = (x - mean) rstd
//              dw = sum over rows of dy x^,  db = sum of dy
//   R turns channels (2 i, 2 i + 1) by the angle  (origin + step * index on pair i's axis) * base^(-2 i' / d)
// The angles come from the token's place in the grid and not from tables: in turns, product and reduction to [-1/2, 1/2] in 64 bits
// (far positions keep their precision), cosine and sine of what is left in 32.  A CTA forms those of a few tokens at a time, one per
// thread, in shared memory.
//
// Bound by HBM: each value read once and written once.  D / 8 lanes own a head's row, 8 values each, so that pairs lie inside a lane
// and the means are shuffles inside the row's lanes.  A CTA's rows of lanes are dealt to the heads of one token, and to several tokens
// where there are fewer heads.  All arithmetic is fp32, rounded once.
// Measured: forward, 2 x 17776 x 48 x 64 bf16, layer norm, 148 us (874 MB, 5.9 TB/s); backward, 32681 x 24 x 128 bf16, RMS norm, 202 us
// (1205 MB, 5.96 TB/s).  The way there, us of the two:
//   every lane the four angles of its own pairs, a token's loads issued together      216 / 381
//   angles by the CTA, queries loaded while keys are worked on                        170 / 259
//   channel pairs in packed arithmetic, fixed distances between heads (a quarter fewer instructions)    171 / 243
//   loads by asynchronous copies into a ring, so that more warps fit                  147 / 213
//   a pair's rate formed by the thread that has its angles (it was read from a table among the parameters)     148 / 202
// The sums for the weights stay in a lane's registers over all its rows, are added up in the CTA and then over CTAs, in a fixed order.
#include "norm_rope_grid.cuh"

#include "flash_common.cuh"

namespace dtb {

namespace {

using namespace flash;              // packed fp32 pairs

constexpr int kThreads = 128;
constexpr int kBackwardPerSm = 3;       // CTAs of the backward pass per SM and tensor (what the scratch is sized for)

// Eight values as they lie in memory.
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
__device__ __forceinline__ void load8(Raw8<uint16_t>& r, const uint16_t* p) { r.a = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load8(Raw8<float>& r, const float* p) {
  r.a = *reinterpret_cast<const uint4*>(p);
  r.b = *(reinterpret_cast<const uint4*>(p) + 1);
}
// The same by an asynchronous copy into shared memory (kThreads pieces of 16 bytes apart); zeros where not `valid`.
__device__ __forceinline__ void copy16(uint4* to, const void* from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint4* to, const uint16_t* from, bool valid) { copy16(to, from, valid); }
__device__ __forceinline__ void copy8(uint4* to, const float* from, bool valid) {
  copy16(to, from, valid);
  copy16(to + kThreads, from + 4, valid);
}
__device__ __forceinline__ void read8(Raw8<uint16_t>& r, const uint4* from) { r.a = from[0]; }
__device__ __forceinline__ void read8(Raw8<float>& r, const uint4* from) {
  r.a = from[0];
  r.b = from[kThreads];
}

// Eight values are held as the four channel pairs that turn together, (re, im) in one 64-bit register pair: half the instructions
// for whatever treats both alike.
__device__ __forceinline__ void unpack8(const Raw8<uint16_t>& r, uint64_t (&x)[4]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, uint64_t (&x)[4]) {
  x[0] = pack2(__uint_as_float(r.a.x), __uint_as_float(r.a.y));
  x[1] = pack2(__uint_as_float(r.a.z), __uint_as_float(r.a.w));
  x[2] = pack2(__uint_as_float(r.b.x), __uint_as_float(r.b.y));
  x[3] = pack2(__uint_as_float(r.b.z), __uint_as_float(r.b.w));
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
__device__ __forceinline__ float sum_of(uint64_t v) {
  float a, b;
  unpack2(v, a, b);
  return a + b;
}

// x becomes x^ = (x - mean) rstd; returns rstd.
template <int D, bool kRms>
__device__ __forceinline__ float standardise(uint64_t (&x)[4], float eps) {
  constexpr int kLanes = D / 8;
  if (!kRms) {
    const float mean = row_sum<kLanes>(sum_of(add2(add2(x[0], x[1]), add2(x[2], x[3])))) * (1.f / D);
    const uint64_t shift = pack2(-mean, -mean);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = add2(x[i], shift);
  }
  const uint64_t sq = fma2(x[0], x[0], fma2(x[1], x[1], fma2(x[2], x[2], mul2(x[3], x[3]))));
  const float rstd = rsqrtf(row_sum<kLanes>(sum_of(sq)) * (1.f / D) + eps);
  const uint64_t scale = pack2(rstd, rstd);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], scale);
  return rstd;
}

__device__ __forceinline__ int axis_of(const NormRopeGridParams& p, int pair) { return pair < p.pairs_end[0] ? 0 : pair < p.pairs_end[1] ? 1 : 2; }
// Where pair `pair` stands at index 0 and what it moves by with the index, in turns.  (A power by squaring, off by 2^-52 of itself per
// pair in front of it on its axis, the less the faster the pair turns.  A table of all pairs among the parameters was read at another
// place by each thread and made a launch a microsecond longer.)
__device__ __forceinline__ double2 rate_of(const NormRopeGridParams& p, int pair) {
  const int a = axis_of(p, pair), i = pair - (a == 0 ? 0 : p.pairs_end[a - 1]);
  double rate = 0.15915494309189533577, power = p.ratio[a];       // 1 / 2 pi
#pragma unroll
  for (int bit = 1; bit < 64; bit *= 2) {
    if ((i & bit) != 0) rate *= power;
    power *= power;
  }
  return make_double2(p.origin[a] * rate, p.step[a] * rate);
}

// Angle of pair `pair` of token `tok` as (cos, sin): (1, 0) for text, (0, 0), which no angle has, for padding.
__device__ __forceinline__ float2 rotation(const NormRopeGridParams& p, double2 rate, int64_t tok, int pair) {
  const int s = static_cast<int>(tok % p.seq) - p.text_len;
  if (s < 0 || s >= p.video_len) return make_float2(1.f, 0.f);
  const int64_t n = p.first + s;
  if (n >= static_cast<int64_t>(p.shards) * p.shard_len) return make_float2(0.f, 0.f);
  const uint32_t shard = static_cast<uint32_t>(n) / static_cast<uint32_t>(p.shard_len), in = static_cast<uint32_t>(n) - shard * p.shard_len;
  const uint32_t rest = static_cast<uint32_t>(p.shard_rest);
  if (in >= p.shard_places + (shard < rest ? 1u : 0u)) return make_float2(0.f, 0.f);
  const uint32_t at = shard * p.shard_places + min(shard, rest) + in, row = at / static_cast<uint32_t>(p.size_x);
  const uint32_t t = row / static_cast<uint32_t>(p.size_y);
  const int a = axis_of(p, pair);
  const uint32_t index = a == 0 ? t : a == 1 ? row - t * p.size_y : at - row * p.size_x;
  const double turn = fma(rate.y, static_cast<double>(index), rate.x);
  float2 r;
  sincospif(2.f * static_cast<float>(turn - rint(turn)), &r.y, &r.x);
  return r;
}

// How a CTA goes through the tokens: batches of `batch` tokens, in steps of `tokens` tokens times `width` heads (a power of two).
template <int D>
struct Deal {
  static constexpr int kLanes = D / 8;
  static constexpr int kRowsOfLanes = kThreads / kLanes;
  static constexpr int kPairs = D / 2;
  static constexpr int kBatch = kRowsOfLanes;                 // most tokens of a batch: one to each row of lanes
  int width, tokens, batch;
  __host__ __device__ __forceinline__ explicit Deal(int heads) {
    width = 1;
    while (width < kRowsOfLanes && width < heads) width *= 2;
    tokens = kRowsOfLanes / width;
    // at least as many tokens as there are threads for their angles
    batch = tokens > kThreads / kPairs ? tokens : kThreads / kPairs;
  }
  // The angles of the batch from token `first` on.  One batch's are written while slower warps may still read those of the one
  // before it, hence two buffers and one barrier.
  __device__ __forceinline__ void angles(const NormRopeGridParams& p, double2 rate, float2 (*to)[kPairs], int64_t first, int n) const {
    for (int i = threadIdx.x; i < n * kPairs; i += kThreads)
      // (tokens behind the last are padding: what shared memory holds there would be multiplied by 0, and need not be a number)
      to[i / kPairs][i % kPairs] = first + i / kPairs < p.tokens ? rotation(p, rate, first + i / kPairs, threadIdx.x % kPairs) : make_float2(0.f, 0.f);
    __syncthreads();
  }
};

// The four rotations of a lane's pairs.
__device__ __forceinline__ void load_turns(const float2* from, float (&cs)[4], float (&sn)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float4 v = *reinterpret_cast<const float4*>(from + i);
    cs[i] = v.x;
    sn[i] = v.y;
    cs[i + 1] = v.z;
    sn[i + 1] = v.w;
  }
}
__device__ __forceinline__ bool is_padding(const float (&cs)[4], const float (&sn)[4]) { return cs[0] == 0.f && sn[0] == 0.f; }

}  // namespace

// The steps of a CTA in their order: batch, tokens of the batch, heads of a token, queries then keys (kTensors = 2).
template <int kTensors>
struct Cursor {
  int64_t base;           // first token of the batch
  int t, h0, x;
  __device__ __forceinline__ void next(int step_tokens, int step_heads, int batch, int heads, int64_t stride) {
    if (kTensors == 2 && (x ^= 1) != 0) return;
    if ((h0 += step_heads) < heads) return;
    h0 = 0;
    if ((t += step_tokens) < batch) return;
    t = 0;
    base += stride;
  }
};

// How a kernel with U heads to a thread and step goes through the tokens.  kFull: there are at least as many heads as rows of lanes, so
// that a step is of one token (the same for all threads) and the heads of a thread lie a constant apart.
template <int D, int U, bool kFull>
struct Pace {
  using Deal = dtb::Deal<D>;
  static constexpr int kBatch = kFull ? kThreads / Deal::kPairs : Deal::kBatch;       // most tokens of a batch
  int width, tokens, batch, head0, sub;
  __device__ __forceinline__ explicit Pace(const Deal& deal) {
    constexpr int kLanes = D / 8;
    width = kFull ? Deal::kRowsOfLanes : deal.width;
    tokens = kFull ? 1 : deal.tokens;
    batch = kFull ? kBatch : deal.batch;
    head0 = kFull ? threadIdx.x / kLanes : threadIdx.x / kLanes % width;
    sub = kFull ? 0 : threadIdx.x / kLanes / width;
  }
};

// What a thread works on it copies itself, kAhead steps before, into its own places of a ring in shared memory: no barrier, and no
// registers for what is under way.
template <typename T, int D, bool kRms, bool kFull>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 6 : 5) norm_rope_grid_kernel(const __grid_constant__ NormRopeGridParams p) {
  // heads of a step, 16-byte pieces of a lane's part of a row, steps whose loads are under way
  constexpr int U = 3, kPieces = sizeof(T) / 2, kAhead = sizeof(T) == 2 ? 4 : 2;
  using Pace = Pace<D, U, kFull>;
  __shared__ __align__(16) float2 s_turn[2][Pace::kBatch][D / 2];
  __shared__ uint4 s_ring[kAhead][U * kPieces][kThreads];
  const int col = (threadIdx.x % (D / 8)) * 8;
  const int most = max(p.heads[0], p.heads[1]);
  const Deal<D> deal(most);
  const Pace pace(deal);
  uint64_t w[2][4], b[2][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    Raw8<T> r;
    load8(r, static_cast<const T*>(p.weight[x]) + col);
    unpack8(r, w[x]);
    r = Raw8<T>{};
    if (p.bias[x] != nullptr) load8(r, static_cast<const T*>(p.bias[x]) + col);
    unpack8(r, b[x]);
  }
  const int64_t stride = static_cast<int64_t>(gridDim.x) * pace.batch;
  Cursor<2> at{static_cast<int64_t>(blockIdx.x) * pace.batch, 0, 0, 0}, ahead = at;
  int slot = 0;
  auto copy = [&]() {
    const int x = ahead.x;
    const int64_t tok = ahead.base + ahead.t + pace.sub;
    if (ahead.base < p.tokens) {
      const int64_t seq_no = tok / p.seq;
      const T* src = static_cast<const T*>(x ? p.src[1] : p.src[0]) + seq_no * (x ? p.batch_stride[1] : p.batch_stride[0]) +
                     (tok - seq_no * p.seq) * (x ? p.tok_stride[1] : p.tok_stride[0]) + col + (ahead.h0 + pace.head0) * D;
      const int heads = tok < p.tokens ? (x ? p.heads[1] : p.heads[0]) - ahead.h0 - pace.head0 : 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u * pace.width < heads) copy8(&s_ring[slot][u * kPieces][threadIdx.x], src + u * pace.width * D, true);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead.next(pace.tokens, U * pace.width, pace.batch, most, stride);
    if (++slot == kAhead) slot = 0;
  };
  // (rows that were not loaded are worked on all the same and not stored: a row's lanes keep to themselves)
  auto work = [&](int x, int64_t tok, int h0, const float2* turns) {
    float cs[4], sn[4];
    load_turns(turns, cs, sn);
    const bool padding = is_padding(cs, sn);
    T* dst = static_cast<T*>(x ? p.dst[1] : p.dst[0]) + tok * ((x ? p.heads[1] : p.heads[0]) * D) + col + (h0 + pace.head0) * D;
    const int heads = tok < p.tokens ? (x ? p.heads[1] : p.heads[0]) - h0 - pace.head0 : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Raw8<T> raw;
      read8(raw, &s_ring[slot][u * kPieces][threadIdx.x]);
      if (padding) raw = Raw8<T>{};             // (it may hold anything, and 0 times that need not be 0)
      uint64_t v[4];
      unpack8(raw, v);
      standardise<D, kRms>(v, x ? p.eps[1] : p.eps[0]);
      float z[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float re, im;
        unpack2(fma2(v[i], w[x][i], b[x][i]), re, im);
        z[2 * i] = re * cs[i] - im * sn[i];
        z[2 * i + 1] = im * cs[i] + re * sn[i];
      }
      if (u * pace.width < heads) store8(dst + u * pace.width * D, z);
    }
  };
  for (int i = 0; i < kAhead; ++i) copy();
  const double2 rate = rate_of(p, threadIdx.x % (D / 2));        // (a thread forms the angles of one pair only)
  int buffer = 0;
  // (all bounds are the same for all threads of the CTA: barriers and shuffles)
  for (; at.base < p.tokens; at.base += stride) {
    const float2(*turns)[D / 2] = s_turn[buffer];
    deal.angles(p, rate, s_turn[buffer], at.base, pace.batch);
    buffer ^= 1;
    for (int t = 0; t < pace.batch; t += pace.tokens) {
      const int64_t tok = at.base + t + pace.sub;
      for (int h0 = 0; h0 < most; h0 += U * pace.width) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
          work(x, tok, h0, &turns[t + pace.sub][col / 2]);
          copy();
        }
      }
    }
  }
}

// grid: (CTAs, tensor).  kBias: sums for a bias are wanted.
template <typename T, int D, bool kRms, bool kFull, bool kBias>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 6 : 4) norm_rope_grid_backward_kernel(const __grid_constant__ NormRopeGridParams p) {
  constexpr int kLanes = D / 8;
  constexpr int U = sizeof(T) == 2 ? 3 : 2, kPieces = sizeof(T) / 2, kAhead = 2;
  using Pace = Pace<D, U, kFull>;
  constexpr int kRing = kAhead * 2 * U * kPieces * kThreads, kSums = kThreads / kLanes * 2 * D / 4;      // pieces of 16 bytes
  __shared__ __align__(16) float2 s_turn[2][Pace::kBatch][D / 2];
  __shared__ uint4 s_ring[kRing > kSums ? kRing : kSums];           // [step][x, gradient][head][thread]; in the end the sums
  const int x = blockIdx.y;
  const int heads = p.heads[x];
  const int col = (threadIdx.x % kLanes) * 8;
  const Deal<D> deal(heads);
  const Pace pace(deal);
  uint64_t w[4], dw[4], db[4];
  {
    Raw8<T> r;
    load8(r, static_cast<const T*>(p.weight[x]) + col);
    unpack8(r, w);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) dw[i] = db[i] = pack2(0.f, 0.f);
  const float eps = p.eps[x];
  const int64_t stride = static_cast<int64_t>(gridDim.x) * pace.batch;
  Cursor<1> at{static_cast<int64_t>(blockIdx.x) * pace.batch, 0, 0, 0}, ahead = at;
  int slot = 0;
  auto place = [&](int which, int u) { return s_ring + ((slot * 2 + which) * U + u) * kPieces * kThreads + threadIdx.x; };
  // (a row that is not there is 0 and adds nothing)
  auto copy = [&]() {
    const int64_t tok = min(ahead.base + ahead.t + pace.sub, p.tokens - 1);
    const int64_t seq_no = tok / p.seq, s = tok - seq_no * p.seq;
    const int left = ahead.base + ahead.t + pace.sub < p.tokens ? heads - ahead.h0 - pace.head0 : 0;
    const int first = col + (ahead.h0 + pace.head0) * D;
    const T* src = static_cast<const T*>(p.src[x]) + seq_no * p.batch_stride[x] + s * p.tok_stride[x];
    const T* grad = static_cast<const T*>(p.grad[x]) + seq_no * p.grad_batch_stride[x] + s * p.grad_tok_stride[x];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = u * pace.width < left;
      const int h = there ? first + u * pace.width * D : col;
      copy8(place(0, u), src + h, there);
      copy8(place(1, u), grad + h, there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead.next(pace.tokens, U * pace.width, pace.batch, heads, stride);
    if (++slot == kAhead) slot = 0;
  };
  auto work = [&](int64_t tok, int h0, const float2* turns) {
    float cs[4], sn[4];
    load_turns(turns, cs, sn);
    const bool padding = is_padding(cs, sn);
    T* dst = static_cast<T*>(p.dst[x]) + tok * (heads * D) + col + (h0 + pace.head0) * D;
    const int left = tok < p.tokens ? heads - h0 - pace.head0 : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Raw8<T> rx, rg;
      read8(rx, place(0, u));
      read8(rg, place(1, u));
      if (padding) rx = rg = Raw8<T>{};               // (padding, and its gradient, may hold anything)
      uint64_t v[4], g[4];
      unpack8(rx, v);
      unpack8(rg, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float re, im;
        unpack2(g[i], re, im);
        g[i] = pack2(re * cs[i] + im * sn[i], im * cs[i] - re * sn[i]);
      }
      const float rstd = standardise<D, kRms>(v, eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dw[i] = fma2(g[i], v[i], dw[i]);
        if (kBias) db[i] = add2(db[i], g[i]);
        g[i] = mul2(g[i], w[i]);
      }
      const uint64_t gx = fma2(g[0], v[0], fma2(g[1], v[1], fma2(g[2], v[2], mul2(g[3], v[3]))));
      // dx = rstd g - rstd mean(g) - v rstd mean(g v)
      const float of_v = row_sum<kLanes>(sum_of(gx)) * (1.f / D) * -rstd;
      const float shift = kRms ? 0.f : row_sum<kLanes>(sum_of(add2(add2(g[0], g[1]), add2(g[2], g[3])))) * (1.f / D) * -rstd;
      const uint64_t scale = pack2(rstd, rstd), factor = pack2(of_v, of_v), shifts = pack2(shift, shift);
      float z[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack2(fma2(v[i], factor, kRms ? mul2(g[i], scale) : fma2(g[i], scale, shifts)), z[2 * i], z[2 * i + 1]);
      if (u * pace.width < left) store8(dst + u * pace.width * D, z);
    }
  };
  if (p.tokens > 0) {
    for (int i = 0; i < kAhead; ++i) copy();
  }
  const double2 rate = rate_of(p, threadIdx.x % (D / 2));        // (a thread forms the angles of one pair only)
  int buffer = 0;
  for (; at.base < p.tokens; at.base += stride) {
    const float2(*turns)[D / 2] = s_turn[buffer];
    deal.angles(p, rate, s_turn[buffer], at.base, pace.batch);
    buffer ^= 1;
    for (int t = 0; t < pace.batch; t += pace.tokens) {
      for (int h0 = 0; h0 < heads; h0 += U * pace.width) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        work(at.base + t + pace.sub, h0, &turns[t + pace.sub][col / 2]);
        copy();
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();                                     // the ring's memory takes the sums
  grid_launch_dependents();                            // the kernel that adds them up may be set up meanwhile; it waits for this one's end
  float(*s_sum)[2 * D] = reinterpret_cast<float(*)[2 * D]>(s_ring);
  const int row = threadIdx.x / kLanes;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unpack2(dw[i], s_sum[row][col + 2 * i], s_sum[row][col + 2 * i + 1]);
    unpack2(db[i], s_sum[row][D + col + 2 * i], s_sum[row][D + col + 2 * i + 1]);
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
__global__ void __launch_bounds__(1024) norm_rope_grid_sums_kernel(const __grid_constant__ NormRopeGridSums to, const float* partial, int rows) {
  __shared__ float s_sum[32][33];
  grid_dependency_wait();
  const int x = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  const float* from = partial + static_cast<int64_t>(x) * rows * (2 * D) + c;
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
    void* dst = at < D ? to.weight_grad[x] : to.bias_grad[x];
    if (dst != nullptr) store1(static_cast<T*>(dst) + (at < D ? at : at - D), sum);
  }
}

template <typename T, int D, bool kRms>
static cudaError_t launch_forward(const NormRopeGridParams& p, int sm_count, cudaStream_t stream) {
  const int most = p.heads[0] > p.heads[1] ? p.heads[0] : p.heads[1];
  const int batch = Deal<D>(most).batch;
  const int64_t need = (p.tokens + batch - 1) / batch, cap = static_cast<int64_t>(sm_count) * (sizeof(T) == 2 ? 6 : 5);
  const unsigned ctas = static_cast<unsigned>(need < cap ? need : cap);
  if (most >= Deal<D>::kRowsOfLanes) norm_rope_grid_kernel<T, D, kRms, true><<<ctas, kThreads, 0, stream>>>(p);
  else norm_rope_grid_kernel<T, D, kRms, false><<<ctas, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, int D, bool kRms, bool kBias>
static cudaError_t launch_backward_as(const NormRopeGridParams& p, const NormRopeGridSums& sums, int sm_count, cudaStream_t stream) {
  const int least = p.heads[0] < p.heads[1] ? p.heads[0] : p.heads[1], most = p.heads[0] + p.heads[1] - least;
  const int batch = Deal<D>(most).batch;
  const int64_t need = (p.tokens + batch - 1) / batch, cap = static_cast<int64_t>(sm_count) * kBackwardPerSm;
  // (without tokens one CTA still writes its sums, which are 0)
  const int ctas = static_cast<int>(need < 1 ? 1 : need < cap ? need : cap);
  if (least >= Deal<D>::kRowsOfLanes) norm_rope_grid_backward_kernel<T, D, kRms, true, kBias><<<dim3(ctas, 2), kThreads, 0, stream>>>(p);
  else norm_rope_grid_backward_kernel<T, D, kRms, false, kBias><<<dim3(ctas, 2), kThreads, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_attention_kernel(norm_rope_grid_sums_kernel<T, D>, dim3(2 * D / 32, 2), 1024, 0, stream, true, sums, static_cast<const float*>(p.partial), ctas);
}

template <typename T, int D, bool kRms>
static cudaError_t launch_backward(const NormRopeGridParams& p, const NormRopeGridSums& sums, int sm_count, cudaStream_t stream) {
  return sums.bias_grad[0] != nullptr || sums.bias_grad[1] != nullptr ? launch_backward_as<T, D, kRms, true>(p, sums, sm_count, stream)
                                                                      : launch_backward_as<T, D, kRms, false>(p, sums, sm_count, stream);
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

cudaError_t launch_norm_rope_grid_backward(const NormRopeGridParams& p, const NormRopeGridSums& sums, int head_dim, bool bf16, bool rms, int sm_count, cudaStream_t stream) {
  if (head_dim == 64) {
    if (bf16) return rms ? launch_backward<uint16_t, 64, true>(p, sums, sm_count, stream) : launch_backward<uint16_t, 64, false>(p, sums, sm_count, stream);
    return rms ? launch_backward<float, 64, true>(p, sums, sm_count, stream) : launch_backward<float, 64, false>(p, sums, sm_count, stream);
  }
  if (bf16) return rms ? launch_backward<uint16_t, 128, true>(p, sums, sm_count, stream) : launch_backward<uint16_t, 128, false>(p, sums, sm_count, stream);
  return rms ? launch_backward<float, 128, true>(p, sums, sm_count, stream) : launch_backward<float, 128, false>(p, sums, sm_count, stream);
}

}  // namespace dtb
