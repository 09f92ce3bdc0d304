// Attention of few query rows over keys and values in pages: all keys of all sequences dealt evenly to CTAs that stay.
//
// A row is a query and one of the heads that share a key head; a block of up to 16, 32, 48 or 64 rows of one key head meets the keys that any row of
// its sequence sees, [0, first) and [lo, hi), in tiles of 64.  Sequence after sequence, key head after key head, block after block, places
// are numbered through, one per tile and a few in front of each block for what that costs, and each CTA takes as many of them as any other: the
// lengths stand on the device, and so every CTA works out for itself where its share begins.  Per warp of rows and keys a softmax state (m, l, O) is kept:
//     S = Q K^T,  m' = max(m, max S) where that grew by more than 2^8, else m,  P = 2^(c (S - m')),
//     l' = l 2^(c (m - m')) + sum P,  O' = O 2^(c (m - m')) + P V
// The states of the warps are joined in shared memory.  A block that one CTA has all tiles of is written as it is; the parts of one that several
// CTAs have go to scratch, and a second launch, set up while this one runs, joins them in the order of their CTAs.
// Small batches take one launch: a cluster of up to 8 CTAs to each block, which share its tiles out and join their states through distributed
// shared memory, and nothing to add up beforehand.
//
// HBM-bound: a key and a value are read once for the rows of a block.  The last warp loads (TMA, 128-byte swizzle, every lane a page), the others, three for
// blocks of 48 rows and else four, compute with mma.sync, because 16 rows fill an instruction of it and a 128-row tile of tcgen05 would be empty for the most
// part.  With more than 16 rows the warps share the rows out, not the keys, so that what a key costs in shared memory reads stays below what it costs in HBM.
// P is rounded to bf16 for the product (by 2^-8 of each weight at most, as in the other attention kernels); scores, sums and states are fp32.
//
// us, one launch after another, and keys and values a second: 32 heads over 8 of 128, 24 tokens against 200 to 30000 keys each 105 (5.9 TB/s); a
// token of 24 heads of 128 against 119056 keys 209; of 32 over 8 of 64 against 1500 keys 6.8 to 7.2.  What a launch takes beside its keys: 2 us until a share is
// known, 3 until the first tile is there, 2 to 5 for the join.  Five queries of 32 heads over 4 of 64 against seven sequences of 5003 to 20011 keys: 29 us,
// bound by those and by the rate of mma.sync on 40 rows.  Two CTAs to an SM: with one the 24 tokens take 142, with three CTAs to two SMs 110.
#include "flash_common.cuh"
#include "flash_paged.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

namespace dtb {

namespace {

using namespace flash;

constexpr int kKeys = 64;                 // of a tile
constexpr int kBlockCost = 2;             // places in front of a block's tiles
constexpr int kMinPlaces = 2;             // of a CTA's share, unless there are fewer
constexpr int kColumns = 32;              // joined at a time
constexpr int kMostCluster = 8;
constexpr int kPitch = kColumns + 8;      // floats of a row of them in shared memory (rows 8 banks apart)

template <int D, int WM>
struct Cfg {
  static constexpr int kRows = 16 * WM;
  static constexpr int kMathWarps = WM == 3 ? 3 : 4;
  static constexpr int kThreads = (kMathWarps + 1) * 32;
  static constexpr int kWN = kMathWarps / WM;                // warps that share a tile's keys
  static constexpr int kWarpKeys = kKeys / kWN;
  static constexpr int kSlabs = D / 64;
  static constexpr int kSlab = kKeys * 128;                  // bytes of 64 channels of a tile
  static constexpr int kStage = 2 * kSlabs * kSlab;          // K and V
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kJoin = kWN * kRows * kPitch * 4;
  static constexpr int kBytes = 1024 + kStages * kStage + kJoin + kWN * kRows * 8 + 2 * kStages * 8 + 64;
  static_assert(2 * (kBytes + 1024) <= 228 * 1024, "two CTAs to an SM");
};

// What the launch that joins has to know of a block that several CTAs have parts of.  There is one for each block where the host knows that blocks are
// fewer than boundaries between shares, else one for each boundary; only the first one inside a block counts.
struct alignas(16) Join {
  int parts;                 // 0: of none
  int cta, late;             // that has the first part; whether that was not the first block of its share
  int seg, q_begin, kv_head, row0, rows;
};

// A sequence as its rows' keys are walked.
struct Seq {
  WindowSeq w;
  int blocks;                // of rows, for each key head
  int first, lo, hi;         // keys that any row sees: [0, first) and [lo, hi)
  int lead;                  // tiles of the former
  int tiles;                 // in all, 1 where there is no key: the block's rows are written all the same
  int group;                 // query heads of a key head

  __device__ __forceinline__ int begin(int tile) const { return tile < lead ? tile * kKeys : lo + (tile - lead) * kKeys; }
};

template <int R>
__device__ __forceinline__ Seq make_seq(const PagedParams& p, int seg) {
  Seq s;
  s.w = paged_seq(p, seg);
  if (s.w.q_len > p.few_rows) s.w.q_len = 0;
  s.group = p.f.num_heads / p.kv_heads;
  s.blocks = (s.w.q_len * s.group + R - 1) / R;
  const WindowSpan a = window_span(s.w, 0), z = window_span(s.w, max(s.w.q_len - 1, 0));
  s.first = z.first;
  s.hi = z.hi;
  s.lo = max(a.lo, s.first);
  const int n = max(s.hi - s.lo, 0);
  if (n > 0) s.lo &= ~(p.key_align - 1);
  s.lead = (s.first + kKeys - 1) / kKeys;
  s.tiles = s.lead + (n > 0 ? (s.hi - s.lo + kKeys - 1) / kKeys : 0);
  if (s.tiles == 0) s.tiles = 1;
  return s;
}

// A block's rows and what they see together.
struct Block {
  int kv_head, row0, rows;
  int first, lo, hi;

  // of the tile that begins at key a: the keys that some row sees, [from, to)
  __device__ __forceinline__ void seen(int a, bool lead, int& from, int& to) const {
    from = lead ? a : max(a, lo);
    to = min(a + kKeys, lead ? first : hi);
  }
};

template <int R>
__device__ __forceinline__ Block make_block(const PagedParams& p, const Seq& s, int unit) {
  Block b;
  b.kv_head = unit / s.blocks;
  b.row0 = (unit - b.kv_head * s.blocks) * R;
  b.rows = min(R, s.w.q_len * s.group - b.row0);
  const WindowSpan a = window_span(s.w, b.row0 / s.group), z = window_span(s.w, (b.row0 + b.rows - 1) / s.group);
  b.first = z.first;
  b.lo = max(a.lo, z.first);
  b.hi = z.hi;
  return b;
}

// Shares: the first `longer` CTAs have `size` + 1 places, the others `size`.  (Divisions in 32 bits where they do: they are a fifth as long.)
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((a | b) >> 31) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
struct Shares {
  int64_t all, size;
  int ctas, longer;

  __device__ __forceinline__ Shares(int64_t places, int most) {
    all = places;
    const int64_t n = places / kMinPlaces;
    ctas = static_cast<int>(n < 1 ? (places > 0) : n < most ? n : most);
    size = ctas > 0 ? divide(places, ctas) : 0;
    longer = static_cast<int>(places - size * ctas);
  }
  __device__ __forceinline__ int64_t begin(int c) const { return c * size + min(c, longer); }
  __device__ __forceinline__ int of(int64_t place) const {
    const int64_t first = longer * (size + 1);
    return static_cast<int>(place < first ? divide(place, size + 1) : longer + divide(place - first, size));
  }
};

// Places of a sequence's block, and the tiles that lie in front of one of them.
__device__ __forceinline__ int places_of(const Seq& s) { return s.tiles + kBlockCost; }
__device__ __forceinline__ int tiles_before(int place) { return max(place - kBlockCost, 0); }

// The record of the boundary in front of CTA `cta`, whose share begins at `place` of the block.
__device__ __forceinline__ Join make_join(const Shares& sh, const Seq& s, const Block& b, int seg, int cta, int place) {
  Join j = {0, 0, 0, seg, s.w.q_begin, b.kv_head, b.row0, b.rows};
  if (tiles_before(place) > 0) {
    const int64_t begin = sh.begin(cta) - place;
    const int c0 = sh.of(begin + kBlockCost), c1 = sh.of(begin + places_of(s) - 1);      // that have its first tile, and its last
    if (c0 == cta - 1) {
      j.parts = c1 - c0 + 1;
      j.cta = c0;
      j.late = sh.begin(c0) < begin;
    }
  }
  return j;
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d += a b: 16 x 16 (rows x k) by 16 x 8
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
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

// (m, l) of a row whose state was not formed, because a wait gave up: a sum of weights is not negative.
__device__ __forceinline__ float2 lost_state() { return make_float2(0.f, -1.f); }
__device__ __forceinline__ bool is_lost(float l) { return l < 0.f; }

template <int N>
__device__ __forceinline__ void math_warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory"); }

// The lse of a row: of the maximum of its raw scores and the sum of its weights.
__device__ __forceinline__ float lse_of(const PagedParams& p, float m, float l) { return (m * p.f.scale_log2 + log2f(l)) * kLn2; }

// Four columns of a finished row: normalised, merged with the state in memory where the launch accumulates, stored.  `write_lse`: this thread
// writes the row's lse; the threads of a row that read it before are all in its warp (`mask`) or behind a barrier.
template <int D>
__device__ __forceinline__ void store_row4(const PagedParams& p, int seg, int q_begin, int i, int head, int col, float4 acc, float lse, float l,
                                           bool write_lse, uint32_t mask) {
  const int64_t tok = p.f.cu_q != nullptr ? static_cast<int64_t>(q_begin) + i : static_cast<int64_t>(seg) * p.f.seqlen_q + i;
  const int64_t li = lse_index(p.f, seg, head, i, tok), oi = tok * p.f.out_tok_stride + static_cast<int64_t>(head) * D + col;
  const bool empty = l == 0.f;                    // no key seen: nothing to write over a state  (a NaN among the scores is not empty)
  const bool keep = empty && p.f.accumulate != 0;
  float lse_out = -INFINITY;
  if (!keep) {
    float w_new = 0.f, w_old = 0.f;
    if (!empty) merge_weights(p.f.accumulate != 0, p.f.accumulate ? p.f.lse[li] : -INFINITY, lse, l, w_new, w_old, lse_out);
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
  }
  __syncwarp(mask);
  if (write_lse && !keep) p.f.lse[li] = lse_out;
}

// The scratch of a launch: records, then the states' (m, l) and values, two of each CTA (of the first block of its share, and of the last).
template <int D, int R>
struct Scratch {
  Join* joins;
  float2* ml;
  float* o;
  __host__ __device__ Scratch(void* base, int ctas) {
    joins = static_cast<Join*>(base);
    ml = reinterpret_cast<float2*>(joins + ctas);
    o = reinterpret_cast<float*>(ml + 2 * static_cast<int64_t>(ctas) * R);
  }
};

}  // namespace

// grid: the CTAs that share all places out; with kCluster (row blocks x key heads x sequences) clusters, a row block of each sequence's `row_blocks`.
// (Of shares: row_blocks > 0 where joins go by blocks.)
template <int D, int WM, bool kCluster>
__global__ void __launch_bounds__(Cfg<D, WM>::kThreads, 2)
flash_paged_rows_kernel(const __grid_constant__ PagedMap tm_k, const __grid_constant__ PagedMap tm_v, const __grid_constant__ PagedParams p, void* scratch,
                        int row_blocks) {
  namespace cg = cooperative_groups;
  using C = Cfg<D, WM>;
  constexpr int R = C::kRows, WN = C::kWN, KW = C::kWarpKeys, kMathWarps = C::kMathWarps, kThreads = C::kThreads;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  float* s_join = reinterpret_cast<float*>(smem + C::kStages * C::kStage);            // [warp of keys][row][kPitch]
  float2* s_ml = reinterpret_cast<float2*>(s_join + C::kJoin / 4);                     // [warp of keys][row]
  float* s_state = reinterpret_cast<float*>(smem);                                     // of a cluster's CTA: O [row][D], (m, l) [row], over the ring
  float2* s_state_ml = reinterpret_cast<float2*>(s_state + R * D);
  static_assert(R * (D * 4 + 8) <= C::kStages * C::kStage, "states take the ring's place");
  uint64_t* full = reinterpret_cast<uint64_t*>(s_ml + WN * R);
  uint64_t* empty = full + C::kStages;
  __shared__ long long s_sum[kThreads / 32];
  __shared__ Seq s_seq;                     // the share's first sequence, ...
  __shared__ Seq s_seqs[kThreads / 32];     // the one that each warp is at: in registers it would have others spilled
  __shared__ int s_seg, s_unit, s_place;    // ... (key head, row block) of that, and place of the block
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Scratch<D, R> sc(scratch, gridDim.x);

  grid_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kMathWarps);
    }
    fence_mbar_init();
  }
  if (warp == kMathWarps && lane == 0) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  // ------------------------------------------------------------------ this CTA's share
  int seg, unit, place;
  long long left;                           // places
  const int cta = blockIdx.x;
  bool ok = true;                           // after a wait that gave up, the blocks are walked to their barriers and no result is stored
  Seq& s = s_seqs[warp];
  if constexpr (kCluster) {
    // (Nobody leaves here after a failure elsewhere: the others of its cluster wait for it.  Rows are lost by it all the same.)
    const int word = *reinterpret_cast<volatile int*>(p.f.status);
    const int ranks = static_cast<int>(cg::this_cluster().num_blocks()), rank = static_cast<int>(cg::this_cluster().block_rank());
    int id = cta / ranks;
    const int block = id % row_blocks;
    id /= row_blocks;
    seg = id / p.kv_heads;
    const Seq own = make_seq<R>(p, seg);
    if (block >= own.blocks) return;        // all CTAs of the cluster
    unit = (id - seg * p.kv_heads) * own.blocks + block;
    const int t0 = static_cast<int>(static_cast<int64_t>(own.tiles) * rank / ranks), t1 = static_cast<int>(static_cast<int64_t>(own.tiles) * (rank + 1) / ranks);
    place = t0 + kBlockCost;
    left = t1 - t0;
    if (lane == 0) s = own;
    if (__syncthreads_or(word != 0)) ok = false;      // the barriers are there
  } else {
    const int per = (p.f.nseg + kThreads - 1) / kThreads, seg0 = min(static_cast<int>(threadIdx.x) * per, p.f.nseg), seg1 = min(seg0 + per, p.f.nseg);
    auto places = [&](const Seq& s) { return static_cast<long long>(s.blocks) * p.kv_heads * places_of(s); };
    long long sum = 0;
    Seq own;
    for (int i = seg0; i < seg1; ++i) sum += places(own = make_seq<R>(p, i));
    long long upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const long long u = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += u;
    }
    if (lane == 31) s_sum[warp] = upto;
    // CTA-uniform view of the status word: a CTA that starts after a failure elsewhere walks its blocks as after one of its own.  (It does not just leave: the
    // launch behind this one follows the records, and the word may be clear again by then.)
    if (__syncthreads_or(*reinterpret_cast<volatile int*>(p.f.status) != 0)) ok = false;
    long long at = upto - sum, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += s_sum[w];
      all += s_sum[w];
    }
    const Shares shares(all, gridDim.x);
    if (cta >= shares.ctas) {
      if (threadIdx.x == 0 && row_blocks == 0) sc.joins[cta].parts = 0;
      return;
    }
    const long long begin = shares.begin(cta);
    if (begin >= at && begin < at + sum) {
      for (int i = seg0; i < seg1; ++i) {
        if (per > 1) own = make_seq<R>(p, i);
        if (begin < at + places(own)) {
          s_seq = own;
          s_seg = i;
          s_unit = static_cast<int>(divide(begin - at, places_of(own)));
          s_place = static_cast<int>(begin - at - static_cast<long long>(s_unit) * places_of(own));
          break;
        }
        at += places(own);
      }
    }
    __syncthreads();
    seg = s_seg;
    unit = s_unit;
    place = s_place;
    left = shares.begin(cta + 1) - begin;
    if (lane == 0) s = s_seq;
    __syncwarp();
    if (threadIdx.x == 0) {
      const Block b = make_block<R>(p, s, unit);
      const Join j = make_join(shares, s, b, seg, cta, place);
      if (row_blocks == 0) sc.joins[cta] = j;
      else if (j.parts > 0) sc.joins[(seg * p.kv_heads + b.kv_head) * row_blocks + b.row0 / R] = j;
    }
  }
  const int unit0 = unit;
  int stage = 0;
  uint32_t use = 0;                         // parity of the ring's round
  bool first_block = true;
  // the block's tiles that are this CTA's: up to, not with, this one
  auto last_tile = [&]() { return tiles_before(static_cast<int>(min(static_cast<long long>(places_of(s)), place + left))); };
  auto next_block = [&]() {
    left -= min(static_cast<long long>(places_of(s) - place), left);
    place = 0;
    first_block = false;
    if (++unit == s.blocks * p.kv_heads && left > 0) {
      unit = 0;
      Seq next;
      do next = make_seq<R>(p, ++seg); while (next.blocks == 0);
      __syncwarp();
      if (lane == 0) s = next;
      __syncwarp();
    }
  };

  if (warp == kMathWarps) {
    // ---------------------------------------------------------------- loads: a lane per box of tokens
    bool wrapped = false;
    const int box = p.box_rows, boxes = kKeys / box;
    while (ok && left > 0) {
      const Block b = make_block<R>(p, s, unit);
      const int tile = tiles_before(place), to = last_tile();
      const int32_t* row = p.table + static_cast<int64_t>(seg) * p.columns;
      // This lane's entry for a tile, looked up while the loads of the tile before are issued.  (24 tokens of 32 heads over 8 of 64, pages of 16: 62.3 us
      // -> 59.1.)
      auto look_up = [&](int t) {
        const int j = (s.begin(t) + lane * box) >> p.page_shift;
        return lane < boxes && j < p.columns ? row[j] : -1;
      };
      int entry = tile < to ? look_up(tile) : -1;
      for (int t = tile; t < to; ++t) {
        const int a = s.begin(t);
        int page = entry;
        if (t + 1 < to) entry = look_up(t + 1);
        int from, upto_key;
        b.seen(a, t < s.lead, from, upto_key);
        if (from >= upto_key) continue;
        const int key = a + lane * box, n = (upto_key - a + box - 1) / box;       // boxes that hold a key of the tile
        if (page < 0 || page >= p.pages) page = p.pages;         // filled with zeros
        if (wrapped && !warp_wait_or_abort(&empty[stage], use ^ 1, p.f.status, 62)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_expect_tx(&full[stage], n * box * 128 * 2 * C::kSlabs);
        __syncwarp();
        if (lane < n) {
          uint8_t* dst = smem + stage * C::kStage + lane * box * 128;
          const int in_page = key & ((1 << p.page_shift) - 1);
          const int ka = p.k_batch_first ? b.kv_head : in_page, kb = p.k_batch_first ? in_page : b.kv_head;
          const int va = p.v_batch_first ? b.kv_head : in_page, vb = p.v_batch_first ? in_page : b.kv_head;
#pragma unroll
          for (int x = 0; x < C::kSlabs; ++x) tma_load_4d(dst + x * C::kSlab, &tm_k.map, &full[stage], x * 64, ka, kb, page);
#pragma unroll
          for (int x = 0; x < C::kSlabs; ++x) tma_load_4d(dst + (C::kSlabs + x) * C::kSlab, &tm_v.map, &full[stage], x * 64, va, vb, page);
        }
        if (++stage == C::kStages) {
          stage = 0;
          use ^= 1;
          wrapped = true;
        }
      }
      next_block();
    }
  } else {
    // ---------------------------------------------------------------- scores, weights, products
    const int wm = warp / WN, wn = warp % WN;
    const float c = p.f.scale_log2;
    for (bool once = kCluster; once || left > 0; once = false) {
      const int tile = tiles_before(place), to = last_tile(), group = s.group;
      if (!kCluster && tile == to) {                         // places in front of a block that the next CTA begins with
        next_block();
        continue;
      }
      const Block b = make_block<R>(p, s, unit);
      // this thread's rows lane / 4 and lane / 4 + 8 of the warp's 16; rows that there are not see what the last one sees
      int end_first[2], from_w[2], to_w[2];
      uint32_t qf[D / 16][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * wm + (lane >> 2) + 8 * h, row = b.row0 + min(r, b.rows - 1);
        const int i = row / group, g = row % group;
        const WindowSpan w = window_span(s.w, i);
        end_first[h] = w.first;
        from_w[h] = w.lo;
        to_w[h] = w.hi;
        const uint16_t* src = r < b.rows ? p.q + window_offset(p, seg, static_cast<int64_t>(s.w.q_begin) + i, p.q_tok, p.q_batch) + static_cast<int64_t>(b.kv_head * group + g) * D : nullptr;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            qf[k][h + 2 * half] = src != nullptr ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 * half + 2 * (lane & 3)) : 0u;
      }
      float o[D / 8][4];
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      for (int t = tile; t < to; ++t) {
        const int a = s.begin(t);
        const bool lead = t < s.lead;
        int from, upto_key;
        b.seen(a, lead, from, upto_key);
        if (from >= upto_key) continue;
        ok = ok && warp_wait_or_abort(&full[stage], use, p.f.status, 61);
        if (ok) {
          const int key0 = wn * KW;               // of the tile, the warp's first
          const uint32_t ks = smem_u32(smem + stage * C::kStage), vs = ks + C::kSlabs * C::kSlab;
          const bool ragged = from > a || upto_key < a + kKeys;
          if (ragged) {
            // values of keys that no row sees may be anything, and 0 times that is not 0
            for (int u = lane; u < KW * C::kSlabs * 8; u += 32) {
              const int row = key0 + u / (C::kSlabs * 8), piece = u % (C::kSlabs * 8);
              if (a + row < from || a + row >= upto_key)
                *reinterpret_cast<uint4*>(smem + stage * C::kStage + (C::kSlabs + piece / 8) * C::kSlab + row * 128 + piece % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          // (all keys for 16 channels before the next 16: as many chains of products as the warp has keys to feed them)
          float sr[KW / 8][4];
#pragma unroll
          for (int n = 0; n < KW / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sr[n][e] = 0.f;
          const uint32_t k_row = ks + (key0 + ((lane >> 4) << 3) + (lane & 7)) * 128;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t piece = (k >> 2) * C::kSlab + ((((2 * k + ((lane >> 3) & 1)) & 7) ^ (lane & 7)) << 4);
#pragma unroll
            for (int n = 0; n < KW / 16; ++n) {
              uint32_t f[4];
              ldmatrix4(k_row + n * 16 * 128 + piece, f);
              mma16816(sr[2 * n], qf[k], f[0], f[1]);
              mma16816(sr[2 * n + 1], qf[k], f[2], f[3]);
            }
          }
          // columns of the warp's keys that the rows see, [c0, c1)
          int c0[2], c1[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            c0[h] = lead ? 0 : from_w[h] - a - key0;
            c1[h] = (lead ? end_first[h] : to_w[h]) - a - key0;
          }
          if (__any_sync(0xffffffffu, max(c0[0], c0[1]) > 0 || min(c1[0], c1[1]) < KW)) {
#pragma unroll
            for (int n = 0; n < KW / 8; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int h = e >> 1, x = n * 8 + 2 * (lane & 3) + (e & 1);
                if (x < c0[h] || x >= c1[h]) sr[n][e] = -INFINITY;
              }
          }
          float mx[2];
          bool grows = false;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v = fmaxf(sr[0][2 * h], sr[0][2 * h + 1]);
#pragma unroll
            for (int n = 1; n < KW / 8; ++n) v = max3(v, sr[n][2 * h], sr[n][2 * h + 1]);
            mx[h] = fmaxf(m[h], quad_max(v));
            grows = grows || (mx[h] - m[h]) * c > kRescaleThreshold;       // (from -inf without end; -inf - -inf is not)
          }
          if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float f = m[h] == mx[h] ? 1.f : ex2((m[h] - mx[h]) * c);
              m[h] = mx[h];
              l[h] *= f;
#pragma unroll
              for (int i = 0; i < D / 8; ++i) {
                o[i][2 * h] *= f;
                o[i][2 * h + 1] *= f;
              }
            }
          }
          // P, a pair of columns of a row at a time
          uint32_t pr[KW / 8][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float ref = -reference(m[h]) * c;
            const uint64_t c2 = pack2(c, c), ref2 = pack2(ref, ref);
            uint64_t sum2 = pack2(l[h], 0.f);
#pragma unroll
            for (int n = 0; n < KW / 8; ++n) {
              const uint64_t w2 = exp2_mufu2(fma2(pack2(sr[n][2 * h], sr[n][2 * h + 1]), c2, ref2));
              sum2 = add2(sum2, w2);
              float w0, w1;
              unpack2(w2, w0, w1);
              pr[n][h] = pack_bf16x2(w0, w1);
            }
            float s0, s1;
            unpack2(sum2, s0, s1);
            l[h] = s0 + s1;
          }
#pragma unroll
          for (int n = 0; n < KW / 16; ++n) {
            const uint32_t w[4] = {pr[2 * n][0], pr[2 * n][1], pr[2 * n + 1][0], pr[2 * n + 1][1]};
            const int row = key0 + n * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
            const uint32_t at_row = vs + row * 128;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              uint32_t f[4];
              ldmatrix4_trans(at_row + (d >> 2) * C::kSlab + ((((2 * d + (lane >> 4)) & 7) ^ (row & 7)) << 4), f);
              mma16816(o[2 * d], w, f[0], f[1]);
              mma16816(o[2 * d + 1], w, f[2], f[3]);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[stage]);
        }
        if (++stage == C::kStages) {
          stage = 0;
          use ^= 1;
        }
      }
      // join the warps that shared the keys, 32 columns at a time
      const bool whole = !kCluster && tile == 0 && to == s.tiles;
      if (whole && row_blocks > 0 && threadIdx.x == 0) sc.joins[(seg * p.kv_heads + b.kv_head) * row_blocks + b.row0 / R].parts = 0;
      const int slot = 2 * cta + (first_block ? 0 : 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float row_sum = quad_sum(l[h]);
        if ((lane & 3) == 0) s_ml[wn * R + 16 * wm + (lane >> 2) + 8 * h] = ok ? make_float2(m[h], row_sum) : lost_state();
      }
#pragma unroll
      for (int x = 0; x < D / kColumns; ++x) {
#pragma unroll
        for (int i = 0; i < kColumns / 8; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(s_join + (wn * R + 16 * wm + (lane >> 2) + 8 * h) * kPitch + 8 * i + 2 * (lane & 3)) =
                make_float2(o[x * (kColumns / 8) + i][2 * h], o[x * (kColumns / 8) + i][2 * h + 1]);
        math_warps_sync<kMathWarps * 32>();
#pragma unroll 1
        for (int u0 = 0; u0 < b.rows * (kColumns / 4); u0 += kMathWarps * 32) {
          const int u = u0 + static_cast<int>(threadIdx.x), r = u / (kColumns / 4), col = u % (kColumns / 4) * 4;
          float2 ml[WN];                      // (of rows that there are not too: r is below R)
#pragma unroll
          for (int w = 0; w < WN; ++w) ml[w] = s_ml[w * R + r];
          float mm = -INFINITY, least = 0.f;
#pragma unroll
          for (int w = 0; w < WN; ++w) {
            mm = fmaxf(mm, ml[w].x);
            least = fminf(least, ml[w].y);
          }
          const bool lost = is_lost(least), there = r < b.rows && !(whole && lost);
          const uint32_t mask = __ballot_sync(0xffffffffu, there);
          if (!there) continue;
          const float ref = reference(mm);
          float ll = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WN; ++w) {
            const float f = ex2((ml[w].x - ref) * c);
            const float4 v = *reinterpret_cast<const float4*>(s_join + (w * R + r) * kPitch + col);
            ll = fmaf(ml[w].y, f, ll);
            acc.x = fmaf(v.x, f, acc.x);
            acc.y = fmaf(v.y, f, acc.y);
            acc.z = fmaf(v.z, f, acc.z);
            acc.w = fmaf(v.w, f, acc.w);
          }
          const bool last = x == D / kColumns - 1 && col == 0;
          if (whole) {
            const int row = b.row0 + r;
            store_row4<D>(p, seg, s.w.q_begin, row / group, b.kv_head * group + row % group, x * kColumns + col, acc, lse_of(p, mm, ll), ll, last, mask);
          } else if (kCluster) {
            *reinterpret_cast<float4*>(s_state + r * D + x * kColumns + col) = acc;
            if (last) s_state_ml[r] = lost ? lost_state() : make_float2(mm, ll);
          } else {
            *reinterpret_cast<float4*>(sc.o + (static_cast<int64_t>(slot) * R + r) * D + x * kColumns + col) = acc;
            if (last) sc.ml[static_cast<int64_t>(slot) * R + r] = lost ? lost_state() : make_float2(mm, ll);
          }
        }
        math_warps_sync<kMathWarps * 32>();
      }
      next_block();
    }
  }
  if (!ok) __nanosleep(1000000);           // let copies in flight land  (a warp whose waits were all met has met all of its CTA's loads)
  if constexpr (kCluster) {
    // the CTAs' states, four columns of a row per thread, the rows dealt out over the cluster
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int ranks = static_cast<int>(cluster.num_blocks());
    const Block b = make_block<R>(p, s, unit0);
    const float c = p.f.scale_log2;
    for (int u = static_cast<int>(cluster.block_rank()) * kThreads + threadIdx.x; u < b.rows * (D / 4); u += ranks * kThreads) {
      const int r = u / (D / 4), col = u % (D / 4) * 4;
      // (all reads of the other CTAs' memory are under way before one is used)
      float2 ml[kMostCluster];
      float4 v[kMostCluster];
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < ranks) {
          ml[i] = cluster.map_shared_rank(s_state_ml, i)[r];
          v[i] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(s_state, i) + r * D + col);
        }
      }
      float mm = -INFINITY, ll = 0.f;
      float least = 0.f;
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) {
        mm = fmaxf(mm, ml[i].x);
        least = fminf(least, ml[i].y);
      }
      const float ref = reference(mm);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) {
        const float f = ex2((ml[i].x - ref) * c);
        ll = fmaf(ml[i].y, f, ll);
        acc.x = fmaf(v[i].x, f, acc.x);
        acc.y = fmaf(v[i].y, f, acc.y);
        acc.z = fmaf(v[i].z, f, acc.z);
        acc.w = fmaf(v[i].w, f, acc.w);
      }
      const int row = b.row0 + r;
      if (!is_lost(least))
        store_row4<D>(p, seg, s.w.q_begin, row / s.group, b.kv_head * s.group + row % s.group, col, acc, lse_of(p, mm, ll), ll, col == 0,
                      D == 128 ? 0xffffffffu : 0xffffu << (lane & 16));
    }
    cluster.sync();                         // nobody leaves while its shared memory is read
  }
}

// Joins the parts of a block that several CTAs worked on.  grid: (blocks, or boundaries between two of `ctas` shares; CTAs to the rows of one).
// A lane has D / 32 columns; the four warps have a row each, or share the parts of one where there are many.
template <int D, int R>
__global__ void __launch_bounds__(128) flash_paged_join_kernel(const __grid_constant__ PagedParams p, void* scratch, int ctas, int row_blocks) {
  constexpr int kCols = D / 32;
  __shared__ float s_acc[4][D];
  __shared__ float s_sum[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Scratch<D, R> sc(scratch, ctas);
  const int group = p.f.num_heads / p.kv_heads;
  const float c = p.f.scale_log2;
  // (a block that its sequence has not is nobody's, and its record nothing)
  const bool there = row_blocks == 0 || static_cast<int>(blockIdx.x) % row_blocks < make_seq<R>(p, static_cast<int>(blockIdx.x) / row_blocks / p.kv_heads).blocks;
  grid_dependency_wait();
  const int status = *reinterpret_cast<volatile int*>(p.f.status);
  const Join j = sc.joins[blockIdx.x + (row_blocks == 0 ? 1 : 0)];
  if (status != 0 || !there) return;
  auto slot_of = [&](int i) { return static_cast<int64_t>(2 * (j.cta + i) + (i == 0 ? j.late : 0)) * R; };
  if (j.parts == 0) return;
  const int per_row = j.parts <= 16 ? 1 : 4;                                // warps
  const int part = warp % per_row, step = 4 / per_row;                      // ... and rows of a CTA at a time
  for (int r0 = blockIdx.y * step; r0 < j.rows; r0 += gridDim.y * step) {
    const int r = min(r0 + warp / per_row, j.rows - 1);                     // (a warp without a row does the last one once more)
    float mm = -INFINITY, sum = 0.f, acc[kCols] = {};
    bool lost = false;
    for (int i = lane; i < j.parts; i += 32) {
      const float2 ml = sc.ml[slot_of(i) + r];
      mm = fmaxf(mm, ml.x);
      lost = lost || is_lost(ml.y);
    }
    constexpr int kAhead = 8;
    for (int i0 = part; i0 < j.parts; i0 += per_row * kAhead) {
      // (all reads are under way before one is used)
      float2 ml[kAhead];
      float v[kAhead][kCols];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t at = slot_of(min(i0 + per_row * u, j.parts - 1)) + r;
        ml[u] = sc.ml[at];
        const float* src = sc.o + at * D + lane * kCols;
        if constexpr (D == 128) {
          const float4 q = *reinterpret_cast<const float4*>(src);
          v[u][0] = q.x, v[u][1] = q.y, v[u][2] = q.z, v[u][3] = q.w;
        } else {
          const float2 q = *reinterpret_cast<const float2*>(src);
          v[u][0] = q.x, v[u][1] = q.y;
        }
      }
      if (i0 == part) {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
        lost = __any_sync(0xffffffffu, lost);
      }
      const float ref = reference(mm);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i0 + per_row * u >= j.parts) break;
        const float f = ex2((ml[u].x - ref) * c);
        sum = fmaf(ml[u].y, f, sum);
#pragma unroll
        for (int k = 0; k < kCols; ++k) acc[k] = fmaf(v[u][k], f, acc[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kCols; ++k) s_acc[warp][lane * kCols + k] = acc[k];
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (r0 + warp / per_row < j.rows && part == 0 && lane < D / 4 && !lost) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
      for (int w = warp; w < warp + per_row; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(&s_acc[w][lane * 4]);
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
        l += s_sum[w];
      }
      const int row = j.row0 + r;
      store_row4<D>(p, j.seg, j.q_begin, row / group, j.kv_head * group + row % group, lane * 4, a, lse_of(p, mm, l), l, lane == 0, D == 128 ? 0xffffffffu : 0xffffu);
    }
    __syncthreads();
  }
}

// Joins the parts of blocks whose keys the kernel of tiles split: normalised values and lse of each, 256 rows apart.  grid: (blocks, CTAs to a block's rows),
// a warp per row.
template <int D>
__global__ void __launch_bounds__(256) flash_tile_join_kernel(const __grid_constant__ PagedParams p) {
  constexpr int kCols = D / 32, kAhead = 8;
  __shared__ float s_row[8][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  const int status = *reinterpret_cast<volatile int*>(p.f.status);
  const TileJoin j = p.joins[blockIdx.x];
  if (status != 0) return;
  for (int r = blockIdx.y * 8 + warp; r < j.rows; r += gridDim.y * 8) {
    const float* o = static_cast<const float*>(p.parts.out) + (static_cast<int64_t>(j.state) * 256 + r) * D + lane * kCols;
    const float* lse = p.parts.lse + static_cast<int64_t>(j.state) * 256 + r;
    float top = -INFINITY, sum = 0.f, acc[kCols] = {};
    for (int i = lane; i < j.parts; i += 32) top = fmaxf(top, lse[i * 256]);
    for (int i0 = 0; i0 < j.parts; i0 += kAhead) {
      // (all reads are under way before one is used)
      float l[kAhead], v[kAhead][kCols];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t i = min(i0 + u, j.parts - 1);
        l[u] = lse[i * 256];
        if constexpr (D == 128) {
          const float4 q = *reinterpret_cast<const float4*>(o + i * 256 * D);
          v[u][0] = q.x, v[u][1] = q.y, v[u][2] = q.z, v[u][3] = q.w;
        } else {
          const float2 q = *reinterpret_cast<const float2*>(o + i * 256 * D);
          v[u][0] = q.x, v[u][1] = q.y;
        }
      }
      if (i0 == 0) {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      }
      const float ref = reference(top);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i0 + u >= j.parts) break;
        const float f = __expf(l[u] - ref);
        sum += f;
#pragma unroll
        for (int k = 0; k < kCols; ++k) acc[k] = fmaf(v[u][k], f, acc[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kCols; ++k) s_row[warp][lane * kCols + k] = acc[k];
    __syncwarp();
    if (lane < D / 4)
      store_row4<D>(p, j.seg, j.q_begin >> p.pack_shift, (j.q0 + r) >> p.pack_shift, (j.head << p.pack_shift) + ((j.q0 + r) & ((1 << p.pack_shift) - 1)), lane * 4,
                    *reinterpret_cast<const float4*>(&s_row[warp][lane * 4]),
                    top + __logf(sum), sum, lane == 0, D == 128 ? 0xffffffffu : 0xffffu);
    __syncwarp();
  }
}

template <int D>
cudaError_t launch_tile_join(const PagedParams& p, cudaStream_t stream) {
  return launch_attention_kernel(flash_tile_join_kernel<D>, dim3(p.most_states / 2, 8), 256, 0, stream, true, p);
}
template cudaError_t launch_tile_join<64>(const PagedParams&, cudaStream_t);
template cudaError_t launch_tile_join<128>(const PagedParams&, cudaStream_t);

// A cluster to each block, or all blocks shared out: what is expected to finish first, where all CTAs of the clusters can run at once.  A CTA alone on
// its SM takes 0.47 us for a tile at D = 64 and 0.62 at D = 128, over pages of 16 tokens, whose loads are small, 0.69 and 0.97 (the rule has what lies
// between); sharing out and joining take 3.5 us, and lengths that the host does not know are taken to be two thirds of the longest on average.  us, clusters /
// shared out, sequences of one length, pages of 64:
//   keys                              200        1500        4000        8000        16000       32000       64000
//   1 x 8 heads over 1 of 64       6.0/8.0    6.8/9.0     9.2/8.4    12.8/9.2    20.9/11.3   36.3/16.6   67.0/17.8
//   1 x 32 over 8 of 64            6.2/8.2    6.7/8.9     9.0/9.3    12.7/11.1   21.7/13.7   37.5/20.4   68.8/31.7
//   4 x 32 over 8 of 64            6.2/8.8    7.5/10.3   11.1/13.9   16.8/19.9   25.9/30.5   44.7/50.9   81.9/90.7
//   1 x 32 over 8 of 128           6.9/9.0    7.7/10.2   10.8/10.4   16.4/15.1   26.8/21.6   46.5/31.6   85.7/51.4
//   1 x 24 over 24 of 128          7.0/9.6    8.3/11.7   14.6/18.4   21.7/25.8   35.2/40.2   62.6/70.0    117/127
//   3 x 8 over 2 of 128            6.9/9.1    7.7/9.9    10.8/10.5   15.9/12.9   26.6/18.8   46.5/26.6   85.6/41.7
// ... and over pages of 16, at 1500, 4000 and 8000 keys: the second 7.0/8.9, 10.4/9.4, 15.8/11.7, the third 7.9/10.6, 11.9/14.9, 18.1/19.8, the fourth
// 8.4/10.4, 13.0/10.8, 21.3/14.9.  The two thirds cost sequences of one length: the third row's last three are shared out, 11 to 18 % above clusters.
PagedRowsPlan plan_paged_rows(int64_t rows_of_a_head, int64_t keys, int64_t kv_heads, int64_t nseg, int head_dim, int sm_count) {
  PagedRowsPlan plan = {};
  // As few blocks as there can be, and of these the smallest, three warps instead of four.  (us, blocks of 64 and of 48: seven sequences of 5003 to 20011
  // keys, 32 heads over 4 of 64 / 128, five queries 35.5 / 60.2 and 32.7 / 46.8, eight to twelve 51.6 / 89.3 and 45.6 / 68.9.)
  const int64_t r = rows_of_a_head;
  plan.rows = r <= 16 ? 16 : r <= 32 ? 32 : r <= 48 || (r > 64 && r <= 96) ? 48 : 64;
  const int64_t resident = 2 * sm_count, tiles = keys / kKeys + 1;
  plan.row_blocks = static_cast<int>((rows_of_a_head + plan.rows - 1) / plan.rows);
  const int64_t units = plan.row_blocks * kv_heads * nseg;
  int ranks = kMostCluster;
  while (ranks > 1 && (units * ranks > resident || tiles < 2 * ranks)) ranks /= 2;
  const double tile = head_dim == 64 ? 0.55 : 0.8, hbm = static_cast<double>(units * tiles) * kKeys * head_dim * 4 / 6.6e6;
  const double alone = 5.6 + std::max(tile * ((tiles + ranks - 1) / ranks), hbm);
  const double shared = 9. + 1.1 * (nseg > 1 ? 0.65 : 1.) * std::max(tile * units * (tiles + kBlockCost) / resident, hbm);
  if (units * ranks <= resident && alone < shared) {
    plan.cluster = ranks;
    plan.ctas = static_cast<int>(units * ranks);
    return plan;
  }
  const int64_t useful = units * (tiles + 1 + kBlockCost) / kMinPlaces;
  plan.ctas = static_cast<int>(useful < 2 ? 2 : useful < resident ? useful : resident);
  plan.scratch_bytes = plan.ctas * (static_cast<int64_t>(sizeof(Join)) + 2 * plan.rows * (8 + head_dim * 4));
  return plan;
}

namespace {

template <int D, int WM, bool kCluster>
cudaError_t launch_rows(const PagedMap& tk, const PagedMap& tv, const PagedParams& p, const PagedRowsPlan& plan, void* scratch, cudaStream_t stream) {
  using C = Cfg<D, WM>;
  const auto kernel = flash_paged_rows_kernel<D, WM, kCluster>;
  static bool configured[64] = {};
  static std::mutex mu;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!configured[dev & 63]) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
      if (e != cudaSuccess) return e;
      configured[dev & 63] = true;
    }
  }
  if constexpr (kCluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.ctas);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = plan.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, tk, tv, p, scratch, plan.row_blocks);
  }
  // Joins by blocks where they are fewer; rows beside one another as far as the launch stays small, for 1000 CTAs of nothing take 0.75 us and the rows of
  // a CTA 1.5 each.  (us, by boundaries and by blocks: five queries as above 32.5 and 28.7, of one sequence 23.6 and 17.2; 24 tokens 108.5 and 105.5; a
  // token of 8 heads over one of 64 against 60000 keys, 296 parts of one block, 19.1 and 20.4.)
  const int64_t units = static_cast<int64_t>(plan.row_blocks) * p.kv_heads * p.f.nseg;
  const bool by_blocks = units < plan.ctas;
  const int row_blocks = by_blocks ? plan.row_blocks : 0;
  const unsigned joins = by_blocks ? static_cast<unsigned>(units) : plan.ctas - 1;
  const unsigned rows = by_blocks ? static_cast<unsigned>(std::clamp<int64_t>(2048 / units, 4, 16 * WM)) : WM == 1 ? 8 : 16;
  kernel<<<plan.ctas, C::kThreads, C::kBytes, stream>>>(tk, tv, p, scratch, row_blocks);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_attention_kernel(flash_paged_join_kernel<D, 16 * WM>, dim3(joins, rows), 128, 0, stream, true, p, scratch, plan.ctas, row_blocks);
}
template <int D, int WM>
cudaError_t launch_rows(const PagedMap& tk, const PagedMap& tv, const PagedParams& p, const PagedRowsPlan& plan, void* scratch, cudaStream_t stream) {
  return plan.cluster > 0 ? launch_rows<D, WM, true>(tk, tv, p, plan, scratch, stream) : launch_rows<D, WM, false>(tk, tv, p, plan, scratch, stream);
}

}  // namespace

template <int D>
cudaError_t launch_paged_rows(const PagedMap& tk, const PagedMap& tv, const PagedParams& p, const PagedRowsPlan& plan, void* scratch, cudaStream_t stream) {
  if (plan.rows == 16) return launch_rows<D, 1>(tk, tv, p, plan, scratch, stream);
  if (plan.rows == 32) return launch_rows<D, 2>(tk, tv, p, plan, scratch, stream);
  if (plan.rows == 48) return launch_rows<D, 3>(tk, tv, p, plan, scratch, stream);
  return launch_rows<D, 4>(tk, tv, p, plan, scratch, stream);
}

template cudaError_t launch_paged_rows<64>(const PagedMap&, const PagedMap&, const PagedParams&, const PagedRowsPlan&, void*, cudaStream_t);
template cudaError_t launch_paged_rows<128>(const PagedMap&, const PagedMap&, const PagedParams&, const PagedRowsPlan&, void*, cudaStream_t);

}  // namespace dtb
