// Attention over keys and values that lie in pages: what the kernels are given (flash_paged_rows.cu for few query rows, flash_window_sm100.cu
// for many), and how a sequence's keys are found.
//
// Page n of a pool holds P tokens (a power of two, at least 16); key j of sequence b is token j % P of page table[b][j / P].  A page number
// outside the pool stands for keys and values of 0.
#pragma once
#include "flash_common.cuh"
#include "flash_window.cuh"

namespace dtb {

// The kernel of tiles takes the rows of 1 << pack_shift query heads that share a key head as those of one: row r of a sequence is query
// r >> pack_shift and head (r & ((1 << pack_shift) - 1)) of them.  Its f.num_heads, f.seqlen_q and f.total_q count so; `real` does not.
// (A tile of keys is loaded once for these heads, and a few queries of many heads fill its rows.  us, one launch after another, heads apart and together:
// chunks and tokens mixed, 32 heads over 8, 841 -> 752; 45 queries of 16 heads to a key head against 15369 keys of 15 sequences 821 -> 253.)
struct PagedParams : WindowParams {    // (k, v, their strides, cu_k and k_start are not used; seqlens_k is given always)
  int pack_shift;
  FlashParams real;
  const int32_t* table;                // [sequences, columns]
  int columns, pages, page_shift;
  int box_rows;                        // tokens of a tile that one load fetches; divides a page, so that no load crosses one
  int key_align;                       // runs of keys are walked from a multiple of this
  int few_rows;                        // the kernel of few rows takes the sequences with at most this many queries, that of many the others
  // of the kernel of tiles:
  int planned;                         // whether plan_blocks orders them; 0: as they come, row block, head, sequence, the first of them changing fastest
  int blocks;                          // of the grid
  int ctas;                            // that run at once
  int most_states;                     // of parts, or 0: keys are not split
  FlashParams parts;                   // where those go, 256 rows each, ...
  struct TileJoin* joins;              // ... and the blocks they are of, for the launch that joins them: [most_states / 2]
};

// A block whose keys were split.
struct alignas(16) TileJoin {
  int seg, head, q0, rows;             // rows 0: no block
  int q_begin, state, parts, pad;      // its first part's state, and how many there are
};

// A tensor map of the pool [channel, token, head, page] (head before token where heads are nearer to one another), with what its loads go by.
struct alignas(64) PagedMap {
  CUtensorMap map;
  int dim_shift;           // head_dim = 1 << dim_shift
};

// Runs of keys begin where the loads of a tile can: at a multiple of 16 tokens, or of whole tiles where no window moves them.
__device__ __forceinline__ int key_align(const PagedParams& p) { return p.key_align; }
template <class Walk>
__device__ __forceinline__ int front_of(const PagedParams&, const Walk& w) { return w.front; }

__device__ __forceinline__ int paged_keys(const PagedParams& p, int seg) { return max(min(p.seqlens_k[seg], p.columns << p.page_shift), 0); }

// A sequence.  Its keys are numbered through all sequences, seg * columns * P + j.
__device__ __forceinline__ WindowSeq paged_seq(const PagedParams& p, int seg) {
  WindowSeq s;
  const int longest = p.f.seqlen_q >> p.pack_shift;
  s.q_begin = 0;
  int rows = longest;
  if (p.f.cu_q != nullptr) {
    // (what offsets say beyond the rows that there are is not followed)
    const int total = static_cast<int>(p.f.total_q >> p.pack_shift);
    s.q_begin = min(max(p.f.cu_q[seg], 0), total);
    rows = max(min(max(p.f.cu_q[seg + 1], 0), total) - s.q_begin, 0);
  }
  s.q_len = min(rows, longest);          // (the rows that are kept stay where they are: the last one of all is at the last key)
  s.k_begin = seg * (p.columns << p.page_shift);
  s.k_len = paged_keys(p, seg);
  const int64_t x = static_cast<int64_t>(s.k_len) - rows;
  s.from = p.left < 0 ? -kFar : clamp_position(x - p.left);
  s.to = p.right < 0 ? kFar : clamp_position(x + p.right + 1);
  s.sinks = max(min(p.sinks, s.k_len), 0);
  return s;
}
__device__ __forceinline__ WindowSeq window_seq(const PagedParams& p, int seg) {
  WindowSeq s = paged_seq(p, seg);
  if (s.q_len <= p.few_rows) s.q_len = 0;
  s.q_begin <<= p.pack_shift;
  s.q_len <<= p.pack_shift;
  return s;
}
__device__ __forceinline__ int row_shift(const PagedParams& p) { return p.pack_shift; }

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, int a, int b, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(a), "r"(b), "r"(page)
      : "memory");
}

__device__ __forceinline__ void st_relaxed16(void* to, int a, int b, int c, int d) {
  asm volatile("st.relaxed.gpu.global.v4.s32 [%0], {%1, %2, %3, %4};" ::"l"(to), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void prefetch_tmap(const PagedMap* m) { prefetch_tmap(&m->map); }

// A tensor map of the queries [channel, head, token, batch] (batch before token where that has the smaller stride); a box is 64 channels of
// the rows of a tile, that is, of 1 << pack_shift heads of 128 >> pack_shift tokens.
struct alignas(64) QueryMap {
  CUtensorMap map;
  int dim_shift, pack_shift;
};
__device__ __forceinline__ void prefetch_tmap(const QueryMap* m) { prefetch_tmap(&m->map); }
__device__ __forceinline__ void tma_load_token(void* smem_dst, const QueryMap* m, uint64_t* bar, int x, int row, int batch, int batch_first) {
  const int token = row >> m->pack_shift;
  tma_load_4d(smem_dst, &m->map, bar, x & ((1 << m->dim_shift) - 1), (x >> m->dim_shift) << m->pack_shift, batch_first ? batch : token, batch_first ? token : batch);
}

// Loads of tiles over pages.  The thread that walks a block's tiles asks for them, and two warps that have no other role look the pages up and
// issue the loads, a lane to each 64 channels of a box.  (One thread that does all of it is what bounds a launch: 16 loads of 2 KB and 8
// look-ups for a tile at D = 128 and pages of 16, which a step of 1.6 us takes two of.)  A request's place in the queue is taken again only
// when the tile's slot in the ring is, that is, after its loads have landed: there are more places than loads in the ring (checked where the ring's size is
// known), and nothing to wait for.
// (us, from a graph, one thread and two warps: two CogVideoX frames over pages of 64 770 -> 654, as dense keys 637; chunks and tokens over pages of 16
// mixed 1297 -> 924.)
constexpr int kLoadPlaces = 16;
constexpr int kLoadWarps = 2;            // they take requests in turn
struct LoadRequest {
  const PagedMap* map;                   // null: no more
  uint64_t* bar;
  uint8_t* dst;
  int token, head, head_first;
};
struct LoadQueue {
  LoadRequest at[kLoadPlaces];
  uint64_t posted[kLoadPlaces];          // barriers: a request is there
  uint32_t n;                            // requests so far, of the thread that asks
};
__device__ __forceinline__ LoadQueue& load_queue() {
  __shared__ LoadQueue queue;
  return queue;
}
__device__ __forceinline__ void post_load(const LoadRequest& r) {
  LoadQueue& q = load_queue();
  const uint32_t i = q.n++ % kLoadPlaces;
  q.at[i] = r;
  mbar_arrive(&q.posted[i]);
}

// The first 64 channels' call asks for all of a tile: 128 tokens from `token` (counted through all sequences, a multiple of the box).
__device__ __forceinline__ void tma_load_token(void* smem_dst, const PagedMap* m, uint64_t* bar, int x, int token, int /*batch*/, int head_first) {
  if ((x & ((1 << m->dim_shift) - 1)) == 0) post_load(LoadRequest{m, bar, static_cast<uint8_t*>(smem_dst), token, x >> m->dim_shift, head_first});
}

// What the kernel of tiles does for its loads beside its loader: nothing where keys are dense.
__device__ __forceinline__ void init_loads(const WindowParams&) {}
__device__ __forceinline__ void end_loads(const WindowParams&) {}
template <int D>
__device__ __forceinline__ void serve_loads(const WindowParams&, int) {}

__device__ __forceinline__ void init_loads(const PagedParams&) {         // by one thread
  LoadQueue& q = load_queue();
  q.n = 0;
  for (int i = 0; i < kLoadPlaces; ++i) mbar_init(&q.posted[i], 1);
}
__device__ __forceinline__ void end_loads(const PagedParams&) {          // by the thread that asks
  for (int i = 0; i < kLoadWarps; ++i) post_load(LoadRequest{nullptr, nullptr, nullptr, 0, 0, 0});
}
// By a whole warp, the `which`th of them.  What lies behind the table's last column, or in a page outside the pool, is filled with zeros by the
// load (its page number is one past the last).
template <int D>
__device__ __forceinline__ void serve_loads(const PagedParams& p, int which) {
  constexpr int kSlabs = D / 64;
  LoadQueue& q = load_queue();
  const int lane = threadIdx.x & 31, slab = lane % kSlabs, at = lane / kSlabs * p.box_rows;       // this lane's box begins at that token
  const int span = p.columns << p.page_shift;
  for (uint32_t n = which;; n += kLoadWarps) {
    const uint32_t i = n % kLoadPlaces;
    if (!flash::warp_wait_or_abort(&q.posted[i], (n / kLoadPlaces) & 1, p.f.status, 16)) break;
    const LoadRequest r = q.at[i];
    if (r.map == nullptr) break;
    if (at < 128) {
      const int seq = r.token / span, pos = r.token - seq * span + at, j = pos >> p.page_shift;
      int page = -1;
      if (j < p.columns) page = p.table[static_cast<int64_t>(seq) * p.columns + j];
      if (page < 0 || page >= p.pages) page = p.pages;
      const int in_page = pos & ((1 << p.page_shift) - 1);
      tma_load_4d(r.dst + slab * (128 * 128) + at * 128, &r.map->map, r.bar, slab * 64, r.head_first ? r.head : in_page, r.head_first ? in_page : r.head, page);
    }
    __syncwarp();
  }
}

// The blocks of 256 rows of one head that the kernel of tiles takes, in the order in which its CTAs claim them: the sequences with the longest
// walks over keys first, so that short ones fill the end; of a sequence one head after another, whose row blocks read the same keys,
// the end whose rows see more keys first.  Where blocks are fewer than CTAs, or the last round
// of them is far from full, keys are split:
//   - less work than a block of the longest kind for every CTA: all of it into parts of about an even share,
//   - a last round that wastes more than 15 %: the blocks of the last half a round in two.
// Every CTA plans for itself, from lengths that stand on the device.
// Batches of more sequences than there is room for are taken as they come, and no keys are split: of each round of as many blocks as CTAs every CTA has one,
// the next place's in the next round (for sequences alike a place would always be the same row block).  (The host knows the longest sequence's blocks alone;
// a grid with as many for each, claimed one by one, is mostly blocks that there are not.  us, that and this: 300 streams, a prompt of 8192 and tokens, 32
// heads over 8 of 128, 2100 and 862; 16384 streams, 2000 rows and tokens, heads of 64, 20485 and 1808; 400 chunks of 200 rows 1845 and 1692.)
constexpr int kPlanSeqs = 256;
constexpr int kPlanBlocks = 1 << 22;     // sums of them are exact in fp32
constexpr int kPlanThreads = 512;
constexpr int kBlockSteps = 5;           // what a block costs beside its steps of 128 keys, in such steps
struct TilePlan {
  int seqs, blocks, splits;              // sequences; places of blocks and parts; blocks that are split
  uint16_t seq[kPlanSeqs];               // in their order
  uint16_t parts[kPlanSeqs];             // of each of a sequence's blocks from `whole` on
  int row_blocks[kPlanSeqs];             // of each head; negative: the last one first
  int whole[kPlanSeqs];
  int first[kPlanSeqs], first_split[kPlanSeqs], first_state[kPlanSeqs];      // places, split blocks and states in front of it
  // ... or, of sequences as they come:
  int before[kPlanThreads];              // blocks in front of each thread's run of sequences
  int round, turn;                       // blocks of the rounds before, and this CTA's place in this one, of the thread that walks the blocks
};
__device__ __forceinline__ TilePlan& tile_plan() {
  __shared__ TilePlan plan;
  return plan;
}

// The row block that a sequence's block i, counted through its heads, is.
__device__ __forceinline__ int row_block_of(const TilePlan& plan, int seq, int i) {
  const int n = plan.row_blocks[seq];
  return n > 0 ? i % n : -n - 1 - i % -n;
}

// Steps of 128 keys that the queries i0 to i1 walk.
__device__ __forceinline__ int block_steps(const WindowSeq& s, int i0, int i1) {
  const WindowSpan a = window_span(s, i0), z = window_span(s, i1);
  const int lo = max(a.lo, min(s.sinks, z.hi));
  return (max(z.hi - lo, 0) + 127) / 128 + (z.first + 127) / 128;
}

// Sum over the 512 threads, and over those before this one.
template <class T>
__device__ __forceinline__ T plan_sum(T v, T& before) {
  __shared__ T s_warp[kPlanThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T upto = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const T u = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += u;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = upto;
  __syncthreads();
  T all = 0;
  before = upto - v;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  return all;
}

// Threads have runs of that many sequences, and a sequence that many blocks, where they are taken as they come.
__device__ __forceinline__ int run_of_sequences(const PagedParams& p) { return (p.f.nseg + kPlanThreads - 1) / kPlanThreads; }
__device__ __forceinline__ int row_blocks_of(const PagedParams& p, int seg) { return (window_seq(p, seg).q_len + 255) / 256; }

__device__ __forceinline__ void plan_blocks(const WindowParams&) {}
// By all threads.  (Sums are of whole numbers below 2^24 or of estimates: fp32 does.)
__device__ __forceinline__ void plan_blocks(const PagedParams& p) {
  TilePlan& plan = tile_plan();
  const int n = p.f.nseg, t = threadIdx.x;
  grid_launch_dependents();              // (the launch that joins)
  if (!p.planned) {
    const int per = run_of_sequences(p), b0 = min(t * per, n), b1 = min(b0 + per, n);
    int mine = 0, before;
    for (int b = b0; b < b1; ++b) mine += row_blocks_of(p, b) * p.f.num_heads;      // (fewer than rows, which 31 bits hold)
    const int all = plan_sum(mine, before);
    plan.before[t] = before;
    if (t == 0) {
      plan.blocks = all;
      plan.round = 0;
      plan.turn = static_cast<int>(blockIdx.x);
    }
    return;
  }
  __shared__ int s_steps[kPlanSeqs];
  int blocks = 0, longest = 0, q_len = 0;
  bool rising = false;                   // the last rows walk further than the first
  float steps = 0.f;                     // of a block, on average
  if (t < n) {
    const WindowSeq s = window_seq(p, t);
    q_len = s.q_len;
    blocks = (q_len + 255) / 256;
    if (blocks > 0) {
      const int a = block_steps(s, 0, (min(q_len, 256) - 1) >> p.pack_shift), z = block_steps(s, ((blocks - 1) * 256) >> p.pack_shift, (q_len - 1) >> p.pack_shift);
      longest = max(max(a, z), 1);
      rising = z > a;
      steps = 0.5f * (a + z);
    }
    s_steps[t] = longest;
  }
  __syncthreads();
  int rank = 0;
  if (t < n) {
    for (int i = 0; i < n; ++i) rank += s_steps[i] > longest || (s_steps[i] == longest && i < t);
    plan.seq[rank] = static_cast<uint16_t>(t);
    plan.row_blocks[rank] = rising ? -blocks : blocks;
    plan.first[rank] = longest;
    plan.whole[rank] = __float_as_int(steps);
  }
  __syncthreads();
  if (t < n) {
    blocks = abs(plan.row_blocks[t]);
    longest = plan.first[t];
    steps = __int_as_float(plan.whole[t]);
  }
  const int top = max(plan.first[0], 0) + kBlockSteps;
  const int mine = t < n ? blocks * p.f.num_heads : 0;
  const float each = steps + kBlockSteps;
  float blocks_before, work_before, x;
  const float all = plan_sum(static_cast<float>(mine), blocks_before), work = plan_sum(mine * each, work_before);
  const float share = work / p.ctas;
  int parts = 1, whole = mine;
  if (p.most_states > 0 && share < top) {
    float size = fmaxf(1.15f * share, 6.f);
    for (int round = 0; round < 8; ++round, size *= 1.4f) {
      parts = mine > 0 ? max(1, min(min(static_cast<int>(ceilf(longest / size)), longest / 2), 255)) : 1;
      if (plan_sum(parts > 1 ? static_cast<float>(mine) * parts : 0.f, x) <= p.most_states) break;
      parts = 1;
    }
    whole = parts > 1 ? 0 : mine;
  } else if (p.most_states > 0 && all > p.ctas && ceilf(all / p.ctas) * p.ctas > 1.15f * all) {
    parts = longest + kBlockSteps > 0.5f * top && longest >= 4 ? 2 : 1;
    if (parts > 1) whole = max(0, min(mine, static_cast<int>(ceilf((work - 0.5f * top * p.ctas - work_before) / each))));
    if (plan_sum(parts > 1 ? 2.f * (mine - whole) : 0.f, x) > p.most_states) whole = mine;
  }
  if (whole == mine) parts = 1;
  const int split = mine - whole;
  float split_before, state_before, first_before;
  const float splits = plan_sum(static_cast<float>(split), split_before);
  plan_sum(static_cast<float>(split) * parts, state_before);
  const float places = plan_sum(static_cast<float>(whole + split * parts), first_before);
  if (t < n) {
    plan.parts[t] = static_cast<uint16_t>(parts);
    plan.whole[t] = whole;
    plan.first[t] = static_cast<int>(first_before);
    plan.first_split[t] = static_cast<int>(split_before);
    plan.first_state[t] = static_cast<int>(state_before);
  }
  if (t == 0) {
    plan.seqs = n;
    plan.blocks = static_cast<int>(places);
    plan.splits = static_cast<int>(splits);
  }
  __syncthreads();
  // Every CTA leaves what the launch that joins has to know, all of them the same: none is sure to start, since a CTA that runs may take over the block of one
  // that has not begun, whichever that is.
  if (p.most_states > 0) {
    for (int i = t; i < p.most_states / 2; i += kPlanThreads) {
      TileJoin j = {0, 0, 0, 0, 0, 0, 0, 0};
      if (i < plan.splits) {
        int b = 0, end = n;
        while (end - b > 1) {
          const int mid = (b + end) >> 1;
          if (plan.first_split[mid] <= i) b = mid; else end = mid;
        }
        const int k = i - plan.first_split[b], block = plan.whole[b] + k;
        const WindowSeq s = window_seq(p, plan.seq[b]);
        j.seg = plan.seq[b];
        j.head = block / abs(plan.row_blocks[b]);
        j.q0 = row_block_of(plan, b, block) * 256;
        j.rows = min(256, s.q_len - j.q0);
        j.q_begin = s.q_begin;
        j.state = plan.first_state[b] + k * plan.parts[b];
        j.parts = plan.parts[b];
      }
      st_relaxed16(&p.joins[i].seg, j.seg, j.head, j.q0, j.rows);
      st_relaxed16(&p.joins[i].q_begin, j.q_begin, j.state, j.parts, 0);
    }
  }
}

__device__ __forceinline__ void place_block(const PagedParams& p, int& bx, int& by, int& bz, int& splits, int& state) {
  const TilePlan& plan = tile_plan();
  int i = bx;
  splits = 1;
  state = -1;
  if (i >= plan.blocks) {              // (the grid has room for more than there may be)
    bx = 1 << 22;
    by = bz = 0;
    return;
  }
  if (!p.planned) {
    int lo = 0, hi = kPlanThreads;     // the last run that begins at or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (plan.before[mid] <= i) lo = mid; else hi = mid;
    }
    i -= plan.before[lo];
    bz = lo * run_of_sequences(p);
    int row_blocks = row_blocks_of(p, bz);
    while (i >= row_blocks * p.f.num_heads && bz + 1 < p.f.nseg) {
      i -= row_blocks * p.f.num_heads;
      row_blocks = row_blocks_of(p, ++bz);
    }
    by = i / row_blocks;
    bx = i % row_blocks;
    return;
  }
  int lo = 0, hi = plan.seqs;          // the last sequence that begins at or before it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (plan.first[mid] <= i) lo = mid; else hi = mid;
  }
  // (sequences without blocks begin where the next one does, behind the others: there is none with blocks behind them)
  i -= plan.first[lo];
  int part = 0;
  if (i >= plan.whole[lo]) {
    const int k = i - plan.whole[lo];
    splits = plan.parts[lo];
    part = k % splits;
    i = plan.whole[lo] + k / splits;
    if (splits > 1) state = plan.first_state[lo] + k;
  }
  by = i / abs(plan.row_blocks[lo]);
  bx = row_block_of(plan, lo, i);
  bz = plan.seq[lo] * splits + part;
}
__device__ __forceinline__ bool claims_blocks(const PagedParams& p) { return p.planned != 0; }
__device__ __forceinline__ bool next_place(const PagedParams&, int& bx) {
  TilePlan& plan = tile_plan();
  const int ctas = static_cast<int>(gridDim.x);
  if (plan.blocks - plan.round <= ctas) return false;
  plan.round += ctas;
  if (++plan.turn == ctas) plan.turn = 0;
  bx = plan.round + plan.turn;
  return bx < plan.blocks;               // (it is the last round)
}
template <class Item>
__device__ __forceinline__ void place_results(const PagedParams&, Item& w, int state) {
  if (state < 0) return;
  w.part = 1;
  w.head = 0;
  w.q_begin = state * 256 - w.q0;
}

// Where row R of a head (of the tile kernel's, counted through all sequences' rows) is in the results.
struct RowPlace {
  const FlashParams& f;
  int shift, head0;                    // first of the heads that share rows

  __device__ __forceinline__ RowPlace(const PagedParams& p, int head) : f(p.real), shift(p.pack_shift), head0(head << p.pack_shift) {}
  __device__ __forceinline__ int head(int64_t R) const { return head0 + (static_cast<int>(R) & ((1 << shift) - 1)); }
  template <int D>
  __device__ __forceinline__ int64_t out(int64_t R) const { return (R >> shift) * f.out_tok_stride + static_cast<int64_t>(head(R)) * D; }
  // `row` of its sequence
  __device__ __forceinline__ int64_t lse(int64_t R, int seg, int row) const { return flash::lse_index(f, seg, head(R), row >> shift, R >> shift); }
};

// The results of a block that sees no key, by one thread, as the dense kernel's write_none.
struct PagedResults {
  const PagedParams& p;
};
template <class Item>
__device__ __forceinline__ PagedResults results_at(const PagedParams& p, const Item&) { return PagedResults{p}; }
template <int D, class Item>
__device__ __forceinline__ void write_none(const PagedResults& r, const Item& w, const uint8_t* zeros) {
  const PagedParams& p = r.p;
  const RowPlace at(p, w.head);
  if (w.part == 0 && p.f.accumulate) return;
  const int size = p.f.out_dtype == 0 ? 4 : 2;
#pragma unroll 1
  for (int i = w.q0; i < min(w.q0 + 256, w.q_len); ++i) {
    const int64_t R = static_cast<int64_t>(w.q_begin) + i;
    if (w.part != 0) {
      p.parts.lse[R] = -INFINITY;
      bulk_store(static_cast<float*>(p.parts.out) + R * D, zeros, D * 4);
    } else {
      p.f.lse[at.lse(R, w.seg, i)] = -INFINITY;
      bulk_store(static_cast<uint8_t*>(p.f.out) + at.out<D>(R) * size, zeros, D * size);
    }
  }
  bulk_store_commit();
}

// The results of a warp's 32 rows, from row `pos` of the sequence: normalised, merged with the state in memory where the launch accumulates,
// stored; a part's state is fp32, 256 rows one after another.  `ready` waits for the rows and gives this lane's reference and sum,
// `read` says that O is not needed any more.  Rows go through shared memory (4 KB of the warp's, 16-byte pieces XOR-swizzled by row), so
// that 8 lanes write 128 contiguous bytes.
template <int D, class Ready, class Read>
__device__ __forceinline__ bool paged_results(const PagedParams& p, bool part, int seg, int head, int pos, int q_begin, int q_len, uint32_t o_taddr, uint8_t* stage,
                                              const Ready& ready, const Read& read) {
  using namespace flash;
  const int lane = threadIdx.x & 31, r0 = lane >> 3, piece = lane & 7, rows = q_len - pos;
  const int64_t R0 = static_cast<int64_t>(q_begin) + pos;
  const RowPlace at(p, head);
  const float c = p.f.scale_log2;
  const bool accumulate = !part && p.f.accumulate != 0;
  const int64_t li = part ? R0 + lane : at.lse(R0 + lane, seg, pos + lane);
  float* lse = part ? p.parts.lse : p.f.lse;
  float lse_old = -INFINITY;
  if (accumulate && lane < rows) lse_old = lse[li];     // under way while the rows are still being computed
  float2 ml;
  if (!ready(ml)) return false;
  // a row that has seen no key is an empty state, and leaves a state that it is folded into as it is (a NaN among its scores is not that)
  float w_new = 0.f, w_old = lse_old != -INFINITY ? 1.f : 0.f, lse_out = lse_old;
  if (ml.y != 0.f) merge_weights(accumulate, lse_old, (ml.x * c + log2f(ml.y)) * kLn2, ml.y, w_new, w_old, lse_out);
  if (lane < rows) lse[li] = lse_out;
  if (!part && p.f.out_dtype != 0) {
    uint16_t* dst = static_cast<uint16_t*>(p.f.out) + piece * 8;
#pragma unroll 1
    for (int x = 0; x < D / 64; ++x) {
      uint32_t row[32];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t v[32];
        tmem_ld32(o_taddr + x * 64 + q * 32, v);
        tmem_wait_ld<32>(v);
#pragma unroll
        for (int i = 0; i < 16; ++i) row[q * 16 + i] = pack_bf16x2(__uint_as_float(v[2 * i]) * w_new, __uint_as_float(v[2 * i + 1]) * w_new);
      }
      if (x == D / 64 - 1) read();
      if (rows <= 0) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(row[4 * i], row[4 * i + 1], row[4 * i + 2], row[4 * i + 3]);
      __syncwarp();
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int r = it * 4 + r0;
        const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
        if (r < rows) *reinterpret_cast<uint4*>(dst + at.out<D>(R0 + r) + x * 64) = v;
      }
      __syncwarp();        // the stage is written again for the next columns
    }
    return true;
  }
  float* dst = static_cast<float*>(part ? p.parts.out : p.f.out) + piece * 4;
#pragma unroll 1
  for (int q = 0; q < D / 32; ++q) {
    uint32_t row[32];
    tmem_ld32(o_taddr + q * 32, row);
    tmem_wait_ld<32>(row);
    if (q == D / 32 - 1) read();
    if (rows <= 0) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
          make_float4(__uint_as_float(row[4 * i]) * w_new, __uint_as_float(row[4 * i + 1]) * w_new, __uint_as_float(row[4 * i + 2]) * w_new,
                      __uint_as_float(row[4 * i + 3]) * w_new);
    __syncwarp();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int r = it * 4 + r0;
      float4 v = *reinterpret_cast<const float4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
      float4* to = reinterpret_cast<float4*>(dst + (part ? (R0 + r) * D : at.out<D>(R0 + r)) + q * 32);
      if (accumulate) {
        const float wo = __shfl_sync(0xffffffffu, w_old, r);
        if (r < rows && wo != 0.f) {
          const float4 old = *to;
          v.x = fmaf(old.x, wo, v.x);
          v.y = fmaf(old.y, wo, v.y);
          v.z = fmaf(old.z, wo, v.z);
          v.w = fmaf(old.w, wo, v.w);
        }
      }
      if (r < rows) *to = v;
    }
    __syncwarp();
  }
  return true;
}

template <int D>
cudaError_t launch_paged_tiles(const QueryMap& tm_q, const PagedMap& tm_k, const PagedMap& tm_v, const PagedParams& p, cudaStream_t stream);
// ... and, behind that launch, the join of the parts of blocks whose keys it split (with p.f as it is in p.real).
template <int D>
cudaError_t launch_tile_join(const PagedParams& p, cudaStream_t stream);

// Few rows: blocks of 16, 32, 48 or 64.  Scratch, where there is a second launch, holds the states of sequences that more than one CTA works on.
struct PagedRowsPlan {
  int rows;                // of a block
  int row_blocks;          // of the longest sequence, for each key head
  int cluster;             // CTAs that share a block; 0: all share all of them, and a second launch joins
  int ctas;                // at most
  int64_t scratch_bytes;
};
// (rows of a key head's longest sequence; `keys` of the longest sequence, about: more CTAs than that needs would not be used)
PagedRowsPlan plan_paged_rows(int64_t rows_of_a_head, int64_t keys, int64_t kv_heads, int64_t nseg, int head_dim, int sm_count);
template <int D>
cudaError_t launch_paged_rows(const PagedMap& tm_k, const PagedMap& tm_v, const PagedParams& p, const PagedRowsPlan& plan, void* scratch, cudaStream_t stream);

}  // namespace dtb
