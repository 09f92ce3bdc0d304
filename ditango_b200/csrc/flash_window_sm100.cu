// Windowed attention of many query rows: the tiles, units and arithmetic of flash_fwd_sm100.cu (256 query rows of one (sequence, head)
// as two Q tiles that share the tensor core, key tiles of 128, one softmax thread per row, P over S in tensor memory) over the key tiles
// that the rows see and no others, by CTAs that stay and take one block of 256 rows after another, as in
// flash_fwd_persistent_sm100.cu.
//
// Warp roles (512 threads, four warpgroups):
//   warps 0-7    softmax, a warpgroup per Q tile; a finished row leaves its reference and sum in shared memory
//   warps 8-11   results: O out of tensor memory, normalisation, merge with the state in global memory, stores
//   warp  12     blocks, their plans, TMA loads; the results of blocks that see no key
//   warp  13     MMA issuer
//   warps 14-15  loads of keys and values in pages; no role where they are dense
//
// Key tiles of a block: N that cover the window [lo, hi) of its rows, the first one beginning at the first key that any of them sees, then
// the tiles that hold the first tokens.  The rows of Q tile 1 are 128 further on than those of Q tile 0, and so are their windows, by
// exactly one key tile: where no end of the sequence cuts them (`skew`), step t pairs (Q tile 0, key tile t) with (Q tile 1, key tile
// t + 1), and each Q tile walks N - 1 tiles in place of N.  Units u = 2 t + i stay in the order they have there; a key tile then serves
// unit 2 t - 1 and unit 2 t in place of 2 t and 2 t + 1, which only moves the places where a new tile is taken from the ring and an
// old one given back: where the tile of a unit differs from that of the unit before it.
//
// P is rounded to bf16 for the product with V (each weight by 2^-8 of itself at most, as in the other attention kernels: tensor cores take it
// in no wider type at this rate); scores, references, sums and O are fp32.  On normal inputs a result in bf16 is then off by 0.0023 of its
// norm, 0.0017 of which is its own rounding.
//
// What a row sees of a tile is one run of its columns (its window, or its first tokens), so the mask is two bounds per row; 32 columns
// that all rows of a warp see are not looked at.  A row may meet tiles of which it sees nothing, or none of which it sees anything:
// its maximum stays -inf, its weights 0.  The last tile of the window and that of the first tokens may hold fewer than 128 keys: their
// PV runs the steps of 16 keys that hold one, and the rows behind the last key, which may hold anything, are cleared in shared memory
// by the thread that loads them, which waits for that one load.
//
// Blocks are short (a window of 2700 keys: 25 steps, 36 us at D = 64), so what happens once per block counts.  The next block's plan is made, its
// queries and first keys loaded and its first scores computed while the softmax warps finish the block before it, and results leave by
// warps of their own.  The grid has a CTA per block, as if all were to run; CTAs claim further blocks by cluster launch control.  Every
// phase of a barrier is over for all that look at it before the next one can complete; see flash_fwd_persistent_sm100.cu.
//
// Measured: 2 x 17776 x 48 x 64, windows of 1350 either way and 226 first tokens, 1655 us (740 TFLOP/s of what the rows see; the ex2 unit 73 %
// busy), 29764 x 24 x 128, windows of 3600 and 256 first tokens, 2250 us (1136; the power cap, and 8 us a block that no product fills).
// With few blocks their keys are split into parts of as many tiles each, which are attended like blocks of their own and merged by the
// state merge's kernel behind this one (24 heads of 128, 64 queries, window 4096: 66 -> 26 us in six parts).
#include "flash_common.cuh"
#include "flash_paged.cuh"
#include "flash_window.cuh"

#include <mutex>
#include <type_traits>

namespace dtb {

namespace {

using namespace flash;

constexpr int kThreads = 512;
constexpr int kRegsLaunch = 128;    // what __launch_bounds__(512, 1) allots; checked before the first launch
constexpr int kOutWarp = 8;         // first of four
constexpr int kTmaWarp = 12;
constexpr int kMmaWarp = 13;
constexpr int kSplit = 64;          // keys of a tile whose probabilities are handed over first
constexpr int kWork = 4;            // blocks under way in a CTA
constexpr int kWorkReaders = 8 + 4 + 1;
constexpr int kClaimAhead = 8;      // steps before a block's last at which the next block is asked for
// Barriers for tiles that are not full, used in turn.  Each such tile takes two ring slots (K, V), so that the loader is never as
// many of them ahead of the issuer as there are barriers, and a phase is over for the issuer before the next one can complete.
constexpr int kTails = 8;

template <int D>
struct Cfg {
  static constexpr int kSlabs = D / 64;
  // registers of a thread of each role (a block of 25 steps the one way and the other: D = 64 35.7 and 36.6 us, D = 128 54.9 and 54.1)
  static constexpr int kRegsSoftmax = D == 64 ? 176 : 160;
  static constexpr int kRegsOutput = D == 64 ? 104 : 128;
  static constexpr int kRegsOther = D == 64 ? 56 : 64;
  static_assert(2 * kRegsSoftmax + kRegsOutput + kRegsOther == 4 * kRegsLaunch, "register split");
  static constexpr int kTileBytes = 128 * D * 2;          // one Q, K or V tile
  static constexpr int kQBufs = D == 64 ? 2 : 1;          // blocks whose queries are in shared memory
  static constexpr int kStages = D == 64 ? 8 : 4;
  static constexpr int kSBufs = (512 - kQT * D) / kBN;
  static constexpr int kStageOut = 4 * 4096;              // 4 KB per result warp
  // barriers: q_full[QB][2], q_empty[QB], kv_full[S], kv_empty[S], s_full[NB], p_lo[NB], p_hi[NB], pv_done[2], o_final[2],
  // o_free[2], ml_full[2], ml_empty[2], work_full[W], work_empty[W], v_tail[T], claim
  static constexpr int kBars = 3 * kQBufs + 2 * kStages + 3 * kSBufs + 10 + 2 * kWork + kTails + 1;
  static constexpr int kSmemBytes = 1024 + (kQBufs * kQT + kStages) * kTileBytes + kStageOut + kQT * kBM * 8 + kWork * 80 + D * 4 + 16 +
                                    kBars * 8 + 16;
  static constexpr uint32_t kTmemCols = 512;
  static constexpr uint32_t kColS = 0;                    // + buffer * 128
  static constexpr uint32_t kColO = kSBufs * kBN;         // + tile * D
  static_assert(kColO + kQT * D <= 512, "tensor memory");
  static_assert(kSmemBytes <= 232448, "shared memory");
  static_assert(2 * kTails > kStages, "barriers for tiles that are not full");
};

// The key tiles of a block's rows and the order in which its units meet them.
struct Walk {
  int lo, win;        // the window's first key and length; with pages it may begin `front` keys, fewer than 16, before the first one seen
  int front;
  int first;          // first tokens
  int N, n;           // tiles of the window, window steps of a Q tile: N, or N - 1 where Q tile 1 is a tile ahead
  int steps;          // steps in all; 0: nothing to see (such a block only the loader meets), -1: no more blocks

  // for the rows i0 to i1
  __device__ __forceinline__ void plan(int from, int to, int sinks, int k_end, int k_floor, int i0, int i1, int align, int shift) {
    auto span = [&](int i) { return window_span(from, to, sinks, k_end, k_floor, i >> shift); };
    const WindowSpan a = span(i0), z = span(i1);
    first = z.first;
    lo = max(a.lo, min(k_floor, z.hi));
    front = z.hi > lo ? lo & (align - 1) : 0;
    lo -= front;
    win = max(z.hi - lo, 0);
    N = (win + kBN - 1) / kBN;
    n = N;
    if (i1 - i0 >= kBM && N >= 2) {
      const WindowSpan last_of_0 = span(i0 + kBM - 1), first_of_1 = span(i0 + kBM);
      if (first_of_1.lo >= lo + kBN && last_of_0.hi <= lo + kBN * (N - 1)) n = N - 1;
    }
    steps = n + (first + kBN - 1) / kBN;
  }
  __device__ __forceinline__ int tile_of(int u) const {
    const int t = u >> 1;
    return t < n ? t + ((N - n) & u) : N + t - n;
  }
  // whether unit u meets another tile than the unit before it
  __device__ __forceinline__ bool fresh(int u) const { return u == 0 || ((u + (u < 2 * n ? N - n : 0)) & 1) == 0; }
  __device__ __forceinline__ int begin(int tile) const { return tile < N ? lo + tile * kBN : (tile - N) * kBN; }
  __device__ __forceinline__ int valid(int tile) const { return min(kBN, tile < N ? win - tile * kBN : first - (tile - N) * kBN); }
};

// A block as the roles that do not load see it.
struct Item {
  Walk walk;
  int q0, head, seg;
  int q_begin, q_len;            // where its sequence begins in the results, and its length
  int from, to, sinks;           // of its sequence, see WindowSeq
  int k_end, k_floor;            // see window_span
  int part;                      // 1: a part's state, which a launch behind this one joins with the others
};
static_assert(sizeof(Item) <= 80, "shared-memory layout");

// Bits [a, b) of a word, as far as they lie in it.
__device__ __forceinline__ uint32_t run_of_bits(int a, int b) {
  uint32_t x, y;         // (shl.b32 by 32 and more gives 0)
  asm("shl.b32 %0, 1, %1;" : "=r"(x) : "r"(min(max(a, 0), 32)));
  asm("shl.b32 %0, 1, %1;" : "=r"(y) : "r"(min(max(b, 0), 32)));
  return (y - 1u) & ~(x - 1u);
}

// 64 bf16 columns of a warp's 32 rows, a row per lane, to rows `pitch` elements apart: through shared memory (4 KB of the warp's), so that
// 8 lanes write the 128 contiguous bytes of a row.  The 16-byte pieces are XOR-swizzled by row against bank conflicts.
__device__ __forceinline__ void store_rows64_bf16(uint8_t* stage, uint16_t* dst, int64_t pitch, int rows, const uint32_t* row) {
  const int lane = threadIdx.x & 31, r0 = lane >> 3, piece = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(row[4 * i], row[4 * i + 1], row[4 * i + 2], row[4 * i + 3]);
  __syncwarp();
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int r = it * 4 + r0;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
    if (r < rows) *reinterpret_cast<uint4*>(dst + r * pitch + piece * 8) = v;
  }
  __syncwarp();        // the stage is written again for the next columns
}

// The results of a block that sees no key, by one thread: empty states (out = 0, lse = -inf).  A state that it were folded into stays
// as it is.
template <int D>
__device__ __forceinline__ void write_none(const FlashParams& p, const Item& w, const uint8_t* zeros) {
  if (p.accumulate) return;
  const int size = p.out_dtype == 0 ? 4 : 2;
#pragma unroll 1
  for (int i = w.q0; i < min(w.q0 + kQT * kBM, w.q_len); ++i) {
    const int64_t tok = static_cast<int64_t>(w.q_begin) + i;
    p.lse[lse_index(p, w.seg, w.head, i, tok)] = -INFINITY;
    bulk_store(static_cast<uint8_t*>(p.out) + (tok * p.out_tok_stride + w.head * D) * size, zeros, D * size);
  }
  bulk_store_commit();
}

// Where things are in shared memory.  Every role makes its own from an address that the compiler cannot see through (see
// flash_fwd_persistent_sm100.cu).
template <int D>
struct Shared {
  using C = Cfg<D>;
  uint8_t* s_q;
  uint8_t* s_kv;
  uint8_t* s_out;
  float2* s_ml;           // [tile][row]: reference and sum of a finished row
  Item* s_work;
  uint8_t* s_zero;        // a row of zeros
  uint8_t* s_claim;
  uint64_t* q_full;       // [block buffer][tile]
  uint64_t* q_empty;      // [block buffer]: the block's last S has read both tiles
  uint64_t* kv_full;
  uint64_t* kv_empty;
  uint64_t* s_full;       // [buffer]: S(u) is in tensor memory
  uint64_t* p_lo;         // [buffer]: first part of P(u) written (one arrival per softmax warp)
  uint64_t* p_hi;         // [buffer]: the rest of P(u) written
  uint64_t* pv_done;      // [tile]: PV(u) has completed
  uint64_t* o_final;      // [tile]: O of the block is complete
  uint64_t* o_free;       // [tile]: ... and has been read (one arrival per result warp)
  uint64_t* ml_full;      // [tile]: references and sums of the block's rows are in s_ml
  uint64_t* ml_empty;     // [tile]: ... and have been read
  uint64_t* work_full;    // [slot]
  uint64_t* work_empty;   // [slot]: no role looks at the slot's block any more
  uint64_t* v_tail;       // [in turn]: what lies behind the keys of a tile that is not full has been cleared
  uint64_t* claim;
  uint32_t* tmem_slot;

  __device__ __forceinline__ explicit Shared(uint8_t* smem) {
    s_q = smem;
    s_kv = s_q + C::kQBufs * kQT * C::kTileBytes;
    s_out = s_kv + C::kStages * C::kTileBytes;
    s_ml = reinterpret_cast<float2*>(s_out + C::kStageOut);
    s_work = reinterpret_cast<Item*>(s_ml + kQT * kBM);
    s_zero = reinterpret_cast<uint8_t*>(s_work + kWork);
    s_claim = s_zero + D * 4;
    q_full = reinterpret_cast<uint64_t*>(s_claim + 16);
    q_empty = q_full + 2 * C::kQBufs;
    kv_full = q_empty + C::kQBufs;
    kv_empty = kv_full + C::kStages;
    s_full = kv_empty + C::kStages;
    p_lo = s_full + C::kSBufs;
    p_hi = p_lo + C::kSBufs;
    pv_done = p_hi + C::kSBufs;
    o_final = pv_done + 2;
    o_free = o_final + 2;
    ml_full = o_free + 2;
    ml_empty = ml_full + 2;
    work_full = ml_empty + 2;
    work_empty = work_full + kWork;
    v_tail = work_empty + kWork;
    claim = v_tail + kTails;
    tmem_slot = reinterpret_cast<uint32_t*>(q_full + C::kBars);
  }
};
// 0, as far as the compiler knows any number.
__device__ __forceinline__ uint32_t opaque_zero() {
  uint32_t z = 0;
  asm volatile("" : "+r"(z));
  return z;
}

// Cluster launch control: ask for a block of this grid that has not started yet ...
__device__ __forceinline__ void claim_request(void* response16, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(response16)), "r"(smem_u32(bar)) : "memory");
}
// ... and read the answer: false when there was none left (not to be asked again then).
__device__ __forceinline__ bool claim_answer(const void* response16, int& x, int& y, int& z) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %3, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, %2, _}, r;\n\t}"
      : "=&r"(x), "=&r"(y), "=&r"(z), "=&r"(ok)
      : "r"(smem_u32(response16))
      : "memory");
  return ok != 0;
}

}  // namespace

// grid: (row blocks, heads, sequences x parts); in pages as plan_blocks deals them out.  Keys and values dense (CUtensorMap, WindowParams) or in
// pages (PagedMap, PagedParams): the two differ in how a sequence and a tile's rows are found.
template <int D, class QMap, class Map, class Params>
__global__ void __launch_bounds__(kThreads, 1)
flash_window_kernel(const __grid_constant__ QMap tm_q, const __grid_constant__ Map tm_k,
                    const __grid_constant__ Map tm_v, const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int NB = C::kSBufs;
  extern __shared__ uint8_t smem_raw[];
  // (an offset and not a rounded address: the compiler then still knows that it is shared memory)
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  const Shared<D> sh(smem);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // ------------------------------------------------------------------ set-up
  if (threadIdx.x == kTmaWarp * 32) {
    for (int i = 0; i < C::kQBufs; ++i) {
      mbar_init(&sh.q_full[2 * i], 1);
      mbar_init(&sh.q_full[2 * i + 1], 1);
      mbar_init(&sh.q_empty[i], 1);
    }
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_lo[i], 4);
      mbar_init(&sh.p_hi[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.pv_done[i], 1);
      mbar_init(&sh.o_final[i], 1);
      mbar_init(&sh.o_free[i], 4);
      mbar_init(&sh.ml_full[i], 4);
      mbar_init(&sh.ml_empty[i], 4);
    }
    for (int i = 0; i < kWork; ++i) {
      mbar_init(&sh.work_full[i], 1);
      mbar_init(&sh.work_empty[i], kWorkReaders);
    }
    for (int i = 0; i < kTails; ++i) mbar_init(&sh.v_tail[i], 1);
    mbar_init(sh.claim, 1);
    init_loads(p);
    fence_mbar_init();
  }
  plan_blocks(p);
  if (warp == kMmaWarp + 1 && lane < D / 4) {
    reinterpret_cast<uint4*>(sh.s_zero)[lane] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(sh.tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  // CTA-uniform view of the status word: a CTA that starts after a failure elsewhere does no work.
  const int aborted = __syncthreads_or(*reinterpret_cast<volatile int*>(p.f.status) != 0);
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(sh.tmem_slot);

  // The next block as every role but the loader sees it: its slot, or -1 when there is none.  Slots are given back by
  // one arrival per reading warp.
  uint32_t fetched = 0;
  auto take = [&](const Shared<D>& sh, bool there) {
    const uint32_t slot = fetched++ % kWork;
    return there && sh.s_work[slot].walk.steps >= 0 ? static_cast<int>(slot) : -1;
  };
  auto fetch = [&](const Shared<D>& sh) {                       // by one thread
    return take(sh, wait_or_abort(&sh.work_full[fetched % kWork], (fetched / kWork) & 1, p.f.status, 51));
  };
  auto fetch_warp = [&](const Shared<D>& sh) {                  // by a whole warp
    return take(sh, warp_wait_or_abort(&sh.work_full[fetched % kWork], (fetched / kWork) & 1, p.f.status, 51));
  };
  auto give_back = [&](const Shared<D>& sh, int slot) {         // by a whole warp
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.work_empty[slot]);
  };

  if (warp >= kTmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsOther));
    if (aborted) {
      // fall through to the tear-down
    } else if (warp > kMmaWarp) {
      serve_loads<D>(p, warp - kMmaWarp - 1);
    } else if (warp == kTmaWarp) {
      // ------------------------------------------------------------ blocks and TMA loads
      const Shared<D> sh(smem + opaque_zero());
      if (elect_one()) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        int it = 0;                // K and V tiles loaded, over all blocks
        int tails = 0;             // of them V tiles that were not full
        int items = 0;             // blocks with keys
        int published = 0;
        uint32_t claims = 0;
        bool live = true, asked = false;
        int bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z, splits = p.splits, state = -1;
        auto ask = [&]() {
          asked = true;
          if (!claims_blocks(p)) return;
          fence_proxy_async_smem();            // the answer before this one has been read
          mbar_expect_tx(sh.claim, 16);
          claim_request(sh.s_claim, sh.claim);
        };
        auto publish = [&](const Item& w) {
          const int slot = published % kWork, round = published / kWork;
          if (round > 0 && !wait_or_abort(&sh.work_empty[slot], (round - 1) & 1, p.f.status, 14)) return false;
          sh.s_work[slot] = w;
          mbar_arrive(&sh.work_full[slot]);
          ++published;
          return true;
        };
        for (;;) {
          Item w;
          place_block(p, bx, by, bz, splits, state);
          const int seg = bz / splits, part = bz % splits;
          w.head = by;
          w.seg = seg;
          w.q0 = bx * (kQT * kBM);
          const WindowSeq s = window_seq(p, seg);
          w.q_begin = (p.f.cu_q != nullptr ? s.q_begin : seg * p.f.seqlen_q) + part * static_cast<int>(p.f.total_q);
          w.q_len = s.q_len;
          w.from = s.from;
          w.to = s.to;
          w.sinks = s.sinks;
          w.k_end = s.k_len;
          w.k_floor = s.sinks;
          w.part = 0;
          place_results(p, w, state);
          asked = false;
          if (w.q0 < w.q_len) {
            const int i1 = min(w.q0 + kQT * kBM, w.q_len) - 1;
            w.walk.plan(w.from, w.to, w.sinks, w.k_end, w.k_floor, w.q0, i1, key_align(p), row_shift(p));
            if (splits > 1) {
              // as many tiles to each part, the first tokens to the last one
              const int begin = w.walk.lo, end = begin + w.walk.win;
              const int keys = (w.walk.N + (w.walk.first + kBN - 1) / kBN + splits - 1) / splits * kBN;
              // (the first tile may begin in front of the window's keys)
              w.k_floor = max(min(begin + part * keys, end), w.k_floor);
              if (part + 1 < splits) {
                w.k_end = min(begin + (part + 1) * keys, end);
                w.sinks = 0;
              }
              w.walk.plan(w.from, w.to, w.sinks, w.k_end, w.k_floor, w.q0, i1, key_align(p), row_shift(p));
            }
            const Walk walk = w.walk;
            const int n_units = 2 * walk.steps;
            if (n_units == 0) {
              // The other roles do not meet it.  (The issuer asks for the block behind the one under way before it ends that one: with
              // a run of such blocks in between, more than there are slots, each role would wait for another.)
              write_none<D>(results_at(p, w), w, sh.s_zero);
            } else {
              if (!publish(w)) break;
              const int qb = items % C::kQBufs, q_round = items / C::kQBufs;
              const int kv_head = by / (p.f.num_heads / p.kv_heads);
              const int batch = p.f.cu_q != nullptr ? 0 : seg;
              int k_tile = -1, v_tile = -1;
              auto load_kv = [&](const auto* tm, int tile, int batch_first) {
                const int stage = it % C::kStages;
                const int round = it / C::kStages;
                ++it;
                if (round > 0 && !wait_or_abort(&sh.kv_empty[stage], (round - 1) & 1, p.f.status, 11)) return false;
                mbar_expect_tx(&sh.kv_full[stage], C::kTileBytes);
                for (int x = 0; x < C::kSlabs; ++x)
                  tma_load_token(sh.s_kv + stage * C::kTileBytes + x * kSlabBytes, tm, &sh.kv_full[stage], kv_head * D + x * 64, s.k_begin + walk.begin(tile), batch, batch_first);
                return true;
              };
              auto load_k = [&](int u) {
                if (walk.tile_of(u) == k_tile) return true;
                k_tile = walk.tile_of(u);
                return load_kv(&tm_k, k_tile, p.k_batch_first);
              };
              auto load_v = [&](int u) {
                if (walk.tile_of(u) == v_tile) return true;
                v_tile = walk.tile_of(u);
                if (!load_kv(&tm_v, v_tile, p.v_batch_first)) return false;
                const int keys = walk.valid(v_tile), front = u == 0 ? front_of(p, walk) : 0;
                if ((keys & 15) == 0 && front == 0) return true;
                // What lies behind the tile's last key in its step of 16, and before its first one, is cleared.  (Nobody gives the slot back
                // before that: the issuer waits for v_tail, so the phase waited for here is the one that this load completes.)
                const int stage = (it - 1) % C::kStages;
                if (!wait_or_abort(&sh.kv_full[stage], ((it - 1) / C::kStages) & 1, p.f.status, 12)) return false;
#pragma unroll 1
                for (int x = 0; x < C::kSlabs; ++x) {
                  uint8_t* behind = sh.s_kv + stage * C::kTileBytes + x * kSlabBytes + keys * 128;     // whole rows of 128 bytes: the swizzle stays inside
#pragma unroll 1
                  for (int i = 0; i < (-keys & 15) * 8; ++i) *reinterpret_cast<uint4*>(behind + i * 16) = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
                  for (int i = 0; i < front * 8; ++i) *reinterpret_cast<uint4*>(sh.s_kv + stage * C::kTileBytes + x * kSlabBytes + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();                     // the MMA reads shared memory through the asynchronous proxy
                mbar_arrive(&sh.v_tail[tails++ % kTails]);
                return true;
              };
              if (q_round > 0 && !wait_or_abort(&sh.q_empty[qb], (q_round - 1) & 1, p.f.status, 13)) break;
              // in the order in which the issuer consumes them
              for (int t = 0; live && t < kQT; ++t) {
                uint64_t* full = &sh.q_full[qb * 2 + t];
                mbar_expect_tx(full, C::kTileBytes);
                for (int x = 0; x < C::kSlabs; ++x)
                  tma_load_token(sh.s_q + (qb * kQT + t) * C::kTileBytes + x * kSlabBytes, &tm_q, full, by * D + x * 64, s.q_begin + w.q0 + t * kBM, batch, p.q_batch_first);
                live = load_k(t);
              }
              for (int u = 2; live && u < NB && u < n_units; ++u) live = load_k(u);
              for (int u = 0; live && u < n_units; ++u) {
                if (u == 2 * (walk.steps > kClaimAhead ? walk.steps - kClaimAhead : 0)) ask();
                live = load_v(u);
                if (live && u + NB < n_units) live = load_k(u + NB);
              }
              if (!live) break;
              ++items;
            }
          }
          if (!asked) ask();
          bool more;
          if (claims_blocks(p)) {
            if (!wait_or_abort(sh.claim, claims & 1, p.f.status, 15)) break;
            ++claims;
            more = claim_answer(sh.s_claim, bx, by, bz);
          } else {
            more = next_place(p, bx);
          }
          if (!more) {
            w.walk.steps = -1;
            publish(w);
            break;
          }
        }
        bulk_store_wait();               // the zeros have been read
      }
      __syncwarp();
      if (lane == 0) end_loads(p);
    } else {
      // ------------------------------------------------------------ MMA issuer
      const Shared<D> sh(smem + opaque_zero());
      if (elect_one()) {
        constexpr uint32_t idesc_qk = idesc_bf16_f32(kBM, kBN, false, false);
        constexpr uint32_t idesc_pv = idesc_bf16_f32(kBM, D, false, true);
        const uint32_t kv_addr = smem_u32(sh.s_kv);
        const uint64_t q_desc = smem_desc_sw128(smem_u32(sh.s_q), 16, 1024);    // K-major
        const uint64_t k_desc = smem_desc_sw128(kv_addr, 16, 1024);          // K-major
        const uint64_t v_desc = smem_desc_sw128(kv_addr, kSlabBytes, 1024);  // MN-major, slab pitch leading
        // S = Q K^T of the operands that `ready_s` found
        auto issue_s = [&](uint64_t a0, uint64_t b0, uint32_t d) {
#pragma unroll
          for (int k16 = 0; k16 < D / 16; ++k16) {
            const uint32_t off = ((k16 >> 2) * kSlabBytes + (k16 & 3) * 32) >> 4;
            mma_ss(d, a0 + off, b0 + off, idesc_qk, k16 > 0);
          }
        };
        // O_tile (+)= P V over half of the tile's eight steps of 16 keys, from step `k0`, as far as `steps` go; P (bf16 pairs) at
        // the start of S buffer `buf`.  Full tiles have no limit to test.
        auto issue_pv = [&](int tile, int stage, int buf, bool acc, int k0, int steps) {
          const uint64_t b0 = v_desc + static_cast<uint32_t>(stage * (C::kTileBytes >> 4)) + static_cast<uint32_t>(k0 * 2048 >> 4);
          const uint32_t d = tmem_base + C::kColO + tile * D;
          const uint32_t a = tmem_base + C::kColS + buf * kBN + k0 * 8;
          if (steps == kBN / 16) {
#pragma unroll
            for (int kk = 0; kk < kSplit / 16; ++kk) mma_ts(d, a + kk * 8, b0 + (kk * 2048 >> 4), idesc_pv, (acc || kk > 0) ? 1u : 0u);
          } else {
#pragma unroll 1
            for (int kk = 0; kk < min(kSplit / 16, steps - k0); ++kk) mma_ts(d, a + kk * 8, b0 + (kk * 2048 >> 4), idesc_pv, (acc || kk > 0) ? 1u : 0u);
          }
        };
        int stage = 0;             // next ring slot to consume
        uint32_t round = 0;        // its parity
        auto next_kv = [&](int& held, int code) {
          if (!wait_or_abort(&sh.kv_full[stage], round, p.f.status, code)) return false;
          tc_fence_after();
          held = stage;
          if (++stage == C::kStages) { stage = 0; round ^= 1; }
          return true;
        };
        // (What is worked out per unit is kept short: one thread runs this, and a unit takes 0.65 us at D = 64.  With the tiles of
        // units u, u + 1, u + NB and u + NB + 1 compared, 2 x 8888 x 24 x 64 without a window took 1386 us.)
        Walk ahead;                // of the block whose S are issued; PV's may still be a block behind
        int ahead_units = 0;
        auto next_item = [&]() {
          const int slot = fetch(sh);
          if (slot < 0) return false;
          ahead = sh.s_work[slot].walk;
          mbar_arrive(&sh.work_empty[slot]);
          ahead_units = 2 * ahead.steps;
          return true;
        };
        int k_stage = 0, v_stage = 0, tails = 0;
        int q_tile = 0;            // of the block ahead: its first tile in s_q, ...
        uint32_t q_use = 0;        // ... and the parity of its loads
        uint32_t o_use = 1;        // parity of the reads of the O before this block's
        bool first = true;
        int buf = 0;               // S / P buffer of the next PV; units are numbered through all blocks
        uint32_t use = 0;          // parity of its barriers
        // S(un) of the block ahead into buffer `b`: operands, K taken where the unit's tile is a new one ...
        uint64_t s_a = 0, s_b = 0;
        auto ready_s = [&](int un) {
          if (ahead.fresh(un) && !next_kv(k_stage, 22)) return false;
          s_a = q_desc + static_cast<uint32_t>((q_tile + (un & 1)) * (C::kTileBytes >> 4));
          s_b = k_desc + static_cast<uint32_t>(k_stage * (C::kTileBytes >> 4));
          return true;
        };
        // ... and what follows its MMAs, K given back where the next unit's tile is another
        auto commit_s = [&](int un, int b) {
          mma_commit(&sh.s_full[b]);
          const bool last = un + 1 == ahead_units;
          if (last || ahead.fresh(un + 1)) mma_commit(&sh.kv_empty[k_stage]);
          if (last) mma_commit(&sh.q_empty[q_tile >> 1]);
        };
        // S(un) itself, un < NB
        auto put_s = [&](int un, int b) {
          if (!ready_s(un)) return false;
          if (un < 2 && !wait_or_abort(&sh.q_full[q_tile + un], q_use, p.f.status, 21)) return false;
          tc_fence_after();
          issue_s(s_a, s_b, tmem_base + C::kColS + b * kBN);
          commit_s(un, b);
          return true;
        };
        bool ok = next_item(), more = ok;
        for (int u = 0; ok && u < NB && u < ahead_units; ++u) ok = put_s(u, u);
        while (ok && more) {
          const Walk walk = ahead;
          const int n_units = ahead_units;
          // the units that first meet the last tile of the window and that of the first tokens, which need not be full
          const int u_window = walk.N > 0 ? 2 * walk.n - 2 + (walk.N - walk.n) : -1, u_first = walk.steps > walk.n ? n_units - 2 : -1;
          int v_steps = kBN / 16;
          // unit u's tile of V, a new one, and how many steps of 16 keys of it count
          auto next_v = [&](int u) {
            if (!next_kv(v_stage, 23)) return false;
            v_steps = kBN / 16;
            const bool front = u == 0 && front_of(p, walk) > 0;
            if (u != u_window && u != u_first && !front) return true;
            const int keys = u == u_window ? walk.valid(walk.N - 1) : u == u_first ? walk.valid(walk.N + walk.steps - walk.n - 1) : kBN;
            v_steps = (keys + 15) >> 4;
            if ((keys & 15) == 0 && !front) return true;
            const int n = tails++;
            return wait_or_abort(&sh.v_tail[n % kTails], (n / kTails) & 1, p.f.status, 28);
          };
          // Everything that S(u + NB) needs is waited for in front of P(u): behind P(u) there are the MMAs alone, for the
          // softmax warps of this Q tile then wait for them.
          auto pv = [&](int u) {
            const int half = u & 1;
            if (u < 2 && !first && !wait_or_abort(&sh.o_free[half], o_use, p.f.status, 30)) return false;
            if (!wait_or_abort(&sh.p_lo[buf], use, p.f.status, 24 + half)) return false;
            tc_fence_after();
            issue_pv(half, v_stage, buf, u > 1, 0, v_steps);
            if (!wait_or_abort(&sh.p_hi[buf], use, p.f.status, 26 + half)) return false;
            tc_fence_after();
            issue_pv(half, v_stage, buf, true, kSplit / 16, v_steps);
            return true;
          };
          for (int u = 0; ok && u < n_units - 2; ++u) {
            const bool more_s = u + NB < n_units;
            ok = (!walk.fresh(u) || next_v(u)) && (!more_s || ready_s(u + NB)) && pv(u);
            if (!ok) break;
            mma_commit(&sh.pv_done[u & 1]);
            if (more_s) {
              issue_s(s_a, s_b, tmem_base + C::kColS + buf * kBN);
              commit_s(u + NB, buf);
            }
            if (walk.fresh(u + 1)) mma_commit(&sh.kv_empty[v_stage]);
            if (++buf == NB) { buf = 0; use ^= 1; }
          }
          if (!ok) break;
          // The block's last two units.  In the S buffers that they leave go the first units of the next block, so that the softmax warps
          // find their scores while O is still being read: a third buffer is free now, the others behind their PV.  (The ring has the
          // last unit's V in front of the next block's K, so it is taken first.)
          const bool apart = walk.fresh(n_units - 1);
          ok = !walk.fresh(n_units - 2) || next_v(n_units - 2);
          int v_last = v_stage, steps_last = v_steps;
          if (ok && apart) {
            const int v = v_stage, steps = v_steps;
            ok = next_v(n_units - 1);
            v_last = v_stage;
            steps_last = v_steps;
            v_stage = v;
            v_steps = steps;
          }
          if (!ok) break;
          more = next_item();
          if (more) {
            q_tile += kQT;
            if (q_tile == kQT * C::kQBufs) { q_tile = 0; q_use ^= 1; }
            if (NB > 2) ok = put_s(0, buf == 0 ? NB - 1 : buf - 1);
          }
#pragma unroll 1
          for (int half = 0; ok && half < kQT; ++half) {
            ok = pv(n_units - 2 + half);
            if (!ok) break;
            mma_commit(&sh.o_final[half]);
            // An arrival that nothing waits for could still be under way when the CTA ends and its shared memory gets a new
            // owner: behind the last PV of all there is only o_final.
            if (more) {
              mma_commit(&sh.pv_done[half]);
              if (half == 1 || apart) mma_commit(&sh.kv_empty[v_stage]);
              if (half + NB - 2 < ahead_units) ok = put_s(half + NB - 2, buf);
            }
            v_stage = v_last;
            v_steps = steps_last;
            if (++buf == NB) { buf = 0; use ^= 1; }
          }
          first = false;
          o_use ^= 1;
        }
      }
      __syncwarp();
    }
  } else if (warp >= kOutWarp) {
    // -------------------------------------------------------------- results
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsOutput));
    if (!aborted) {
      const Shared<D> sh(smem + opaque_zero());
      const int quarter = warp & 3;
      const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      uint8_t* stage = sh.s_out + quarter * 4096;
      const float c = p.f.scale_log2;
      const bool accumulate = p.f.accumulate != 0;
      uint32_t item_use = 0;
      for (int slot; (slot = fetch_warp(sh)) >= 0;) {
        const int q0 = sh.s_work[slot].q0, head = sh.s_work[slot].head, seg = sh.s_work[slot].seg;
        const int q_begin = sh.s_work[slot].q_begin, q_len = sh.s_work[slot].q_len;
        const int part = sh.s_work[slot].part;
        give_back(sh, slot);
        bool ok = true;
        if constexpr (std::is_same<Params, PagedParams>::value) {
          for (int tile = 0; ok && tile < kQT; ++tile)
            ok = paged_results<D>(p, part != 0, seg, head, q0 + tile * kBM + quarter * 32, q_begin, q_len, lane_base + C::kColO + tile * D, stage, [&](float2& ml) {
              if (!warp_wait_or_abort(&sh.ml_full[tile], item_use, p.f.status, 42)) return false;
              ml = sh.s_ml[tile * kBM + quarter * 32 + lane];
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh.ml_empty[tile]);
              if (!warp_wait_or_abort(&sh.o_final[tile], item_use, p.f.status, 41)) return false;
              tc_fence_after();
              return true;
            }, [&]() {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh.o_free[tile]);
            });
        } else {
#pragma unroll 1
          for (int tile = 0; ok && tile < kQT; ++tile) {
            const uint32_t o_taddr = lane_base + C::kColO + tile * D;
            const int warp_pos = q0 + tile * kBM + quarter * 32;      // position of the warp's first row
            const int rows = q_len - warp_pos;
            const int64_t tok0 = static_cast<int64_t>(q_begin) + warp_pos;
            const int64_t li = lse_index(p.f, seg, head, warp_pos + lane, tok0 + lane);
            const int64_t col = static_cast<int64_t>(head) * D;
            float lse_old = -INFINITY;
            if (accumulate && lane < rows) lse_old = p.f.lse[li];     // under way while the rows are still being computed
            ok = warp_wait_or_abort(&sh.ml_full[tile], item_use, p.f.status, 42);
            if (!ok) break;
            const float2 ml = sh.s_ml[tile * kBM + quarter * 32 + lane];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.ml_empty[tile]);
            // a row that has seen no key is an empty state, and leaves a state that it is folded into as it is (a NaN among its scores is not that)
            float w_new = 0.f, w_old = lse_old != -INFINITY ? 1.f : 0.f, lse_out = lse_old;
            if (ml.y != 0.f) merge_weights(accumulate, lse_old, (ml.x * c + log2f(ml.y)) * kLn2, ml.y, w_new, w_old, lse_out);
            ok = warp_wait_or_abort(&sh.o_final[tile], item_use, p.f.status, 41);
            if (!ok) break;
            tc_fence_after();
            if (lane < rows) p.f.lse[li] = lse_out;
            auto o_read = [&]() {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh.o_free[tile]);
            };
            if (p.f.out_dtype != 0) {
              // bf16: 64 columns at a time, rounded as they are read, so that the next block's products do not wait long for O.  (A block of
              // 25 steps, D = 64 and 128: 35.5 and 55.0 us; 36.6 and 54.8 with 32 fp32 columns staged at a time, 36.5 and 56.0 with
              // every lane storing its row from registers.)
              uint16_t* dst = static_cast<uint16_t*>(p.f.out) + tok0 * p.f.out_tok_stride + col;
#pragma unroll 1
              for (int x = 0; x < D / 64; ++x) {
                uint32_t orow[32];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  uint32_t v[32];
                  tmem_ld32(o_taddr + x * 64 + q * 32, v);
                  tmem_wait_ld<32>(v);
#pragma unroll
                  for (int i = 0; i < 16; ++i)
                    orow[q * 16 + i] = pack_bf16x2(__uint_as_float(v[2 * i]) * w_new, __uint_as_float(v[2 * i + 1]) * w_new);
                }
                if (x == D / 64 - 1) o_read();
                if (rows > 0) store_rows64_bf16(stage, dst + x * 64, p.f.out_tok_stride, rows, orow);
              }
              continue;
            }
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
              uint32_t orow[32];
              tmem_ld32(o_taddr + q * 32, orow);
              tmem_wait_ld<32>(orow);
              if (q == D / 32 - 1) o_read();
              OldRows old;
              if (accumulate) load_old_rows32(p.f, tok0, rows, col + q * 32, old);
              if (rows > 0) store_rows32(p.f, stage, tok0, rows, col + q * 32, orow, old, w_new, w_old);
            }
          }
        }
        if (!ok) break;
        item_use ^= 1;
      }
    }
  } else {
    // -------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
    if (!aborted) {
      const Shared<D> sh(smem + opaque_zero());
      const int tile = warp >> 2;
      const int quarter = warp & 3;
      const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t o_taddr = lane_base + C::kColO + tile * D;
      const float c = p.f.scale_log2;
      int buf = tile;            // S / P buffer of the next key tile
      uint32_t use = 0;          // parity of its barriers
      uint32_t pv_use = 1;       // parity of PV of the key tile before
      uint32_t ml_use = 2;        // parity of the reads of the rows before; 2: there are none
      bool ok = true;
      for (int slot; ok && (slot = fetch_warp(sh)) >= 0;) {
        // The columns of a step's tile that the row sees, [c0, c1); both move on by a tile a step, and at the first tokens, `window`
        // steps on, become [0, first).
        int left, window, first, c0, c1;
        {
          const Item& w = sh.s_work[slot];
          left = w.walk.steps;
          window = w.walk.n;
          // (a row behind the last one sees what the last one sees)
          const WindowSpan span = window_span(w.from, w.to, w.sinks, w.k_end, w.k_floor, min(w.q0 + tile * kBM + quarter * 32 + lane, w.q_len - 1) >> row_shift(p));
          const int base = w.walk.lo + ((w.walk.N - window) & tile) * kBN;
          c0 = span.lo - base;
          c1 = span.hi - base;
          first = span.first;
        }
        give_back(sh, slot);
        float m = -INFINITY;     // running max of raw scores (lazily updated); -inf: the row has seen no key yet
        float l = 0.f;           // running sum of exp2((s - m) * c)
        bool begun = false;
        for (; left > 0; --left, --window, c0 -= kBN, c1 -= kBN) {
          if (window == 0) {
            c0 = 0;
            c1 = first;
          }
          const uint32_t s_taddr = lane_base + C::kColS + buf * kBN;   // S(u), then P(u) over its first half
          const bool masked = __any_sync(0xffffffffu, c0 > 0 || c1 < kBN);
          ok = warp_wait_or_abort(&sh.s_full[buf], use, p.f.status, 31 + tile);
          if (!ok) break;
          tc_fence_after();
          uint32_t sr[kBN];
          tmem_ld32(s_taddr, sr);
          tmem_ld32(s_taddr + 32, sr + 32);
          tmem_wait_ld<64>(sr);
          tmem_ld32(s_taddr + 64, sr + 64);      // in flight while the first half is scanned
          tmem_ld32(s_taddr + 96, sr + 96);
          auto hide = [&](int i0) {
#pragma unroll
            for (int w = i0; w < i0 + 64; w += 32) {
              if (__any_sync(0xffffffffu, c0 > w || c1 < w + 32)) {
                const uint32_t seen = run_of_bits(c0 - w, c1 - w);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if ((seen & (1u << i)) == 0) sr[w + i] = 0xff800000u;   // -inf
              }
            }
          };
          if (masked) hide(0);
          float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
          auto scan = [&](int i0) {
#pragma unroll
            for (int i = i0; i < i0 + 64; i += 8) {
              mx0 = max3(mx0, __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
              mx1 = max3(mx1, __uint_as_float(sr[i + 2]), __uint_as_float(sr[i + 3]));
              mx2 = max3(mx2, __uint_as_float(sr[i + 4]), __uint_as_float(sr[i + 5]));
              mx3 = max3(mx3, __uint_as_float(sr[i + 6]), __uint_as_float(sr[i + 7]));
            }
          };
          scan(0);
          tmem_wait_ld<64>(sr + 64);
          if (masked) hide(64);
          scan(64);
          const float m_new = fmaxf(max3(m, mx0, mx1), fmaxf(mx2, mx3));
          if (!begun) {
            m = m_new;
            begun = true;
          } else {
            // (a row's first score is growth without end, a row without any grows by a NaN, that is, not)
            const bool grow = (m_new - m) * c > kRescaleThreshold;
            if (__any_sync(0xffffffffu, grow)) {
              // O is rescaled in place: PV of this Q tile's key tile before must have drained (PV(u) is not issued before this
              // group hands over P(u))
              ok = warp_wait_or_abort(&sh.pv_done[tile], pv_use, p.f.status, 33 + tile);
              if (!ok) break;
              tc_fence_after();
              const float f = m == -INFINITY ? 0.f : ex2((m - m_new) * c);       // without a key so far O and l are 0
#pragma unroll
              for (int q = 0; q < D / 16; ++q) {
                uint32_t orow[16];
                tmem_ld16(o_taddr + q * 16, orow);
                tmem_wait_ld<16>(orow);
#pragma unroll
                for (int i = 0; i < 16; ++i) orow[i] = __float_as_uint(__uint_as_float(orow[i]) * f);
                tmem_st16(o_taddr + q * 16, orow);
              }
              tmem_wait_st();
              l *= f;
              m = m_new;
            }
          }
          // p = 2^(s*c - m*c), at most 2^8; 0 for what is hidden, also while m is -inf.  (All on the ex2 unit: with one pair of eight on
          // the FMA units, which the kernels without masks gain from, a block of 25 steps at D = 64 took 37.3 us in place of 35.7; with the
          // next tile's scores asked for under the second half, where they are there by then, 38.2.)
          const float ref = m == -INFINITY ? 0.f : -m * c;
          const uint64_t c2 = pack2(c, c), nmc2 = pack2(ref, ref);
          uint64_t sum0 = pack2(0.f, 0.f), sum1 = sum0;
          auto exp_part = [&](int i0, int i1) {
#pragma unroll
            for (int i = i0; i < i1; i += 2) {
              const uint64_t x = fma2(pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), c2, nmc2);
              const uint64_t pp = exp2_mufu2(x);
              if (i & 2) sum1 = add2(sum1, pp); else sum0 = add2(sum0, pp);
              float p0, p1;
              unpack2(pp, p0, p1);
              sr[i >> 1] = pack_bf16x2(p0, p1);
            }
          };
          exp_part(0, kSplit);
          tmem_st32(s_taddr, sr);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_lo[buf]);
          exp_part(kSplit, kBN);
          tmem_st32(s_taddr + 32, sr + 32);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_hi[buf]);
          float s0, s1, s2, s3;
          unpack2(sum0, s0, s1);
          unpack2(sum1, s2, s3);
          l += (s0 + s1) + (s2 + s3);
          pv_use ^= 1;
          buf += 2;
          if (buf >= NB) { buf -= NB; use ^= 1; }
        }
        if (!ok) break;
        if (ml_use < 2) ok = warp_wait_or_abort(&sh.ml_empty[tile], ml_use, p.f.status, 43);
        if (!ok) break;          // the rows before these have not been read
        sh.s_ml[tile * kBM + quarter * 32 + lane] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.ml_full[tile]);
        ml_use = (ml_use & 1) ^ (ml_use < 2);
      }
    }
  }

  // ------------------------------------------------------------------ tear-down
  if (*reinterpret_cast<volatile int*>(p.f.status) != 0) __nanosleep(1000000);   // let copies in flight land
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

static dim3 tile_grid(const WindowParams& p) { return dim3((p.f.seqlen_q + kQT * kBM - 1) / (kQT * kBM), p.f.num_heads, p.f.nseg * p.splits); }
static dim3 tile_grid(const PagedParams& p) { return dim3(p.blocks); }

template <int D, class QMap, class Map, class Params>
static cudaError_t launch_tiles(const QMap& tq, const Map& tk, const Map& tv, const Params& p, cudaStream_t stream) {
  using C = Cfg<D>;
  static bool configured[64] = {};
  static std::mutex mu;
  const auto kernel = flash_window_kernel<D, QMap, Map, Params>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!configured[dev & 63]) {
      // the register hand-over waits for good unless the kernel starts with what it was computed for
      cudaFuncAttributes fa;
      e = cudaFuncGetAttributes(&fa, kernel);
      if (e == cudaSuccess && fa.numRegs != kRegsLaunch) e = cudaErrorInvalidKernelImage;
      if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
      if (e != cudaSuccess) return e;
      configured[dev & 63] = true;
    }
  }
  kernel<<<tile_grid(p), kThreads, C::kSmemBytes, stream>>>(tq, tk, tv, p);
  return cudaGetLastError();
}

template <int D>
cudaError_t launch_window_tiles(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const WindowParams& p, cudaStream_t stream) {
  return launch_tiles<D>(tq, tk, tv, p, stream);
}
template <int D>
cudaError_t launch_paged_tiles(const QueryMap& tq, const PagedMap& tk, const PagedMap& tv, const PagedParams& p, cudaStream_t stream) {
  static_assert(kLoadPlaces >= Cfg<D>::kStages + kLoadWarps, "requests that have not been read, and those that end the queue, have places of their own");
  return launch_tiles<D>(tq, tk, tv, p, stream);
}

template cudaError_t launch_window_tiles<64>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const WindowParams&, cudaStream_t);
template cudaError_t launch_window_tiles<128>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const WindowParams&, cudaStream_t);
template cudaError_t launch_paged_tiles<64>(const QueryMap&, const PagedMap&, const PagedMap&, const PagedParams&, cudaStream_t);
template cudaError_t launch_paged_tiles<128>(const QueryMap&, const PagedMap&, const PagedMap&, const PagedParams&, cudaStream_t);

}  // namespace dtb
