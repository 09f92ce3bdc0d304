// Windowed attention of many query rows: the pipeline of flash_fwd_sm100.cu (256 query rows of one (sequence, head) to a CTA as two
// Q tiles that share the tensor core, key tiles of 128, one softmax thread per row, P over S in tensor memory) over the key tiles that
// its rows see and no others.
//
// Key tiles of a CTA: N that cover the window [lo, hi) of its rows, the first one beginning at the first key that any of them sees, then
// the tiles that hold the first tokens.  The rows of Q tile 1 are 128 further on than those of Q tile 0, and so are their windows, by
// exactly one key tile: where no end of the sequence cuts them (`skew`), step t pairs (Q tile 0, key tile t) with (Q tile 1, key tile
// t + 1), and each Q tile walks N - 1 tiles in place of N.  Units u = 2 t + i stay in the order they have there; a key tile then serves
// unit 2 t - 1 and unit 2 t in place of 2 t and 2 t + 1, which only moves the places where a new tile is taken from the ring and an
// old one given back: where the tile of a unit differs from that of the unit before it.
//
// What a row sees of a tile is one run of its columns (its window, or its first tokens), so the mask is two bounds per row; a warp whose
// rows see all of a tile does not look at them.  A row may meet tiles of which it sees nothing, or none of which it sees anything:
// its maximum stays -inf, its weights 0.  The last tile of the window and that of the first tokens may hold fewer than 128 keys: their
// PV runs the steps of 16 keys that hold one, and the rows behind the last key, which may hold anything, are cleared in shared memory
// by the thread that loads them, which waits for that one load.
//
// Bound by the softmax warps (the exponentials), like flash_fwd_sm100.cu, whose comment has the reasons for the tile sizes.
#include "flash_common.cuh"
#include "flash_window.cuh"

#include <mutex>

namespace dtb {

namespace {

using namespace flash;

constexpr int kThreads = 384;
constexpr int kRegsLaunch = 168;    // what __launch_bounds__(384, 1) allots; checked before the first launch
constexpr int kRegsSoftmax = 208;   // 2 x 128 x (208 - 168) registers taken ...
constexpr int kRegsOther = 88;      // ... are the 128 x (168 - 88) the third warpgroup gives up
static_assert(2 * kRegsSoftmax + kRegsOther == 3 * kRegsLaunch, "register split");
constexpr int kTmaWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kSplit = 64;          // keys of a tile whose probabilities are handed over first
constexpr int kPolyPairs = 1;       // pairs of every 8 pairs of scores, exponentiated on the FMA units

template <int D>
struct Cfg {
  static constexpr int kSlabs = D / 64;
  static constexpr int kTileBytes = kBM * D * 2;          // one Q tile
  static constexpr int kKvTileBytes = kBN * D * 2;      // one K or V tile
  static constexpr int kStages = (D == 128) ? 5 : 10;
  static constexpr int kSBufs = (512 - kQT * D) / kBN;
  // barriers: q_full[2], kv_full[S], kv_empty[S], s_full[NB], p_lo[NB], p_hi[NB], pv_done[2], o_final[2], v_tail[2]
  static constexpr int kBars = 2 + 2 * kStages + 3 * kSBufs + 2 + 2 + 2;
  static constexpr int kSmemBytes = 1024 + kQT * kTileBytes + kStages * kKvTileBytes + kBars * 8 + 16;
  static constexpr uint32_t kTmemCols = 512;
  static constexpr uint32_t kColS = 0;                    // + buffer * 128
  static constexpr uint32_t kColO = kSBufs * kBN;       // + tile * D
  static_assert(kColO + kQT * D <= 512, "tensor memory");
  static_assert(kSmemBytes <= 232448, "shared memory");
};

// The key tiles of a CTA's rows and the order in which its units meet them.
struct Walk {
  int lo, win;        // the window's first key and length
  int first;          // first tokens
  int N, skew, n;     // tiles of the window, whether Q tile 1 is a tile ahead, window steps of a Q tile
  int steps, tiles;   // steps in all, tiles in all

  // `second`: whether there are rows behind the first 128; rows i0 (first), i_mid (128 further), i1 (last)
  __device__ __forceinline__ Walk(const WindowParams& p, const WindowSeq& s, int i0, int i1) {
    const WindowSpan a = window_span(p, s, i0), z = window_span(p, s, i1);
    first = z.first;
    lo = max(a.lo, first);
    win = max(z.hi - lo, 0);
    N = (win + kBN - 1) / kBN;
    skew = 0;
    if (i1 - i0 >= kBM && N >= 2) {
      const WindowSpan last_of_0 = window_span(p, s, i0 + kBM - 1), first_of_1 = window_span(p, s, i0 + kBM);
      skew = first_of_1.lo >= lo + kBN && last_of_0.hi <= lo + kBN * (N - 1);
    }
    n = N - skew;
    steps = n + (first + kBN - 1) / kBN;
    tiles = N + (first + kBN - 1) / kBN;
  }
  __device__ __forceinline__ int tile_of(int u) const {
    const int t = u >> 1;
    return t < n ? t + (skew & u) : N + t - n;
  }
  __device__ __forceinline__ int begin(int tile) const { return tile < N ? lo + tile * kBN : (tile - N) * kBN; }
  __device__ __forceinline__ int valid(int tile) const { return min(kBN, tile < N ? win - tile * kBN : first - (tile - N) * kBN); }
};

// Bits [a, b) of a word, as far as they lie in it.
__device__ __forceinline__ uint32_t run_of_bits(int a, int b) {
  uint32_t x, y;         // (shl.b32 by 32 and more gives 0)
  asm("shl.b32 %0, 1, %1;" : "=r"(x) : "r"(min(max(a, 0), 32)));
  asm("shl.b32 %0, 1, %1;" : "=r"(y) : "r"(min(max(b, 0), 32)));
  return (y - 1u) & ~(x - 1u);
}

}  // namespace

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
flash_window_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ WindowParams p) {
  using C = Cfg<D>;
  constexpr int NB = C::kSBufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  uint8_t* s_kv = smem + kQT * C::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_kv + C::kStages * C::kKvTileBytes);
  uint64_t* q_full = bars;                    // [tile]
  uint64_t* kv_full = q_full + 2;
  uint64_t* kv_empty = kv_full + C::kStages;
  uint64_t* s_full = kv_empty + C::kStages;   // [buffer]: S(u) is in tensor memory
  uint64_t* p_lo = s_full + NB;               // [buffer]: first part of P(u) written (one arrival per softmax warp)
  uint64_t* p_hi = p_lo + NB;                 // [buffer]: the rest of P(u) written
  uint64_t* pv_done = p_hi + NB;              // [tile]: PV(u) has completed
  uint64_t* o_final = pv_done + 2;            // [tile]: the last PV of the tile has completed
  uint64_t* v_tail = o_final + 2;             // [first or second tile that is not full]: what lies behind its keys has been cleared
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int seg = blockIdx.z;
  const int head = blockIdx.y;
  const int kv_head = head / (p.f.num_heads / p.kv_heads);
  const WindowSeq s = window_seq(p, seg);
  const int q0 = blockIdx.x * (kQT * kBM);
  if (q0 >= s.q_len) return;
  const int q_tokens = p.f.cu_q != nullptr ? s.q_begin : seg * p.f.seqlen_q;     // in the results
  const int batch = p.f.cu_q != nullptr ? 0 : seg;
  const Walk walk(p, s, q0, min(q0 + kQT * kBM, s.q_len) - 1);
  if (walk.steps <= 0) {
    if (p.f.accumulate == 0 && *reinterpret_cast<volatile int*>(p.f.status) == 0 && threadIdx.x < kQT * kBM)
      write_empty_row<D>(p.f, seg, head, q_tokens, s.q_len, q0 + static_cast<int>(threadIdx.x));
    return;
  }
  const int n_units = kQT * walk.steps;

  // ------------------------------------------------------------------ set-up
  if (threadIdx.x == kTmaWarp * 32) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_final[i], 1);
      mbar_init(&v_tail[i], 1);
    }
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_lo[i], 4);
      mbar_init(&p_hi[i], 4);
    }
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  // CTA-uniform view of the status word: a CTA that starts after a failure elsewhere does no work.
  const int aborted = __syncthreads_or(*reinterpret_cast<volatile int*>(p.f.status) != 0);
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp >= kTmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (aborted || warp > kMmaWarp) {
      // fall through to the tear-down
    } else if (warp == kTmaWarp) {
      // ------------------------------------------------------------ TMA producer
      if (elect_one()) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        auto load_q = [&](int t) {
          mbar_expect_tx(&q_full[t], C::kTileBytes);
          for (int x = 0; x < C::kSlabs; ++x)
            tma_load_token(s_q + t * C::kTileBytes + x * kSlabBytes, &tm_q, &q_full[t], head * D + x * 64, s.q_begin + q0 + t * kBM, batch, p.q_batch_first);
        };
        int it = 0, k_tile = -1, v_tile = -1, tails = 0;
        auto load_kv = [&](const CUtensorMap* tm, int tile, int batch_first) {
          const int stage = it % C::kStages;
          const int round = it / C::kStages;
          ++it;
          if (round > 0 && !wait_or_abort(&kv_empty[stage], (round - 1) & 1, p.f.status, 11)) return false;
          mbar_expect_tx(&kv_full[stage], C::kKvTileBytes);
          for (int x = 0; x < C::kSlabs; ++x)
            tma_load_token(s_kv + stage * C::kKvTileBytes + x * kSlabBytes, tm, &kv_full[stage], kv_head * D + x * 64, s.k_begin + walk.begin(tile), batch, batch_first);
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
          const int keys = walk.valid(v_tile);
          if ((keys & 15) == 0) return true;
          // What lies behind the tile's last key in its step of 16 is cleared.  (Nobody gives the slot back before that: the
          // issuer waits for v_tail, so the phase waited for here is the one that this load completes.)
          const int stage = (it - 1) % C::kStages;
          if (!wait_or_abort(&kv_full[stage], ((it - 1) / C::kStages) & 1, p.f.status, 12)) return false;
#pragma unroll 1
          for (int x = 0; x < C::kSlabs; ++x) {
            uint8_t* behind = s_kv + stage * C::kKvTileBytes + x * kSlabBytes + keys * 128;     // whole rows of 128 bytes: the swizzle stays inside
#pragma unroll 1
            for (int i = 0; i < (16 - (keys & 15)) * 8; ++i) *reinterpret_cast<uint4*>(behind + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();                     // the MMA reads shared memory through the asynchronous proxy
          mbar_arrive(&v_tail[tails++]);
          return true;
        };
        // in the order in which the issuer consumes them
        load_q(0);
        bool live = load_k(0);
        load_q(1);
        for (int u = 1; live && u < NB && u < n_units; ++u) live = load_k(u);
        for (int u = 0; live && u < n_units; ++u) {
          live = load_v(u);
          if (live && u + NB < n_units) live = load_k(u + NB);
        }
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        constexpr uint32_t idesc_qk = idesc_bf16_f32(kBM, kBN, false, false);
        constexpr uint32_t idesc_pv = idesc_bf16_f32(kBM, D, false, true);
        const uint32_t kv_addr = smem_u32(s_kv);

        // Descriptors are built once; a tile, stage or K step only moves the start-address field (units
        // of 16 bytes, no carry out of the field: shared memory ends below 2^18).
        const uint64_t q_desc = smem_desc_sw128(smem_u32(s_q), 16, 1024);    // K-major
        const uint64_t k_desc = smem_desc_sw128(kv_addr, 16, 1024);          // K-major
        const uint64_t v_desc = smem_desc_sw128(kv_addr, kSlabBytes, 1024);  // MN-major, slab pitch leading
        // S = Q_tile K^T into S buffer `buf`
        auto issue_s = [&](int tile, int stage, int buf) {
          const uint64_t a0 = q_desc + static_cast<uint32_t>(tile * (C::kTileBytes >> 4));
          const uint64_t b0 = k_desc + static_cast<uint32_t>(stage * (C::kKvTileBytes >> 4));
          const uint32_t d = tmem_base + C::kColS + buf * kBN;
#pragma unroll
          for (int k16 = 0; k16 < D / 16; ++k16) {
            const uint32_t off = ((k16 >> 2) * kSlabBytes + (k16 & 3) * 32) >> 4;
            mma_ss(d, a0 + off, b0 + off, idesc_qk, k16 > 0);
          }
        };
        // O_tile (+)= P V over half of the tile's eight steps of 16 keys, from step `k0`, as far as `steps` go; P (bf16 pairs) at
        // the start of S buffer `buf`.  Full tiles have no limit to test.
        auto issue_pv = [&](int tile, int stage, int buf, bool acc, int k0, int steps) {
          const uint64_t b0 = v_desc + static_cast<uint32_t>(stage * (C::kKvTileBytes >> 4)) + static_cast<uint32_t>(k0 * 2048 >> 4);
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
          if (!wait_or_abort(&kv_full[stage], round, p.f.status, code)) return false;
          tc_fence_after();
          held = stage;
          if (++stage == C::kStages) { stage = 0; round ^= 1; }
          return true;
        };
        int k_tile = -1, v_tile = -1, k_stage = 0, v_stage = 0, v_steps = 0, tails = 0;
        bool ok = true;
        // S(un) into buffer `buf`; K is taken where the unit's tile is a new one, and given back where the next unit's is another
        auto do_s = [&](int un, int buf) {
          const int tile = walk.tile_of(un);
          if (tile != k_tile && !next_kv(k_stage, 22)) return false;
          k_tile = tile;
          if (un < 2) {
            if (!wait_or_abort(&q_full[un], 0, p.f.status, 21)) return false;
            tc_fence_after();
          }
          issue_s(un & 1, k_stage, buf);
          mma_commit(&s_full[buf]);
          if (un + 1 < n_units && walk.tile_of(un + 1) != tile) mma_commit(&kv_empty[k_stage]);
          return true;
        };
        for (int u = 0; ok && u < NB && u < n_units; ++u) ok = do_s(u, u);
        int buf = 0;
        uint32_t use = 0;          // parity of the buffer's barriers
        // The last unit of each Q tile commits to o_final alone: nothing waits for its pv_done or for the ring slot, and an arrival
        // that nothing waits for could still be under way when the CTA ends and its shared memory gets a new owner.
        for (int u = 0; ok && u < n_units; ++u) {
          const int half = u & 1, tile = walk.tile_of(u);
          if (tile != v_tile) {
            if (!next_kv(v_stage, 23)) { ok = false; break; }
            v_tile = tile;
            const int keys = walk.valid(tile);
            v_steps = (keys + 15) >> 4;
            if ((keys & 15) != 0 && !wait_or_abort(&v_tail[tails++], 0, p.f.status, 28)) { ok = false; break; }
          }
          ok = wait_or_abort(&p_lo[buf], use, p.f.status, 24 + half);
          if (!ok) break;
          tc_fence_after();
          issue_pv(half, v_stage, buf, u > 1, 0, v_steps);
          ok = wait_or_abort(&p_hi[buf], use, p.f.status, 26 + half);
          if (!ok) break;
          tc_fence_after();
          issue_pv(half, v_stage, buf, true, kSplit / 16, v_steps);
          if (u >= n_units - 2) {
            mma_commit(&o_final[half]);
          } else {
            if (NB > 2) mma_commit(&pv_done[half]);
            if (walk.tile_of(u + 1) != tile) mma_commit(&kv_empty[v_stage]);
            if (u + NB < n_units) ok = do_s(u + NB, buf);
          }
          if (++buf == NB) { buf = 0; use ^= 1; }
        }
      }
      __syncwarp();
    }
  } else {
    // -------------------------------------------------------------- softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int tile = warp >> 2;
    const int quarter = warp & 3;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t o_taddr = lane_base + C::kColO + tile * D;
    const float c = p.f.scale_log2;
    // (a row behind the last one sees what the last one sees)
    const WindowSpan span = window_span(p, s, min(q0 + tile * kBM + quarter * 32 + lane, s.q_len - 1));
    float m = -INFINITY;   // running max of raw scores (lazily updated); -inf: the row has seen no key yet
    float l = 0.f;         // running sum of exp2((s - m) * c)
    bool ok = !aborted;
    int buf = tile;
    uint32_t use = 0;

    for (int j = 0; ok && j < walk.steps; ++j) {
      const uint32_t s_taddr = lane_base + C::kColS + buf * kBN;   // S(u), then P(u) over its first half
      // the columns that the row sees
      const bool window = j < walk.n;
      const int base = walk.begin(walk.tile_of(2 * j + tile));
      const int c0 = window ? span.lo - base : 0, c1 = (window ? span.hi : span.first) - base;
      const bool masked = __any_sync(0xffffffffu, c0 > 0 || c1 < kBN);
      ok = warp_wait_or_abort(&s_full[buf], use, p.f.status, 31 + tile);
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
          const uint32_t seen = run_of_bits(c0 - w, c1 - w);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((seen & (1u << i)) == 0) sr[w + i] = 0xff800000u;   // -inf
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
      if (j == 0) {
        m = m_new;
      } else {
        // (a row's first score is growth without end, a row without any grows by a NaN, that is, not)
        const bool grow = (m_new - m) * c > kRescaleThreshold;
        if (__any_sync(0xffffffffu, grow)) {
          // O is rescaled in place: PV(u-2), the unit of this Q tile before this one, must have drained (PV(u) is not
          // issued before this group hands over P(u)).  With two buffers S(u) was issued behind PV(u-2), so it has.
          if (NB > 2) {
            ok = warp_wait_or_abort(&pv_done[tile], (j - 1) & 1, p.f.status, 33 + tile);
            if (!ok) break;
            tc_fence_after();
          }
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
      // p = 2^(s*c - m*c), at most 2^8; 0 for what is hidden, also while m is -inf
      const float ref = m == -INFINITY ? 0.f : -m * c;
      const uint64_t c2 = pack2(c, c), nmc2 = pack2(ref, ref);
      uint64_t sum0 = pack2(0.f, 0.f), sum1 = sum0;
      auto exp_part = [&](int i0, int i1) {
#pragma unroll
        for (int i = i0; i < i1; i += 2) {
          const uint64_t x = fma2(pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), c2, nmc2);
          const uint64_t pp = ((i >> 1) & 7) >= 8 - kPolyPairs ? exp2_poly2(x) : exp2_mufu2(x);
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
      if (lane == 0) mbar_arrive(&p_lo[buf]);
      exp_part(kSplit, kBN);
      tmem_st32(s_taddr + 32, sr + 32);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_hi[buf]);
      float s0, s1, s2, s3;
      unpack2(sum0, s0, s1);
      unpack2(sum1, s2, s3);
      l += (s0 + s1) + (s2 + s3);
      buf += 2;
      if (buf >= NB) { buf -= NB; use ^= 1; }
    }

    if (ok) ok = warp_wait_or_abort(&o_final[tile], 0, p.f.status, 41);
    if (ok) {
      tc_fence_after();
      const int warp_pos = q0 + tile * kBM + quarter * 32;      // position of the warp's first row
      const int rows = s.q_len - warp_pos;
      const int64_t tok0 = static_cast<int64_t>(q_tokens) + warp_pos;
      float w_new = l > 0.f ? 1.f / l : 0.f, w_old = 0.f;
      if (lane < rows) {
        const int64_t li = lse_index(p.f, seg, head, warp_pos + lane, tok0 + lane);
        const float lse_old = p.f.accumulate ? p.f.lse[li] : -INFINITY;
        float lse_out = -INFINITY;
        if (l > 0.f) {
          merge_weights(p.f.accumulate != 0, lse_old, (m * c + log2f(l)) * kLn2, l, w_new, w_old, lse_out);
        } else if (lse_old != -INFINITY) {                      // nothing seen: the state stays as it is
          w_old = 1.f;
          lse_out = lse_old;
        }
        p.f.lse[li] = lse_out;
      }
      // staged in this warp's part of its Q tile, which the last S instruction has read
      uint8_t* stage = s_q + tile * C::kTileBytes + quarter * (C::kTileBytes / 4);
      static_assert(C::kTileBytes / 4 >= 4096, "32 rows x 128 bytes");
#pragma unroll
      for (int q = 0; q < D / 32; ++q) {
        uint32_t orow[32];
        tmem_ld32(o_taddr + q * 32, orow);
        tmem_wait_ld<32>(orow);
        OldRows old;
        if (p.f.accumulate) load_old_rows32(p.f, tok0, rows, static_cast<int64_t>(head) * D + q * 32, old);
        if (rows > 0) store_rows32(p.f, stage, tok0, rows, static_cast<int64_t>(head) * D + q * 32, orow, old, w_new, w_old);
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

template <int D>
cudaError_t launch_window_tiles(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const WindowParams& p, cudaStream_t stream) {
  using C = Cfg<D>;
  static bool configured[64] = {};
  static std::mutex mu;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!configured[dev & 63]) {
      // the register hand-over waits for good unless the kernel starts with what it was computed for
      cudaFuncAttributes fa;
      e = cudaFuncGetAttributes(&fa, flash_window_kernel<D>);
      if (e == cudaSuccess && fa.numRegs != kRegsLaunch) e = cudaErrorInvalidKernelImage;
      if (e == cudaSuccess) e = cudaFuncSetAttribute(flash_window_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
      if (e != cudaSuccess) return e;
      configured[dev & 63] = true;
    }
  }
  const dim3 grid((p.f.seqlen_q + kQT * kBM - 1) / (kQT * kBM), p.f.num_heads, p.f.nseg);
  flash_window_kernel<D><<<grid, kThreads, C::kSmemBytes, stream>>>(tq, tk, tv, p);
  return cudaGetLastError();
}

template cudaError_t launch_window_tiles<64>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const WindowParams&, cudaStream_t);
template cudaError_t launch_window_tiles<128>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const WindowParams&, cudaStream_t);

}  // namespace dtb
