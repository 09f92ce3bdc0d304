"""The loader and the MMA issuer of the windowed attention kernel, replayed on the CPU.

Both are taken out of the kernel's source with the walk over key tiles that they share, compiled for the host against stubs that record
what they wait for, load, multiply and commit, and played against each other here: every wait has to be met, every product has to
find the key tile that its unit is due in the ring slot it reads, and the tiles of a row, over all parts that the keys are split into, have
to hold the keys it sees, once each."""
import os
import re
import shutil
import subprocess

import pytest

from tests.test_flash_issuer_cpu import CSRC, _block

STUBS = r"""
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>
#define __device__
#define __forceinline__ inline
using std::max; using std::min;
struct CUtensorMap { int x; };
constexpr int kQueriesLast = INT32_MIN;
struct FlashParams { int* status; const int32_t *cu_q, *cu_k; int seqlen_q, seqlen_k, num_heads, nseg, accumulate; int64_t total_q; };
struct WindowParams { FlashParams f; const int32_t* seqlens_k; int kv_heads, left, right, sinks, q_start, k_start, q_batch_first, k_batch_first, v_batch_first, splits; };
%(seq)s
%(span)s
%(constants)s
%(cfg)s
%(walk)s
%(item)s
constexpr int D = %(head_dim)d;
using C = Cfg<D>;
constexpr int NB = C::kSBufs;
struct Arrays {
  uint64_t q_full[2 * C::kQBufs], q_empty[C::kQBufs], kv_full[C::kStages], kv_empty[C::kStages], s_full[NB], p_lo[NB], p_hi[NB], pv_done[2];
  uint64_t o_final[2], o_free[2], work_full[kWork], work_empty[kWork], v_tail[kTails], claim[1];
  uint8_t s_q[C::kQBufs * kQT * C::kTileBytes], s_kv[C::kStages * C::kTileBytes], s_claim[16];
  Item s_work[kWork];
} sh_;
template <int>
struct Shared {
  uint64_t *q_full = sh_.q_full, *q_empty = sh_.q_empty, *kv_full = sh_.kv_full, *kv_empty = sh_.kv_empty, *s_full = sh_.s_full, *p_lo = sh_.p_lo;
  uint64_t *p_hi = sh_.p_hi, *pv_done = sh_.pv_done, *o_final = sh_.o_final, *o_free = sh_.o_free, *work_full = sh_.work_full;
  uint64_t *work_empty = sh_.work_empty, *v_tail = sh_.v_tail, *claim = sh_.claim, *s_zero = nullptr;
  uint8_t *s_q = sh_.s_q, *s_kv = sh_.s_kv, *s_claim = sh_.s_claim;
  Item* s_work = sh_.s_work;
  explicit Shared(uint8_t*) {}
};
uint32_t opaque_zero() { return 0; }
CUtensorMap tm_q, tm_k, tm_v;
struct uint4 { uint32_t x, y, z, w; };
uint4 make_uint4(uint32_t, uint32_t, uint32_t, uint32_t) { return uint4{1, 1, 1, 1}; }
constexpr uint32_t idesc_bf16_f32(int, int, bool, bool) { return 0; }
uint32_t smem_u32(const void* x) { return x == sh_.s_q ? 0u : uint32_t(C::kQBufs * kQT * C::kTileBytes); }
uint64_t smem_desc_sw128(uint32_t addr, uint32_t, uint32_t) { return addr >> 4; }
std::vector<Item> items, nones;        // blocks with keys, blocks without
template <int> void write_none(const FlashParams&, const Item& w, const uint64_t*) { nones.push_back(w); }
void bulk_store_wait() {}
void event(const char* what, const uint64_t* bar, int extra) {
#define BAR(b) if (bar >= sh_.b && bar < sh_.b + sizeof(sh_.b) / 8) std::printf("%%s %%s %%d %%d\n", what, #b, int(bar - sh_.b), extra)
  BAR(q_full); BAR(q_empty); BAR(o_free); BAR(kv_full); BAR(kv_empty); BAR(s_full); BAR(p_lo); BAR(p_hi); BAR(pv_done); BAR(o_final); BAR(v_tail);
  BAR(work_full); BAR(work_empty); BAR(claim);
}
bool wait_or_abort(uint64_t* bar, uint32_t parity, int*, int) { event("wait", bar, int(parity)); return true; }
void mbar_expect_tx(uint64_t* bar, uint32_t) { event("expect", bar, 0); }
void mbar_arrive(uint64_t* bar) {
  if (bar >= sh_.work_full && bar < sh_.work_full + kWork) items.push_back(sh_.s_work[bar - sh_.work_full]);
  if (bar >= sh_.v_tail && bar < sh_.v_tail + kTails) {
    int cleared = 0, first = -1;        // rows of 128 bytes that were cleared
    for (int i = 0; i < int(sizeof(sh_.s_kv) / 128); ++i)
      if (sh_.s_kv[i * 128] != 0) { ++cleared; if (first < 0) first = i; }
    for (auto& x : sh_.s_kv) x = 0;
    std::printf("cleared %%d %%d\n", cleared, first);
  }
  event("arrive", bar, 0);
}
void fence_proxy_async_smem() {}
void prefetch_tmap(const CUtensorMap*) {}
void tma_load_token(void* dst, const CUtensorMap* m, uint64_t*, int x, int token, int batch, int) {
  std::printf("load %%s %%d %%d\n", m == &tm_q ? "q" : m == &tm_k ? "k" : "v",
              m == &tm_q ? int((uint8_t*)dst - sh_.s_q) / kSlabBytes : int((uint8_t*)dst - sh_.s_kv) / kSlabBytes, token);
}
void mma_commit(uint64_t* bar) { event("commit", bar, 0); }
void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t, uint32_t) { std::printf("S %%u %%llu %%llu\n", d, (unsigned long long)a, (unsigned long long)b); }
void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t, uint32_t acc) {
  std::printf("PV %%u %%u %%llu %%u\n", d, a, (unsigned long long)b, acc);
}
void tc_fence_after() {}
bool elect_one() { return true; }
// blocks of the launch in their order, every `stride`th of them to this CTA
int next_block, stride, n_blocks, row_blocks, heads;
struct { int x, y, z; } blockIdx;
void claim_request(void*, uint64_t* bar) { event("arrive", bar, 0); }
bool claim_answer(const void*, int& x, int& y, int& z) {
  next_block += stride;
  if (next_block >= n_blocks) return false;
  x = next_block %% row_blocks; y = next_block / row_blocks %% heads; z = next_block / (row_blocks * heads);
  return true;
}
int main(int, char** argv) {
  WindowParams p = {};
  p.f.seqlen_q = std::atoi(argv[1]); p.f.seqlen_k = std::atoi(argv[2]); p.left = std::atoi(argv[3]); p.right = std::atoi(argv[4]);
  p.sinks = std::atoi(argv[5]); p.q_start = std::atoi(argv[6]); p.k_start = std::atoi(argv[7]);
  p.f.num_heads = std::atoi(argv[8]); p.kv_heads = p.f.num_heads; p.f.nseg = 1; next_block = std::atoi(argv[9]); stride = std::atoi(argv[10]);
  row_blocks = (p.f.seqlen_q + 255) / 256;
  p.splits = std::atoi(argv[11]); p.f.total_q = p.f.seqlen_q; heads = p.f.num_heads;
  n_blocks = row_blocks * heads * p.splits;
  blockIdx.x = next_block %% row_blocks; blockIdx.y = next_block / row_blocks %% heads; blockIdx.z = next_block / (row_blocks * heads);
  uint8_t* smem = nullptr;
  const uint32_t tmem_base = 0;
  std::printf("loader 0\n");
%(loader)s
  std::printf("issuer 0\n");
  uint32_t fetched = 0;
  auto fetch = [&](const Shared<D>& sh) {
    event("wait", &sh.work_full[fetched %% kWork], (fetched / kWork) & 1);
    const uint32_t slot = fetched++ %% kWork;
    sh.s_work[slot] = items[fetched - 1];
    return sh.s_work[slot].walk.steps >= 0 ? int(slot) : -1;
  };
%(issuer)s
  std::printf("blocks 0\n");
  items.insert(items.end(), nones.begin(), nones.end());
  for (const Item& w : items) {
    if (w.walk.steps < 0) continue;
    std::printf("block %%d %%d %%d %%d %%d %%d\n", w.q0, w.walk.steps, w.walk.N, w.walk.n, w.head, w.q_begin / int(p.f.total_q));
    for (int i = w.q0; i < min(w.q0 + 256, w.q_len); ++i) {
      const WindowSpan s = window_span(w.from, w.to, w.sinks, w.k_end, w.k_floor, i);
      std::printf("row %%d %%d %%d %%d\n", i, s.first, s.lo, s.hi);
    }
    for (int u = 0; u < 2 * w.walk.steps; ++u) { const int t = w.walk.tile_of(u); std::printf("unit %%d %%d %%d %%d\n", u, t, w.walk.begin(t), w.walk.valid(t)); }
  }
}
"""


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    kernel = open(os.path.join(CSRC, "flash_window_sm100.cu")).read()
    common = open(os.path.join(CSRC, "flash_common.cuh")).read()
    window = open(os.path.join(CSRC, "flash_window.cuh")).read()
    constants = "\n".join(re.findall(r"^constexpr int k\w+ = [^;]*;", common, re.M) + re.findall(r"^constexpr int k\w+ = [^;]*;", kernel, re.M))
    seq = window[window.index("struct WindowSeq"):window.index("// Keys that query i sees")]
    span = window[window.index("struct WindowSpan"):window.index("// Element offset")]
    parts = dict(constants=constants, seq=seq, span=span, cfg="template <int D>\nstruct Cfg " + _block(kernel, kernel.index("struct Cfg")) + ";",
                 walk="struct Walk " + _block(kernel, kernel.index("struct Walk")) + ";",
                 item="struct Item " + _block(kernel, kernel.index("struct Item")) + ";",
                 loader=_role(kernel, "- blocks and TMA loads"), issuer=_role(kernel, "- MMA issuer"))
    built = {}
    for head_dim in (64, 128):
        d = tmp_path_factory.mktemp("walk")
        src, exe = str(d / "walk.cpp"), str(d / "walk")
        with open(src, "w") as f:
            f.write(STUBS % dict(parts, head_dim=head_dim))
        r = subprocess.run([gxx, "-std=c++17", "-O0", "-w", src, "-o", exe], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        built[head_dim] = exe

    def run(head_dim, *args):
        r = subprocess.run([built[head_dim], *map(str, args)], capture_output=True, text=True)
        assert r.returncode == 0
        return [line.split() for line in r.stdout.splitlines()]
    return run


def _role(kernel, title):
    """A role's own view of shared memory and the code of its elected thread, as a scope."""
    return "{ const Shared<D> sh(smem);\n" + _block(kernel, kernel.index("if (elect_one())", kernel.index(title))) + "\n}"


def _play(head_dim, loader, issuer):
    """Runs the two event lists against each other; returns the products as (event, slab of the ring, what was loaded there)."""
    slabs, stages, q_bytes = head_dim // 64, {64: 8, 128: 4}[head_dim], {64: 4, 128: 2}[head_dim] * 128 * head_dim * 2
    phase = {}                              # (barrier, index) -> completed phases
    ring = {}                               # slab of the ring -> (tensor, token)
    done, products = lambda b: phase.get(b, 0), []

    def passes(ev):
        # (a wait on a parity passes while the phase under way has the other one)
        return done((ev[1], ev[2])) % 2 != int(ev[3])

    def complete(b):
        phase[b] = done(b) + 1
    at, loads, published, taken = [0, 0], 0, 0, 0         # blocks that the loader has published, and that the issuer has read
    while at[0] < len(loader) or at[1] < len(issuer):
        moved = False
        while at[0] < len(loader):
            ev = loader[at[0]]
            # a block's slot is free once the issuer has read it, and the warps of the results have, which do so when the block before is final
            if ev[0] == "wait" and ev[1] == "work_empty":
                n = published - 4
                if taken <= n or done(("o_final", "1")) < n:
                    break
            elif ev[0] == "wait" and not passes(ev):
                break
            if ev[:2] == ["arrive", "work_full"]:
                published += 1
            if ev[0] == "expect":
                last = (ev[1], ev[2])
            elif ev[0] == "load":
                if ev[1] != "q":
                    assert int(ev[2]) // slabs == int(last[1])
                    ring[int(ev[2])] = (ev[1], int(ev[3]))
                loads += 1
                if loads % slabs == 0:
                    complete(last)
            elif ev[0] == "arrive":
                complete((ev[1], ev[2]))
            at[0] += 1
            moved = True
        while at[1] < len(issuer):
            ev = issuer[at[1]]
            # softmax: P(u) follows S(u) at once
            if ev[0] == "wait" and ev[1] in ("p_lo", "p_hi"):
                assert done(("s_full", ev[2])) > done((ev[1], ev[2]))
                complete((ev[1], ev[2]))
            # ... and O is read once it is final
            if ev[0] == "wait" and ev[1] == "o_free":
                assert done(("o_final", ev[2])) > done(("o_free", ev[2]))
                complete((ev[1], ev[2]))
            if ev[0] == "wait" and not passes(ev):
                break
            if ev[:2] == ["arrive", "work_empty"]:
                taken += 1
            if ev[0] in ("commit", "arrive"):
                complete((ev[1], ev[2]))
            elif ev[0] in ("S", "PV"):
                off = int(ev[3]) * 16 - q_bytes            # from the ring's start
                slab = off // (128 * 128)
                assert 0 <= slab < stages * slabs
                products.append((ev, slab, ring[slab]))
            at[1] += 1
            moved = True
        assert moved, ("stuck", loader[at[0]:at[0] + 1], issuer[at[1]:at[1] + 1])
    return products, phase


def _blocks(ev):
    """[(q0, steps, N, n, head, part, rows, units)]"""
    out = []
    for e in ev[ev.index(["blocks", "0"]) + 1:]:
        n = [int(x) for x in e[1:]]
        if e[0] == "block":
            out.append((*n, [], []))
        else:
            out[-1][6 if e[0] == "row" else 7].append(tuple(n))
    return out


CASES = [  # Sq, Sk, left, right, sinks, q_start, k_start
    (300, 300, 100, 100, 0, 0, 0), (700, 700, 200, 200, 130, 0, 0), (1000, 4000, 1500, 0, 226, 3000, 0), (513, 2000, 300, 77, 13, 700, 0),
    (256, 256, 0, 0, 0, 0, 0), (600, 600, 0, 0, 300, 0, 0), (400, 450, 100, 500, 405, 0, 400), (400, 450, 50, 0, 950, 1000, 900),
    (1024, 1024, 2 ** 30, 2 ** 30, 0, 0, 0), (800, 3000, 128, 127, 128, 1100, 0), (300, 100, 20, 10, 4, -50, 0), (2000, 2000, 255, 256, 64, 0, 0),
    (260, 5000, 700, 700, 1, 2500, 0), (500, 60, 10, 10, 0, 0, 0), (1500, 1500, 20, 20, 5, 0, 0), (1500, 1500, 100, 0, 0, 0, 0),
    (2600, 100, 50, 50, 0, 0, 0), (3500, 200, 40, 10, 0, -2900, 0), (4000, 700, 30, 30, 0, -1700, 0)]


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("heads,grid,splits", [(1, 1, 1), (3, 2, 1), (2, 148, 1), (2, 3, 2), (1, 148, 5), (1, 2, 8)])
def test_every_unit_meets_its_tile_and_every_row_its_keys(replay, case, head_dim, heads, grid, splits):
    Sq, Sk, left, right, sinks, q_start, k_start = case
    n_blocks = -(-Sq // 256) * heads * splits
    shares, most = {}, {}                # (head, row) -> keys that it sees, over the parts; (head, q0) -> steps of each part
    covered, slabs, q_bufs = 0, head_dim // 64, {64: 2, 128: 1}[head_dim]
    for cta in range(min(grid, n_blocks)):
        ev = replay(head_dim, *case, heads, cta, grid, splits)
        blocks = _blocks(ev)
        covered += len(blocks)
        for q0, steps, N, n, head, part, rows, units in blocks:
            most.setdefault((head, q0), []).append(steps)
            assert len(units) == 2 * steps
            for i, first, lo, hi in rows:
                x = q_start + i
                seen = [j for j in range(Sk) if j + k_start <= x + right and (j + k_start >= x - left or j + k_start < sinks)]
                share = list(range(first)) + list(range(lo, hi))
                shares.setdefault((head, i), []).extend(share)
                assert splits > 1 or share == seen
                # the columns that the kernel lets the row see, unit by unit of its Q tile
                met = []
                for u, tile, base, valid in units[(i - q0) // 128::2]:
                    c0, c1 = (lo - base, hi - base) if tile < N else (0, first - base)
                    assert min(c1, 128) <= valid             # nothing behind the tile's last key
                    met += range(base + max(c0, 0), base + min(max(c1, 0), 128))
                assert sorted(met) == share
            if not steps:
                assert all(first == 0 and lo >= hi for _, first, lo, hi in rows)
        at = ev.index(["issuer", "0"])
        loader, issuer = ev[1:at], ev[at + 1:ev.index(["blocks", "0"])]
        real = [b for b in blocks if b[1] > 0]
        units = [(*u, i % q_bufs) for i, b in enumerate(real) for u in b[7]]
        products, phase = _play(head_dim, loader, issuer)
        # S: one after another, from the unit's tile of K and its block's queries; PV: the same of V, over the steps of 16 keys that hold one
        s = [p for p in products if p[0][0] == "S"]
        assert len(s) == len(units) * head_dim // 16
        for n, (e, slab, held) in enumerate(s):
            u, tile, base, valid, q_buf = units[n // (head_dim // 16)]
            assert held == ("k", base) and int(e[2]) * 16 // (128 * head_dim * 2) == 2 * q_buf + u % 2
        pv = [p for p in products if p[0][0] == "PV"]
        k = 0
        for u, tile, base, valid, _ in units:
            for step in range(-(-valid // 16)):
                e, slab, held = pv[k]
                inside = int(e[3]) * 16 % (128 * 128 * slabs)
                assert held == ("v", base) and inside == step * 2048 and int(e[4]) == int(u > 1 or step > 0)
                k += 1
        assert k == len(pv)
        # tiles that are not full are cleared behind their last key, up to a multiple of 16
        clears = [(int(e[1]), int(e[2])) for e in loader if e[0] == "cleared"]
        ragged = [r for b in blocks for r in dict.fromkeys((tile, valid) for _, tile, _, valid in b[7] if valid % 16)]
        assert len(clears) == len(ragged) <= 2 * len(blocks)
        for (count, first), (_, valid) in zip(clears, ragged):
            assert count == (16 - valid % 16) * slabs and first % 128 == valid
        if not real:
            continue
        # the last commits are those that the epilogue waits for, each with its last products in front of it
        finals = [i for i, e in enumerate(issuer) if e[:2] == ["commit", "o_final"]]
        last_mma = max(i for i, e in enumerate(issuer) if e[0] in ("S", "PV"))
        assert [issuer[i][2] for i in finals] == ["0", "1"] * len(real) and finals[-1] == len(issuer) - 1
        assert all(i < last_mma for i, e in enumerate(issuer) if e[0] == "commit" and e[1] != "o_final")
        # one completion of pv_done for every unit, but the CTA's last two
        assert all(phase.get(("pv_done", str(h)), 0) == sum(b[1] for b in real) - 1 for h in (0, 1))
        # the queries' memory is given back behind the last S that reads it
        given = [sum(x[0] == "S" for x in issuer[:i]) for i, e in enumerate(issuer) if e[:2] == ["commit", "q_empty"]]
        assert given == [sum(2 * b[1] for b in real[:i + 1]) * head_dim // 16 for i in range(len(real))]
    assert covered == n_blocks and len(shares) == Sq * heads
    for (head, i), share in shares.items():
        x = q_start + i
        assert sorted(share) == [j for j in range(Sk) if j + k_start <= x + right and (j + k_start >= x - left or j + k_start < sinks)]
    if splits > 1:                       # an even share each
        for steps in most.values():
            assert len(steps) == splits and max(steps) <= -(-sum(steps) // splits) + max(1, -(-sinks // 128))


def test_windows_that_no_end_cuts_take_a_tile_less(replay):
    """2701 keys for each row: 23 tiles hold those of 128 rows, 24 those of 256; two more hold the 226 first ones."""
    ev = replay(64, 17776, 17776, 1350, 1350, 226, 0, 0, 1, 30, 70, 1)
    q0, steps, N, n = _blocks(ev)[0][:4]
    assert (q0, N, n, steps) == (256 * 30, 24, 23, 23 + 2)


FAR = 2 ** 30


@pytest.mark.parametrize("left,right,sinks,q_start,k_start", [
    (-1, 0, 0, FAR, 0), (-1, 5, 0, FAR, -FAR), (-1, -1, 0, FAR, -FAR), (-1, -1, 0, -FAR, FAR), (40, -1, 0, -FAR, 0), (40, -1, 7, -FAR, FAR),
    (-1, 0, 0, -FAR, 0), (40, -1, 0, FAR, -FAR), (40, -1, 3, FAR, 0), (FAR, FAR, 0, FAR, -FAR), (FAR, FAR, 0, -FAR, FAR), (FAR, 0, 0, FAR, 0)])
@pytest.mark.parametrize("splits", [1, 3])
def test_no_limit_is_none_at_any_position(replay, left, right, sinks, q_start, k_start, splits):
    """At the ends of the positions that are accepted, where a limit of 2^30 does hide keys."""
    Sq, Sk = 600, 300
    seen, blocks = {}, 0
    for block in range(3 * splits):
        for q0, steps, N, n, head, part, rows, units in _blocks(replay(64, Sq, Sk, left, right, sinks, q_start, k_start, 1, block, 3 * splits, splits)):
            blocks += 1
            for i, first, lo, hi in rows:
                seen.setdefault(i, []).extend(list(range(first)) + list(range(lo, hi)))
    assert blocks == 3 * splits and len(seen) == Sq
    for i, keys in seen.items():
        x = q_start + i
        assert sorted(keys) == [j for j in range(Sk) if (right < 0 or j + k_start <= x + right) and (left < 0 or j + k_start >= x - left or j + k_start < sinks)]
