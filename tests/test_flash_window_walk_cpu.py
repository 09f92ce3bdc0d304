"""The loader and the MMA issuer of the windowed attention kernel, replayed on the CPU.

Both are taken out of the kernel's source with the walk over key tiles that they share, compiled for the host against stubs that record
what they wait for, load, multiply and commit, and played against each other here: every wait has to be met, every product has to
find the key tile that its unit is due in the ring slot it reads, and the tiles of a row have to hold the keys it sees, once each."""
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
#define __device__
#define __forceinline__ inline
#define __restrict__
using std::max; using std::min;
struct CUtensorMap { int x; };
constexpr int kQueriesLast = INT32_MIN;
struct FlashParams { int* status; const int32_t *cu_q, *cu_k; int seqlen_q, seqlen_k; };
struct WindowParams { FlashParams f; const int32_t* seqlens_k; int left, right, sinks, q_start, k_start, q_batch_first, k_batch_first, v_batch_first; };
%(seq)s
%(span)s
%(constants)s
%(cfg)s
%(walk)s
constexpr int D = %(head_dim)d;
using C = Cfg<D>;
constexpr int NB = C::kSBufs;
constexpr int kRing = C::kStages;
uint64_t q_full[2], kv_full[kRing], kv_empty[kRing], s_full[NB], p_lo[NB], p_hi[NB], pv_done[2], o_final[2], v_tail[2];
uint8_t s_q[kQT * C::kTileBytes], s_kv[kRing * C::kKvTileBytes];
CUtensorMap tm_q, tm_k, tm_v;
struct uint4 { uint32_t x, y, z, w; };
uint4 make_uint4(uint32_t, uint32_t, uint32_t, uint32_t) { return uint4{1, 1, 1, 1}; }
constexpr uint32_t idesc_bf16_f32(int, int, bool, bool) { return 0; }
uint32_t smem_u32(const void* x) { return x == s_q ? 0u : uint32_t(kQT * C::kTileBytes); }
uint64_t smem_desc_sw128(uint32_t addr, uint32_t, uint32_t) { return addr >> 4; }
void event(const char* what, const uint64_t* bar, int extra) {
#define BAR(b) if (bar >= b && bar < b + sizeof(b) / 8) std::printf("%%s %%s %%d %%d\n", what, #b, int(bar - b), extra)
  BAR(q_full); BAR(kv_full); BAR(kv_empty); BAR(s_full); BAR(p_lo); BAR(p_hi); BAR(pv_done); BAR(o_final); BAR(v_tail);
}
bool wait_or_abort(uint64_t* bar, uint32_t parity, int*, int) { event("wait", bar, int(parity)); return true; }
void mbar_expect_tx(uint64_t* bar, uint32_t) { event("expect", bar, 0); }
void mbar_arrive(uint64_t* bar) {
  int cleared = 0, first = -1;        // rows of 128 bytes that were cleared
  for (int i = 0; i < int(sizeof(s_kv) / 128); ++i) {
    if (s_kv[i * 128] != 0) { ++cleared; if (first < 0) first = i; }
  }
  for (auto& x : s_kv) x = 0;
  std::printf("cleared %%d %%d\n", cleared, first);
  event("arrive", bar, 0);
}
void fence_proxy_async_smem() {}
void prefetch_tmap(const CUtensorMap*) {}
void tma_load_token(void* dst, const CUtensorMap* m, uint64_t*, int x, int token, int batch, int) {
  std::printf("load %%s %%d %%d\n", m == &tm_q ? "q" : m == &tm_k ? "k" : "v",
              m == &tm_q ? int((uint8_t*)dst - s_q) / kSlabBytes : int((uint8_t*)dst - s_kv) / kSlabBytes, token);
}
void mma_commit(uint64_t* bar) { event("commit", bar, 0); }
void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t, uint32_t) { std::printf("S %%u %%llu %%llu\n", d, (unsigned long long)a, (unsigned long long)b); }
void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t, uint32_t acc) {
  std::printf("PV %%u %%u %%llu %%u\n", d, a, (unsigned long long)b, acc);
}
void tc_fence_after() {}
bool elect_one() { return true; }
int main(int, char** argv) {
  WindowParams p = {};
  p.f.seqlen_q = std::atoi(argv[1]); p.f.seqlen_k = std::atoi(argv[2]); p.left = std::atoi(argv[3]); p.right = std::atoi(argv[4]);
  p.sinks = std::atoi(argv[5]); p.q_start = std::atoi(argv[6]); p.k_start = std::atoi(argv[7]);
  const int q0 = std::atoi(argv[8]), head = 0, kv_head = 0, batch = 0;
  const WindowSeq s = window_seq(p, 0);
  const Walk walk(p, s, q0, min(q0 + kQT * kBM, s.q_len) - 1);
  std::printf("walk %%d %%d %%d %%d\n", walk.steps, walk.tiles, walk.skew, walk.N);
  for (int i = q0; i < min(q0 + kQT * kBM, s.q_len); ++i) { WindowSpan w = window_span(p, s, i); std::printf("row %%d %%d %%d %%d\n", i, w.first, w.lo, w.hi); }
  for (int u = 0; u < kQT * walk.steps; ++u) { const int t = walk.tile_of(u); std::printf("unit %%d %%d %%d %%d\n", u, t, walk.begin(t), walk.valid(t)); }
  if (walk.steps <= 0) return 0;
  const int n_units = kQT * walk.steps;
  const uint32_t tmem_base = 0;
  std::printf("loader 0\n");
%(loader)s
  std::printf("issuer 0\n");
%(issuer)s
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
                 loader=_block(kernel, kernel.index("if (elect_one())", kernel.index("- TMA producer"))),
                 issuer=_block(kernel, kernel.index("if (elect_one())", kernel.index("- MMA issuer"))))
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


def _play(head_dim, loader, issuer, n_units):
    """Runs the two event lists against each other; returns the products as (kind, unit half, slab of the ring, token loaded there)."""
    slabs, stages, nb = head_dim // 64, {64: 10, 128: 5}[head_dim], {64: 3, 128: 2}[head_dim]
    phase = {}                              # (barrier, index) -> completed phases
    ring = {}                               # slab of the ring -> (tensor, token)
    done, products, cleared = lambda b: phase.get(b, 0), [], {}

    def passes(ev):
        # (a wait on a parity passes while the phase under way has the other one)
        return done((ev[1], ev[2])) % 2 != int(ev[3])

    def complete(b):
        phase[b] = done(b) + 1
    at = [0, 0]
    while at[0] < len(loader) or at[1] < len(issuer):
        moved = False
        while at[0] < len(loader):
            ev = loader[at[0]]
            if ev[0] == "wait" and not passes(ev):
                break
            if ev[0] == "expect":
                last = (ev[1], ev[2])
            elif ev[0] == "load":
                if ev[1] != "q":
                    assert int(ev[2]) // slabs == int(last[1])
                    ring[int(ev[2])] = (ev[1], int(ev[3]))
                if sum(e[0] == "load" for e in loader[:at[0] + 1]) % slabs == 0:
                    complete(last)
            elif ev[0] == "cleared":
                cleared[last[1]] = (int(ev[1]), int(ev[2]))
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
            if ev[0] == "wait" and not passes(ev):
                break
            if ev[0] == "commit":
                complete((ev[1], ev[2]))
            elif ev[0] in ("S", "PV"):
                off = int(ev[3]) * 16 - 2 * 128 * head_dim * 2            # from the ring's start
                slab = off // (128 * 128)
                assert 0 <= slab < stages * slabs
                products.append((ev, slab, ring[slab]))
            at[1] += 1
            moved = True
        assert moved, ("stuck", loader[at[0]:at[0] + 1], issuer[at[1]:at[1] + 1])
    return products, phase


CASES = [  # Sq, Sk, left, right, sinks, q_start, k_start
    (300, 300, 100, 100, 0, 0, 0), (700, 700, 200, 200, 130, 0, 0), (1000, 4000, 1500, 0, 226, 3000, 0), (513, 2000, 300, 77, 13, 700, 0),
    (256, 256, 0, 0, 0, 0, 0), (600, 600, 0, 0, 300, 0, 0), (400, 450, 100, 500, 405, 0, 400), (400, 450, 50, 0, 950, 1000, 900),
    (1024, 1024, 2 ** 30, 2 ** 30, 0, 0, 0), (800, 3000, 128, 127, 128, 1100, 0), (300, 100, 20, 10, 4, -50, 0), (2000, 2000, 255, 256, 64, 0, 0),
    (260, 5000, 700, 700, 1, 2500, 0), (500, 60, 10, 10, 0, 0, 0)]


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("case", CASES)
def test_every_unit_meets_its_tile_and_every_row_its_keys(replay, case, head_dim):
    Sq, Sk, left, right, sinks, q_start, k_start = case
    for q0 in range(0, Sq, 256):
        ev = replay(head_dim, *case, q0)
        cut = [i for i, e in enumerate(ev) if e[0] in ("loader", "issuer")]
        head = ev[:cut[0]] if cut else ev
        steps, tiles, skew, N = (int(x) for x in head[0][1:])
        units = [tuple(int(x) for x in e[1:]) for e in head if e[0] == "unit"]
        rows = [tuple(int(x) for x in e[1:]) for e in head if e[0] == "row"]
        assert len(units) == 2 * steps
        for i, first, lo, hi in rows:
            x = q_start + i
            seen = [j for j in range(Sk) if j + k_start <= x + right and (j + k_start >= x - left or j + k_start < sinks)]
            assert seen == list(range(first)) + list(range(lo, hi))
            # the columns that the kernel lets the row see, unit by unit of its Q tile
            met = []
            for u, tile, base, valid in units[(i - q0) // 128::2]:
                c0, c1 = (lo - base, hi - base) if tile < N else (0, first - base)
                assert min(c1, 128) <= valid             # nothing behind the tile's last key
                met += range(base + max(c0, 0), base + min(max(c1, 0), 128))
            assert sorted(met) == seen
        if not steps:
            assert not cut and all(first == 0 and lo >= hi for _, first, lo, hi in rows)
            continue
        loader, issuer = ev[cut[0] + 1:cut[1]], ev[cut[1] + 1:]
        products, phase = _play(head_dim, loader, issuer, 2 * steps)
        # S: one after another, from the unit's tile of K; PV: the same of V, over the steps of 16 keys that hold one
        slabs = head_dim // 64
        s = [p for p in products if p[0][0] == "S"]
        assert len(s) == len(units) * head_dim // 16
        for n, (e, slab, held) in enumerate(s):
            u, tile, base, valid = units[n // (head_dim // 16)]
            assert held == ("k", base) and int(e[2]) * 16 // (128 * head_dim * 2) == u % 2
        pv = [p for p in products if p[0][0] == "PV"]
        k = 0
        for u, tile, base, valid in units:
            for step in range(-(-valid // 16)):
                e, slab, held = pv[k]
                inside = (int(e[3]) * 16 - 2 * 128 * head_dim * 2) % (128 * 128 * slabs)
                assert held == ("v", base) and inside == step * 2048 and int(e[4]) == int(u > 1 or step > 0)
                k += 1
        assert k == len(pv)
        # tiles that are not full are cleared behind their last key, up to a multiple of 16
        clears = [(int(e[1]), int(e[2])) for e in loader if e[0] == "cleared"]
        ragged = list(dict.fromkeys((tile, valid) for _, tile, _, valid in units if valid % 16))
        assert len(clears) == len(ragged) <= 2
        for (count, first), (_, valid) in zip(clears, ragged):
            assert count == (16 - valid % 16) * slabs and first % 128 == valid
        # the last commits are those that the epilogue waits for, each with its last products in front of it
        finals = [i for i, e in enumerate(issuer) if e[:2] == ["commit", "o_final"]]
        last_mma = max(i for i, e in enumerate(issuer) if e[0] in ("S", "PV"))
        assert [issuer[i][2] for i in finals] == ["0", "1"] and finals[-1] == len(issuer) - 1
        assert all(i < last_mma for i, e in enumerate(issuer) if e[0] == "commit" and e[1] != "o_final")
        if head_dim == 64:
            assert all(phase.get(("pv_done", str(h)), 0) == steps - 1 for h in (0, 1))


def test_windows_that_no_end_cuts_take_a_tile_less(replay):
    """2701 keys for each row: 22 tiles hold those of 128 rows, 23 those of 256."""
    ev = replay(64, 17776, 17776, 1350, 1350, 226, 0, 0, 256 * 30)
    steps, tiles, skew, N = (int(x) for x in ev[0][1:])
    assert (skew, N, steps) == (1, 24, 23 + 2)
