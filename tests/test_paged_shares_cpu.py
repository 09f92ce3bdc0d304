"""How the kernel of few rows over pages deals its tiles to CTAs, replayed on the CPU.

The walk over sequences, blocks and tiles and the arithmetic of the shares are taken out of the sources and compiled for the host.  Checked:
every block's tiles are walked once, by CTAs one after another; the tiles' keys that a row is shown are those it sees, once each; loads stay
inside pages; and the launch that joins finds each part of a block in the slot that its CTA left it in."""
import os
import random
import re
import shutil
import subprocess

import pytest

from tests.test_flash_issuer_cpu import CSRC

SOURCE = r"""
#include <algorithm>
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <tuple>
#include <vector>
#define __device__
#define __forceinline__ inline
using std::max; using std::min;
#define CHECK(x) do { if (!(x)) { std::printf("failed: %%s, line %%d\n", #x, __LINE__); std::exit(1); } } while (0)
constexpr int kQueriesLast = INT32_MIN;
struct FlashParams { const int32_t *cu_q, *cu_k; int seqlen_q, seqlen_k, num_heads, nseg; int64_t total_q; };
struct WindowParams { FlashParams f; const int32_t* seqlens_k; int kv_heads, left, right, sinks, q_start, k_start; };
struct PagedParams : WindowParams { int pack_shift = 0, columns, pages, page_shift, box_rows, key_align, few_rows; };
%(seq)s
%(span)s
%(paged)s
constexpr int kKeys = 64;
%(constants)s
struct Join { int parts, cta, late, seg, q_begin, kv_head, row0, rows; };
%(walk)s
constexpr int R = %(rows)d;
int main(int argc, char** argv) {
  std::vector<int> a;
  for (int i = 1; i < argc; ++i) a.push_back(std::atoi(argv[i]));
  PagedParams p = {};
  const int n = a[0], most_ctas = a[1];
  p.f.num_heads = a[2]; p.kv_heads = a[3]; p.left = a[4]; p.right = a[5]; p.sinks = a[4] < 0 ? 0 : a[6]; p.page_shift = a[7]; p.few_rows = a[8];
  p.q_start = kQueriesLast;
  p.box_rows = p.key_align = min(1 << p.page_shift, 64);
  std::vector<int32_t> cu(1, 0), lens;
  for (int b = 0; b < n; ++b) { cu.push_back(cu.back() + a[9 + 2 * b]); lens.push_back(a[10 + 2 * b]); p.f.seqlen_q = max(p.f.seqlen_q, a[9 + 2 * b]); p.columns = max(p.columns, (a[10 + 2 * b] >> p.page_shift) + 1); }
  p.f.cu_q = cu.data(); p.f.total_q = cu.back(); p.seqlens_k = lens.data(); p.f.nseg = n;
  auto places = [&](const Seq& s) { return (long long)s.blocks * p.kv_heads * places_of(s); };
  long long all = 0;
  for (int i = 0; i < n; ++i) all += places(make_seq<R>(p, i));
  const Shares sh(all, most_ctas);
  const int ctas = sh.ctas;
  CHECK(sh.begin(0) == 0 && sh.begin(ctas) == all && ctas <= most_ctas && (ctas > 0) == (all > 0));
  // (sequence, unit) -> [(CTA, slot, first tile, last tile)]
  std::map<std::pair<int, int>, std::vector<std::tuple<int, int, int, int>>> parts;
  std::vector<Join> joins(max(ctas, 1));
  for (int c = 0; c < ctas; ++c) {
    const long long begin = sh.begin(c), end = sh.begin(c + 1);
    CHECK(begin < end);
    for (long long x : {begin, end - 1}) CHECK(sh.of(x) == c);
    long long at = 0;
    int seg = 0, unit = 0, place = 0;
    for (;; ++seg) {
      const Seq s = make_seq<R>(p, seg);
      if (begin < at + places(s)) { unit = int(divide(begin - at, places_of(s))); place = int(begin - at - (long long)unit * places_of(s)); break; }
      at += places(s);
    }
    long long left = end - begin;
    Seq s = make_seq<R>(p, seg);
    joins[c] = make_join(sh, s, make_block<R>(p, s, unit), seg, c, place);
    bool first_block = true;
    while (left > 0) {
      CHECK(seg < n && unit < s.blocks * p.kv_heads);
      const int tile = tiles_before(place), to = tiles_before(int(min((long long)places_of(s), place + left)));
      if (tile < to) parts[{seg, unit}].push_back({c, 2 * c + (first_block ? 0 : 1), tile, to});
      left -= min((long long)(places_of(s) - place), left); place = 0; first_block = false;
      if (++unit == s.blocks * p.kv_heads && left > 0) { unit = 0; do s = make_seq<R>(p, ++seg); while (s.blocks == 0); }
    }
  }
  // the blocks: their tiles once each, their rows' keys once each
  const int group = p.f.num_heads / p.kv_heads;
  long long blocks = 0;
  for (int seg = 0; seg < n; ++seg) {
    const Seq s = make_seq<R>(p, seg);
    blocks += s.blocks * p.kv_heads;
    std::set<int> rows;
    for (int unit = 0; unit < s.blocks * p.kv_heads; ++unit) {
      const auto& list = parts.at({seg, unit});
      int next = 0;
      for (size_t i = 0; i < list.size(); ++i) {
        CHECK(std::get<2>(list[i]) == next && std::get<3>(list[i]) > next);
        CHECK(i == 0 || std::get<0>(list[i]) == std::get<0>(list[i - 1]) + 1);
        next = std::get<3>(list[i]);
      }
      CHECK(next == s.tiles);
      const Block b = make_block<R>(p, s, unit);
      CHECK(b.rows > 0 && b.rows <= R);
      if (b.kv_head != 0) continue;
      for (int r = 0; r < b.rows; ++r) {
        const int row = b.row0 + r, i = row / group, x = lens[seg] - (cu[seg + 1] - cu[seg]) + i;
        CHECK(rows.insert(row).second);
        const WindowSpan w = window_span(s.w, i);
        std::vector<int> times(lens[seg] + 64, 0);
        for (int t = 0; t < s.tiles; ++t) {
          const int k0 = s.begin(t);
          const bool lead = t < s.lead;
          int from, upto;
          b.seen(k0, lead, from, upto);
          if (from >= upto) continue;
          CHECK(k0 %% p.box_rows == 0 && k0 >= 0 && upto <= lens[seg] && (upto - k0 + p.box_rows - 1) / p.box_rows * p.box_rows <= kKeys);
          for (int j = k0; j < k0 + kKeys; ++j)
            if (lead ? j < w.first : j >= w.lo && j < w.hi) { CHECK(j >= from && j < upto); ++times[j]; }
        }
        for (int j = 0; j < int(times.size()); ++j) {
          const bool seen = j < lens[seg] && (p.right < 0 || j <= x + p.right) && (p.left < 0 || j >= x - p.left || j < p.sinks);
          CHECK(times[j] == (seen ? 1 : 0));
        }
      }
    }
    CHECK(int(rows.size()) == ((cu[seg + 1] - cu[seg]) <= p.few_rows ? (cu[seg + 1] - cu[seg]) * group : 0));
  }
  // the joins
  std::set<std::pair<int, int>> joined;
  for (int c = 1; c < ctas; ++c) {
    const Join& j = joins[c];
    if (j.parts == 0) continue;
    const Seq s = make_seq<R>(p, j.seg);
    const int unit = j.kv_head * s.blocks + j.row0 / R;
    const Block b = make_block<R>(p, s, unit);
    CHECK(b.kv_head == j.kv_head && b.row0 == j.row0 && b.rows == j.rows && j.q_begin == cu[j.seg]);
    CHECK(joined.insert({j.seg, unit}).second);
    const auto& list = parts.at({j.seg, unit});
    CHECK(j.parts >= 2 && int(list.size()) == j.parts);
    for (int i = 0; i < j.parts; ++i) {
      const int slot = 2 * (j.cta + i) + (i == 0 ? j.late : 0);
      CHECK(std::get<0>(list[i]) == j.cta + i && std::get<1>(list[i]) == slot && slot < 2 * most_ctas);
    }
  }
  long long whole = 0;
  for (auto& [key, list] : parts) { if (list.size() == 1) ++whole; else CHECK(joined.count(key)); }
  CHECK(whole + (long long)joined.size() == blocks && (long long)parts.size() == blocks);
  std::printf("ok %%d\n", ctas);
}
"""


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    kernel = open(os.path.join(CSRC, "flash_paged_rows.cu")).read()
    window = open(os.path.join(CSRC, "flash_window.cuh")).read()
    paged = open(os.path.join(CSRC, "flash_paged.cuh")).read()
    parts = dict(
        seq=window[window.index("struct WindowSeq"):window.index("// Of what number of keys")],
        span=window[window.index("struct WindowSpan"):window.index("// Element offset")],
        paged=paged[paged.index("__device__ __forceinline__ int paged_keys"):paged.index("__device__ __forceinline__ WindowSeq window_seq(const PagedParams")],
        walk=kernel[kernel.index("struct Seq {"):kernel.index("__device__ __forceinline__ void ldmatrix4(")],
        constants="\n".join(re.findall(r"^constexpr int k(?:BlockCost|MinPlaces) = [^;]*;", kernel, re.M)))
    built = {}
    for rows in (16, 32, 48, 64):
        d = tmp_path_factory.mktemp("shares")
        src, exe = str(d / "shares.cpp"), str(d / "shares")
        with open(src, "w") as f:
            f.write(SOURCE % dict(parts, rows=rows))
        r = subprocess.run([gxx, "-std=c++17", "-O1", "-w", src, "-o", exe], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        built[rows] = exe

    def run(rows, *args):
        r = subprocess.run([built[rows], *map(str, args)], capture_output=True, text=True)
        assert r.returncode == 0, (args, r.stdout)
        return int(r.stdout.split()[1])
    return run


@pytest.mark.parametrize("rows", [16, 32, 48, 64])
@pytest.mark.parametrize("seed", range(60))
def test_shares_cover_every_key_of_every_row_once(replay, rows, seed):
    rng = random.Random(seed)
    heads, kv = rng.choice(((1, 1), (4, 4), (8, 1), (6, 2), (8, 2)))
    n = rng.choice((1, 1, 2, 5, 17))
    most_q = rng.choice((1, 4, 40))
    lengths = []
    for _ in range(n):
        k = rng.choice((0, 1, rng.randrange(1, 70), rng.randrange(1, 3000)))
        lengths += [rng.choice((0, 1, rng.randrange(1, most_q + 1))), k]
    window = rng.choice(((-1, -1, 0), (-1, 0, 0), (0, 0, 3), (rng.randrange(200), 0, rng.randrange(100)), (rng.randrange(200), rng.randrange(50), 0),
                         (2 ** 30, 2 ** 30, 7)))
    ctas = replay(rows, n, rng.choice((1, 3, 40, 296)), heads, kv, *window, rng.choice((4, 5, 6, 8)), rng.choice((most_q, 3)), *lengths)
    assert ctas <= 296


def test_one_long_sequence_goes_to_all(replay):
    assert replay(16, 1, 296, 8, 1, -1, 0, 0, 6, 16, 1, 100000) == 296
    assert replay(16, 1, 296, 8, 8, -1, 0, 0, 4, 16, 1, 63) <= 12
    assert replay(16, 1, 296, 8, 1, -1, 0, 0, 4, 16, 1, 0) == 1
