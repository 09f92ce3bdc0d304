"""Which blocks the kernel of tiles over pages takes, and what it leaves for the launch that joins, run on the host.

Checked: every block of 256 rows is placed once, with as many parts as its keys are split into; the parts' keys that a row sees are those it
sees, once each; their states lie side by side in scratch; and the records of the blocks that are joined are the same from any CTA, since
none of them is sure to start: another may take its block before."""
import random

import pytest

from tests.cuda_on_host import compiled, cut, output, source

PROGRAM = r"""
#define DTB_QUERIES_LAST (-2147483647 - 1)
struct CUtensorMap { int x; };
namespace dtb {
namespace flash {}
constexpr int kBM = 128, kQT = 2, kBN = 128;
@flash@
@window@
@paged@
void grid_launch_dependents() {}
void st_relaxed16(void* to, int a, int b, int c, int d) { const int v[4] = {a, b, c, d}; std::memcpy(to, v, 16); }
@plan@
constexpr int kKeys = 64, kBlockCost = 2, kMinPlaces = 2, kMostCluster = 8;
struct alignas(16) Join { int x[8]; };
@rows_plan@
@walk@
@item@
}
using namespace dtb;
@host_plan@
struct DeviceInfo { int sm_count; };
int refuse(int line) { std::printf("failed: refused, line %d\n", line); std::exit(1); }
#define fail(...) refuse(__LINE__)
int main(int argc, char** argv) {
  std::vector<int> a;
  for (int i = 1; i < argc; ++i) a.push_back(std::atoi(argv[i]));
  const int cta = a[0], num_heads = a[1], num_kv_heads = a[2], head_dim = 64, left = a[3], right = a[4], nseg = a[6];
  const bool packed = true;
  PagedParams p = {};
  p.kv_heads = num_kv_heads; p.left = left; p.right = right; p.sinks = left < 0 ? 0 : a[5];
  p.q_start = kQueriesLast; p.splits = 1;
  p.page_shift = 4; p.key_align = left < 0 ? 16 << (cta % 4) : 16;
  std::vector<int32_t> cu(1, 0), lens;
  int seqlen_q = 0;
  for (int b = 0; b < nseg; ++b) {
    cu.push_back(cu.back() + a[7 + 2 * b]);
    lens.push_back(a[8 + 2 * b]);
    seqlen_q = max(seqlen_q, a[7 + 2 * b]);
    p.columns = max(p.columns, (lens[b] >> p.page_shift) + 1);
  }
  const int64_t total_q = cu.back();
  const int seqlen_k = p.columns << p.page_shift;
  p.f.cu_q = cu.data(); p.seqlens_k = lens.data(); p.f.nseg = nseg; p.f.seqlen_q = seqlen_q; p.f.total_q = total_q; p.f.num_heads = num_heads;
  const DeviceInfo info = {148};
  const DeviceInfo* d = &info;
  const PagedPlan plan = plan_paged(nseg, seqlen_q, seqlen_k, total_q, num_heads, num_kv_heads, head_dim, d->sm_count);
  if (!plan.tiles) { std::printf("0 0 0\n"); return 0; }
  const bool mixed = paged_mixed(plan, packed, nseg, seqlen_q, total_q);
  p.few_rows = mixed ? plan.few_rows : -1;
  p.real = p.f;
  PagedParams t = p;
  t.pack_shift = plan.pack_shift;
  [&]() -> int {
@launch@
    return 0;
  }();
  std::vector<TileJoin> joins(t.most_states / 2 + 1);
  std::memset(joins.data(), 0x7f, joins.size() * sizeof(TileJoin));
  t.joins = joins.data();
  const int grid = t.blocks;
  CHECK(t.planned == (nseg <= kPlanSeqs) && (t.planned || (grid <= 148 && t.most_states == 0)));
  // who is placed where
  std::map<std::tuple<int, int, int>, std::vector<Item>> blocks;      // (sequence, head of the tiles, first row) -> its parts
  std::set<int> states;
  int empty = 0;
  // one CTA's plan for all places of the grid, or each CTA's own places
  for (int c = t.planned ? cta % grid : 0, end = t.planned ? c + 1 : grid; c < end; ++c) {
   launch_block(c, grid, kPlanThreads, [&] { plan_blocks(t); });
   CHECK(claims_blocks(t) == (t.planned != 0));
   for (int place = t.planned ? 0 : c;; ++place) {
    if (t.planned && place == grid) break;
    int bx = place, by = 0, bz = 0, splits = t.splits, state = -1;
    bool asked = true;
    const PagedParams& p = t;
@block@
      CHECK(by < t.f.num_heads && seg < nseg && part < splits);
      CHECK((splits > 1) == (state >= 0) && w.part == (state >= 0));
      if (state >= 0) CHECK(state < t.most_states && states.insert(state).second && w.q_begin + w.q0 == state * 256);
      auto& parts = blocks[{seg, by, w.q0}];
      parts.push_back(w);
      CHECK(int(parts.size()) <= splits);
    } else {
      ++empty;
    }
    if (!t.planned) {
      if (!next_place(t, place)) break;
      --place;
    }
   }
  }
  // (a CTA without a block of its own begins at none)
  CHECK(t.planned || empty <= grid);
  const int group = num_heads / num_kv_heads, pack = 1 << t.pack_shift;
  size_t count = 0, split = 0;
  for (int b = 0; b < nseg; ++b) {
    const int n = cu[b + 1] - cu[b];
    if (n <= p.few_rows) continue;
    for (int head = 0; head < num_heads / pack; ++head)
      for (int q0 = 0; q0 < n * pack; q0 += 256) {
        const auto found = blocks.find({b, head, q0});
        CHECK(found != blocks.end());
        ++count;
        const auto& parts = found->second;
        const TileJoin* record = nullptr;
        for (int i = 0; i < t.most_states / 2; ++i)
          if (joins[i].rows != 0 && joins[i].seg == b && joins[i].head == head && joins[i].q0 == q0) { CHECK(record == nullptr); record = &joins[i]; }
        CHECK((record != nullptr) == (parts.size() > 1));
        if (record != nullptr) {
          ++split;
          CHECK(record->rows == min(256, n * pack - q0) && record->q_begin == cu[b] * pack && record->parts == int(parts.size()));
          std::set<int> own;
          for (const Item& w : parts) own.insert((w.q_begin + w.q0) / 256);
          for (int i = 0; i < record->parts; ++i) CHECK(own.count(record->state + i));
        } else {
          CHECK(parts[0].q_begin == cu[b] * pack && parts[0].part == 0);
        }
        if (head != 0 || nseg > 1000) continue;
        for (int i = q0; i < min(q0 + 256, n * pack); i += 37) {
          const int x = lens[b] - n + (i >> t.pack_shift);
          std::vector<int> times(lens[b] + 1, 0);
          for (const Item& w : parts) {
            const WindowSpan s = window_span(w.from, w.to, w.sinks, w.k_end, w.k_floor, i >> t.pack_shift);
            for (int j = 0; j < s.first; ++j) { CHECK(j < w.walk.first); ++times[j]; }
            for (int j = s.lo; j < s.hi; ++j) { CHECK(j >= w.walk.lo + w.walk.front && j < w.walk.lo + w.walk.win); ++times[j]; }
            CHECK(w.walk.lo % t.key_align == 0 || w.walk.win == 0);
          }
          for (int j = 0; j < lens[b]; ++j) CHECK(times[j] == ((right < 0 || j <= x + right) && (left < 0 || j >= x - left || j < p.sinks) ? 1 : 0));
        }
      }
  }
  CHECK(count == blocks.size());
  for (int i = 0; i < t.most_states / 2; ++i) CHECK(joins[i].rows >= 0 && joins[i].rows <= 256);
  std::printf("%d %d %d\n", int(count), int(split), grid);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    kernel, window, paged, fwd, rows, capi = map(source, ("flash_window_sm100.cu", "flash_window.cuh", "flash_paged.cuh", "flash_fwd_sm100.cuh", "flash_paged_rows.cu", "capi.cu"))
    parts = dict(
        flash=cut(fwd, "struct FlashParams", "// With p.overlap_previous"),
        window=cut(window, "constexpr int kQueriesLast", "// Tensor maps of q, k and v"),
        paged=cut(paged, "struct PagedParams", "__device__ __forceinline__ void tma_load_4d") + cut(paged, "struct PagedRowsPlan", "// (rows of a key head's longest"),
        plan=cut(paged, "constexpr int kPlanSeqs", "// Where row R of a head"),
        rows_plan=cut(rows, "PagedRowsPlan plan_paged_rows(", "namespace {"),
        walk=cut(kernel, "struct Walk {", "// A block"), item=cut(kernel, "struct Item {", "static_assert(sizeof(Item)"),
        host_plan=cut(capi, "struct PagedPlan {", "static int check_paged_shape") + cut(capi, "static bool paged_mixed", "DTB_API int dtb_flash_paged_launches"),
        launch=cut(capi, "    t.f.num_heads = num_heads >> plan.pack_shift;", "    t.parts.out = scratch;"),
        block=cut(kernel, "          Item w;\n", "            const Walk walk = w.walk;"))
    return compiled(tmp_path_factory.mktemp("tiles"), PROGRAM, **parts)


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (700, 0, 100), (300, 50, 0), (5, 0, 3)]


@pytest.mark.parametrize("cta", [0, 1, 147])
@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("new,lens,heads", [
    ([200], [30000], (32, 32)), ([300, 2], [9000, 2], (4, 2)), ([1350, 1350], [3000, 5000], (6, 6)), ([700] * 9, [4000] * 9, (8, 2)), ([45] * 3, [9000, 300, 77], (16, 1)),
    ([2500, 1, 1, 800], [2500, 7000, 9, 3000], (8, 2)), ([257], [257], (3, 1))])
def test_every_block_is_placed_once_and_its_parts_are_joined(program, new, lens, heads, window, cta):
    count, split, _ = map(int, output(program, cta, *heads, *window, len(new), *[x for pair in zip(new, lens) for x in pair]).split())
    assert count > 0


@pytest.mark.parametrize("new,lens", [([200, 1, 130] * 100, [220, 90, 140] * 100), ([8192] + [1] * 299, [9000] + [500] * 299), ([1] * 299 + [5000], [500] * 299 + [5000]),
                                      ([0] * 600 + [700, 0, 0, 300] + [0] * 600, [40] * 600 + [800, 3, 0, 300] + [40] * 600), ([70] * 257, [100] * 257),
                                      ([1] * 8000 + [20000] + [1] * 8383, [3] * 16384)])
@pytest.mark.parametrize("heads", [(4, 1), (6, 6)])
def test_more_sequences_than_are_planned(program, new, lens, heads):
    for window in WINDOWS[:1] if len(new) > 2000 else WINDOWS:
        count, split, grid = map(int, output(program, 0, *heads, *window, len(new), *[x for pair in zip(new, lens) for x in pair]).split())
        assert count > 0 and split == 0 and grid <= 148


def test_records_of_split_blocks_come_from_any_of_the_ctas(program):
    assert len({output(program, cta, 32, 32, -1, -1, 0, 1, 200, 60000) for cta in range(0, 64, 4)}) == 1
    assert int(output(program, 3, 32, 32, -1, -1, 0, 1, 200, 60000).split()[1]) == 32


@pytest.mark.parametrize("seed", range(40))
def test_batches_at_random(program, seed):
    rng = random.Random(seed)
    heads = rng.choice(((1, 1), (4, 4), (8, 1), (6, 2), (8, 2), (7, 1)))
    n = rng.choice((1, 2, 7, 40, 256, 257, 700))
    most = rng.choice((20, 300, 1500)) if n < 40 else 300
    pairs = [x for _ in range(n) for x in (rng.choice((0, 1, rng.randrange(most), rng.randrange(most))), rng.choice((0, rng.randrange(100), rng.randrange(6000))))]
    output(program, rng.randrange(200), *heads, *rng.choice(WINDOWS), n, *pairs)
