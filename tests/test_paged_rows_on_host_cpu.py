"""Attention of few rows over pages, shares and join, run on the host with the products left out: every score is 0 and every value too, so that a
row's lse is the logarithm of the number of keys it sees.

CTAs that begin after a failure elsewhere, or give up a wait, are played, and the status word is clear again when the launch that joins looks at
it: what that launch follows has to be what this one has left for it, whatever the scratch held before, and no row is written that a
CTA with a part of it has not finished."""
import re

import pytest

from tests.cuda_on_host import compiled, cut, output, source

PROGRAM = r"""
struct CUtensorMap { int x; };
@flash@
@window@
@paged@
constexpr float kLn2 = 0.6931471805599453f, kRescaleThreshold = 8.0f;
namespace flash {
@lse@
@weights@
}
using flash::lse_index; using flash::merge_weights;
namespace cooperative_groups {
struct cluster_group {
  unsigned num_blocks() const { return 1; }
  unsigned block_rank() const { return 0; }
  void sync() const {}
  template <class T> T* map_shared_rank(T* x, int) const { return x; }
};
inline cluster_group this_cluster() { return {}; }
}
alignas(1024) uint8_t shared_memory[232448];
uint32_t smem_u32(const void* x) { return uint32_t(uintptr_t(x)); }
void mbar_init(uint64_t*, int) {}
void mbar_arrive(uint64_t*) {}
void mbar_expect_tx(uint64_t*, int) {}
void fence_mbar_init() {}
void fence_proxy_async_smem() {}
void prefetch_tmap(const void*) {}
void prefetch_tmap(const PagedMap*) {}
void grid_launch_dependents() {}
void grid_dependency_wait() {}
void tma_load_4d(void*, const CUtensorMap*, uint64_t*, int, int, int, int) {}
void ldmatrix4(uint32_t, uint32_t (&r)[4]) { r[0] = r[1] = r[2] = r[3] = 0; }
void ldmatrix4_trans(uint32_t, uint32_t (&r)[4]) { r[0] = r[1] = r[2] = r[3] = 0; }
void mma16816(float (&)[4], const uint32_t (&)[4], uint32_t, uint32_t) {}
void __nanosleep(int) {}
template <int N> void math_warps_sync() { named_barrier(1, N); }
float ex2(float x) { return std::exp2(x); }
float max3(float a, float b, float c) { return std::fmax(a, std::fmax(b, c)); }
uint64_t pack2(float a, float b) { uint64_t r; const float v[2] = {a, b}; std::memcpy(&r, v, 8); return r; }
void unpack2(uint64_t x, float& a, float& b) { float v[2]; std::memcpy(v, &x, 8); a = v[0]; b = v[1]; }
uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) { float a, b, c, d, e, f; unpack2(x, a, b); unpack2(y, c, d); unpack2(z, e, f); return pack2(std::fma(a, c, e), std::fma(b, d, f)); }
uint64_t add2(uint64_t x, uint64_t y) { float a, b, c, d; unpack2(x, a, b); unpack2(y, c, d); return pack2(a + c, b + d); }
uint64_t exp2_mufu2(uint64_t x) { float a, b; unpack2(x, a, b); return pack2(std::exp2(a), std::exp2(b)); }
uint32_t pack_bf16x2(float, float) { return 0; }
// waits of a CTA's warp, until the one that gives up
int waits_left = -1, gives_up_warp;
bool warp_wait_or_abort(uint64_t*, uint32_t, int* status, int code) {
  const bool mine = (int(threadIdx.x) >> 5) == gives_up_warp, now = mine && waits_left == 0;
  if (__any_sync(0xffffffffu, now || *status != 0)) {
    if (now) *status = code;
    return false;
  }
  if (mine && waits_left > 0 && (threadIdx.x & 31) == 0) --waits_left;
  __syncwarp();
  return true;
}
@kernels@
constexpr int D = @D@, WM = @WM@, R = 16 * WM;
uint32_t state_;
int rnd(int n) { state_ = state_ * 1664525u + 1013904223u; return int((uint64_t(state_ >> 8) * n) >> 24); }
int main(int, char** argv) {
  state_ = std::atoi(argv[1]) * 7919 + 12345;
  const int trouble = std::atoi(argv[2]);          // 0: none; 1: CTAs begin after a failure; 2: one gives up a wait
  PagedParams p = {};
  const int kinds[][2] = {{1, 1}, {4, 4}, {8, 1}, {6, 2}, {8, 2}}, k = rnd(5), n = 1 + rnd(4), most_q = 1 + rnd(9);
  const int H = kinds[k][0], Hk = kinds[k][1], group = H / Hk;
  std::vector<int32_t> cu(1, 0), lens;
  for (int b = 0; b < n; ++b) {
    cu.push_back(cu.back() + (rnd(6) ? 1 + rnd(most_q) : 0));
    lens.push_back(rnd(5) ? rnd(900) : rnd(3));
    p.f.seqlen_q = max(p.f.seqlen_q, cu[b + 1] - cu[b]);
  }
  if (std::atoi(argv[3])) p.f.seqlen_q = max(1, p.f.seqlen_q / 2);          // of longer sequences the rest is left out
  const int T = cu.back(), extra = rnd(3);
  if (T == 0) { std::printf("0 0 0\n"); return 0; }
  const int windows[][3] = {{-1, -1, 0}, {-1, 0, 0}, {0, 0, 3}, {100, 0, 40}, {150, 7, 0}}, w = rnd(5);
  int status = 0;
  p.f.status = &status;
  p.f.num_heads = H; p.kv_heads = Hk; p.f.nseg = n; p.f.total_q = T + extra; p.f.out_tok_stride = H * D; p.f.lse_layout = rnd(2);
  p.f.scale_log2 = 0.125f * 1.4426950408889634f;
  p.left = windows[w][0]; p.right = windows[w][1]; p.sinks = windows[w][2];
  p.q_start = kQueriesLast; p.splits = 1;
  p.page_shift = 4 + rnd(3); p.columns = (900 >> p.page_shift) + 1; p.pages = 1000; p.few_rows = 1000;
  p.box_rows = p.key_align = min(1 << p.page_shift, 64);
  std::vector<int32_t> table(n * p.columns, 3);
  std::vector<uint16_t> q((T + extra) * H * D, 0);
  std::vector<float> out((T + extra) * H * D, 7.f), lse((T + extra) * H, 7.f);
  p.f.cu_q = cu.data(); p.seqlens_k = lens.data(); p.table = table.data(); p.q = q.data(); p.q_tok = H * D; p.f.out = out.data(); p.f.lse = lse.data();
  // as the launcher does
  const int ctas = 2 + rnd(14), blocks_of_longest = (p.f.seqlen_q * group + R - 1) / R, units = blocks_of_longest * Hk * n;
  const bool by_blocks = units < ctas;
  const int row_blocks = by_blocks ? blocks_of_longest : 0;
  const size_t bytes = ctas * (sizeof(Join) + 2 * R * (8 + D * 4)), guard = 4096;
  std::vector<uint4> memory((bytes + 2 * guard) / 16 + 1);
  std::memset(memory.data(), 0x7f, memory.size() * 16);
  uint8_t* scratch = reinterpret_cast<uint8_t*>(memory.data()) + guard;
  std::set<int> late;
  const int who = rnd(ctas), from = rnd(5);
  gives_up_warp = rnd(Cfg<D, WM>::kThreads / 32);
  PagedMap map = {};
  int gave_up = -1;
  for (int c = 0; c < ctas; ++c) {
    if (trouble == 1 && rnd(3) == 0) late.insert(c);
    status = late.count(c) ? 5 : 0;
    waits_left = trouble == 2 && c == who ? from : -1;
    launch_block(c, ctas, Cfg<D, WM>::kThreads, [&] { flash_paged_rows_kernel<D, WM, false>(map, map, p, scratch, row_blocks); });
    if (status != 0 && !late.count(c)) gave_up = c;
  }
  status = 0;
  const int joins = by_blocks ? units : ctas - 1;
  for (int j = 0; j < joins; ++j) {
    // (rows beside one another are tested on the device; here a CTA takes them all)
    launch_block(j, joins, 128, [&] { flash_paged_join_kernel<D, R>(p, scratch, ctas, row_blocks); });
  }
  for (size_t i = 0; i < guard; ++i) CHECK(scratch[-1 - int(i)] == 0x7f && scratch[bytes + i] == 0x7f);
  // who has parts of which block
  long long all = 0;
  for (int b = 0; b < n; ++b) { const Seq s = make_seq<R>(p, b); all += (long long)s.blocks * Hk * places_of(s); }
  const Shares shares(all, ctas);
  long long at = 0;
  int written = 0, kept = 0, joined = 0;
  for (int b = 0; b < n; ++b) {
    const Seq s = make_seq<R>(p, b);
    for (int unit = 0; unit < s.blocks * Hk; ++unit, at += places_of(s)) {
      const int c0 = shares.of(at + kBlockCost), c1 = shares.of(at + places_of(s) - 1);
      bool lost = false;
      for (int c = c0; c <= c1; ++c) lost = lost || late.count(c);
      const bool maybe = gave_up >= c0 && gave_up <= c1;
      joined += c1 > c0;
      const Block block = make_block<R>(p, s, unit);
      int written_rows = 0;
      for (int r = 0; r < block.rows; ++r) {
        const int row = block.row0 + r, i = row / group, head = block.kv_head * group + row % group, tok = cu[b] + i, x = lens[b] - (cu[b + 1] - cu[b]) + i;
        int seen = 0;
        for (int j = 0; j < lens[b]; ++j) seen += (p.right < 0 || j <= x + p.right) && (p.left < 0 || j >= x - p.left || j < p.sinks);
        float& l = lse[p.f.lse_layout == 1 ? tok * H + head : head * (T + extra) + tok];
        bool untouched = l == 7.f, right = seen == 0 ? l == -INFINITY : std::fabs(l - std::log(float(seen))) < 1e-4f;
        for (int d = 0; d < D; ++d) { float& o = out[(tok * H + head) * D + d]; untouched = untouched && o == 7.f; right = right && o == 0.f; o = 9.f; }
        CHECK(lost ? untouched : maybe ? untouched || right : right);
        written_rows += right; kept += untouched;
        l = 9.f;
      }
      written += written_rows;
    }
  }
  // (each row was looked at once, and those left out and behind the last one are as they were)
  int b = 0;
  for (int t = 0; t < T + extra; ++t)
    for (int h = 0; h < H; ++h) {
      while (b < n && t >= cu[b + 1]) ++b;
      const float want = b < n && t - cu[b] < p.f.seqlen_q ? 9.f : 7.f;
      CHECK(lse[p.f.lse_layout == 1 ? t * H + h : h * (T + extra) + t] == want);
      for (int d = 0; d < D; ++d) CHECK(out[(t * H + h) * D + d] == want);
    }
  std::printf("%d %d %d\n", written, kept, joined);
}
"""

SIZES = [(64, 1), (64, 2), (64, 3), (64, 4), (128, 1)]


@pytest.fixture(scope="module")
def programs(tmp_path_factory):
    kernel, window, paged, common, fwd = map(source, ("flash_paged_rows.cu", "flash_window.cuh", "flash_paged.cuh", "flash_common.cuh", "flash_fwd_sm100.cuh"))
    kernels = cut(kernel, "constexpr int kKeys", "// Joins the parts of blocks whose keys the kernel of tiles split")
    kernels = kernels.replace(cut(kernels, "__device__ __forceinline__ void ldmatrix4(", "__device__ __forceinline__ float quad_max"), "")
    kernels = re.sub(r"template <int N>\n__device__ __forceinline__ void math_warps_sync\(\)[^\n]*\n", "", kernels)
    kernels = kernels.replace("extern __shared__ uint8_t smem_raw[];", "uint8_t* smem_raw = shared_memory;").replace("}  // namespace\n", "")
    parts = dict(
        flash=cut(fwd, "struct FlashParams", "// With p.overlap_previous"),
        window=cut(window, "constexpr int kQueriesLast", "// Tensor maps of q, k and v"),
        paged=cut(paged, "struct PagedParams", "__device__ __forceinline__ void tma_load_4d"),
        lse=cut(common, "__device__ __forceinline__ int64_t lse_index", "// A row of a (segment, head)"),
        weights=cut(common, "__device__ __forceinline__ void merge_weights", "// Host: one launch"), kernels=kernels)
    return {size: compiled(tmp_path_factory.mktemp("rows"), PROGRAM, D=str(size[0]), WM=str(size[1]), **parts) for size in SIZES}


@pytest.mark.parametrize("trouble", [0, 1, 2])
@pytest.mark.parametrize("size", SIZES)
def test_a_launch_that_joins_follows_what_this_one_left(programs, size, trouble):
    written = kept = joined = 0
    for seed in range(12):
        a, b, c = map(int, output(programs[size], seed, trouble, 0).split())
        written, kept, joined = written + a, kept + b, joined + c
    assert written > 0 and joined > 0 and (kept > 0) == (trouble > 0)


@pytest.mark.parametrize("size", SIZES)
def test_rows_that_are_kept_of_a_longer_sequence_stay_at_their_positions(programs, size):
    for seed in range(12):
        output(programs[size], seed, 0, 1)
