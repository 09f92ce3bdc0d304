"""The kernel that makes tables of pages longer, run on the host over numbers of rows that no buffer is made for here."""
import pytest

from tests.cuda_on_host import compiled, cut, output, source

PROGRAM = r"""
int64_t tokens;
struct Slots {                            // notes where it is written, and holds nothing
  alignas(16) static int32_t sink[4];
  static int64_t stored;
  int32_t* operator+(int64_t i) const { CHECK(i >= 0 && i % 4 == 0 && i + 4 <= tokens); stored += 4; return sink; }
  int32_t& operator[](int64_t i) const { CHECK(i >= 0 && i < tokens); ++stored; return sink[0]; }
};
alignas(16) int32_t Slots::sink[4];
int64_t Slots::stored;
struct ExtendParams {
  int32_t* table;
  const int32_t *seqlens, *new_lens, *free_pages, *free_count;
  Slots slots;
  int32_t *cu_seqlens, *seqlens_out, *count_out, *missing;
  int streams, columns, pages, page_shift, tokens;
};
constexpr int kExtendThreads = 512;
int s_mem_[1 << 10];
@helpers@
@kernel@
int main(int, char** argv) {
  tokens = std::atoll(argv[1]);
  const int ctas = std::atoi(argv[2]), free_pages_count = std::atoi(argv[3]);
  int32_t table[8] = {0, -1, -1, -1, -1, -1, -1, -1}, lens[2] = {16, 0}, news[2] = {20, 3}, free_pages[8] = {7, 6, 5, 4, 3, 2, 1, 0}, count = free_pages_count;
  int32_t cu[3], out[2], count_out, missing;
  const ExtendParams p = {table, lens, news, free_pages, &count, {}, cu, out, &count_out, &missing, 2, 4, 8, 4, int(tokens)};
  for (int x : {0, ctas - 1}) launch_block(x, ctas, kExtendThreads, [&] { extend_pages_kernel(p); });
  std::printf("%lld %d %d\n", (long long)Slots::stored, missing, cu[2]);
}
"""


@pytest.fixture(scope="module")
def extend(tmp_path_factory):
    text = source("pages.cu")
    kernel = cut(text, "__global__ void __launch_bounds__(kExtendThreads) extend_pages_kernel", "// The pages [jb, je) of a stream go")
    kernel = kernel.replace("extern __shared__ int s_mem[];", "int* s_mem = s_mem_;")
    helpers = cut(text, "template <typename T>\n__device__ __forceinline__ T warp_inclusive", "}  // namespace")
    return compiled(tmp_path_factory.mktemp("extend"), PROGRAM, helpers=helpers, kernel=kernel)


@pytest.mark.parametrize("tokens", [2 ** 31 - 5, 2 ** 31 - 8, 2 ** 31 - 300000])
@pytest.mark.parametrize("free", [6, 1])                 # (room for the three pages, and not)
def test_rows_up_to_the_largest_number_are_stored_once(extend, tokens, free):
    ctas = 148
    stored, missing, new = map(int, output(extend, tokens, ctas, free).split())
    assert (missing, new) == ((0, 23) if free == 6 else (2, 0))
    # two of the CTAs: those threads' rows, four at a time or, of a call that was refused, one
    step = 4 if free == 6 else 1
    threads = 512
    expected = sum(max(0, min(tokens, at + step * threads) - at) for x in (0, ctas - 1) for at in range(x * step * threads, tokens, step * threads * ctas))
    assert stored == expected
