// Tables of pages, made longer and shorter on the device, and tokens written into their slots.
//
// Stream b of length l_b holds ceil(l_b / P) pages, page j its tokens [j P, (j + 1) P).  With n_b new tokens it needs
//     need_b = ceil((l_b + n_b) / P) - ceil(l_b / P)
// more, which are taken from the end of the list of free pages, the streams one after another: the k-th page of all, k = sum_{a < b} need_a + j,
// is free[count - 1 - k].  Both prefix sums (of n and of need) are formed by every CTA for itself, so that no CTA waits for another and one
// launch does all; tokens and pages find their stream by a search in them.  Bound by latency: a launch, three dependent reads and the sums (one token
// for each of 7 streams 4.4 us, 1350 for each of 256 6.2, one launch after another; an empty kernel takes 2).
#include "pages.cuh"
#include "row_access.cuh"

#include <cooperative_groups.h>

#include <mutex>

namespace dtb {

namespace {

constexpr int kExtendThreads = 512;
constexpr int kReleaseThreads = 1024;
constexpr int kWriteThreads = 128;

template <typename T>
__device__ __forceinline__ T warp_inclusive(T v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const T u = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += u;
  }
  return v;
}

// The largest i of [0, n) with at[i] <= x; at[0] <= x, at rises (not strictly).
__device__ __forceinline__ int last_not_above(const int* at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int tokens, int shift) { return static_cast<int>((static_cast<uint32_t>(tokens) + (1u << shift) - 1u) >> shift); }

}  // namespace

__global__ void __launch_bounds__(kExtendThreads) extend_pages_kernel(const ExtendParams p) {
  extern __shared__ int s_mem[];
  int* s_cu = s_mem;                     // [streams + 1] first new token of each stream
  int* s_pg = s_cu + p.streams + 1;      // [streams + 1] first new page
  int* s_len = s_pg + p.streams + 1;     // [streams]
  constexpr int kWarps = kExtendThreads / 32;
  __shared__ long long s_sums[2][kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = *p.free_count;
  const long long capacity = static_cast<long long>(p.columns) << p.page_shift;      // below 2^31

  // this thread's streams, one after another
  const int per = (p.streams + kExtendThreads - 1) / kExtendThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, p.streams), b1 = min(b0 + per, p.streams);
  long long tokens = 0, pages = 0;
  bool bad = count < 0 || count > p.pages;
  for (int b = b0; b < b1; ++b) {
    const int len = p.seqlens[b], n = p.new_lens[b];
    if (len < 0 || n < 0 || static_cast<long long>(len) + n > capacity) {
      bad = true;
      continue;
    }
    tokens += n;
    pages += pages_of(len + n, p.page_shift) - pages_of(len, p.page_shift);
  }
  const long long t_in = warp_inclusive(tokens), p_in = warp_inclusive(pages);
  if (lane == 31) {
    s_sums[0][warp] = t_in;
    s_sums[1][warp] = p_in;
  }
  bad = __syncthreads_or(bad);
  long long t_at = t_in - tokens, p_at = p_in - pages, t_all = 0, p_all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      t_at += s_sums[0][w];
      p_at += s_sums[1][w];
    }
    t_all += s_sums[0][w];
    p_all += s_sums[1][w];
  }
  bad = bad || t_all > p.tokens;
  const bool refused = bad || p_all > count;
  const bool first_cta = blockIdx.x == 0;
  for (int b = b0; b < b1; ++b) {
    const int len = p.seqlens[b], n = refused ? 0 : p.new_lens[b];
    s_cu[b] = static_cast<int>(t_at);
    s_pg[b] = static_cast<int>(p_at);
    s_len[b] = len;
    if (first_cta) {
      p.cu_seqlens[b] = refused ? 0 : static_cast<int>(t_at);
      p.seqlens_out[b] = len + n;
    }
    t_at += n;
    if (!refused) p_at += pages_of(len + n, p.page_shift) - pages_of(len, p.page_shift);
  }
  if (threadIdx.x == 0) {
    s_cu[p.streams] = static_cast<int>(t_all);
    s_pg[p.streams] = static_cast<int>(p_all);
    if (first_cta) {
      p.cu_seqlens[p.streams] = refused ? 0 : static_cast<int>(t_all);
      *p.count_out = refused ? count : count - static_cast<int>(p_all);
      const long long lack = p_all - count;
      *p.missing = bad ? -1 : static_cast<int>(lack > 0 ? lack : 0);
    }
  }
  __syncthreads();

  const int id = blockIdx.x * kExtendThreads + threadIdx.x, threads = gridDim.x * kExtendThreads;
  // (a step from the last of nearly 2^31 rows would wrap around)
  auto next = [&](int t, int step) { return t < p.tokens - step ? t + step : p.tokens; };
  if (refused) {
    for (int t = id; t < p.tokens; t = next(t, threads)) p.slots[t] = -1;
    return;
  }
  // four tokens of a thread, which mostly are of one stream
  const int n_tokens = static_cast<int>(t_all), mask = (1 << p.page_shift) - 1;
  for (int t0 = 4 * id; t0 < p.tokens; t0 = next(t0, 4 * threads)) {
    int slot[4] = {-1, -1, -1, -1};
    if (t0 < n_tokens) {
      int b = last_not_above(s_cu, p.streams, t0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + i;
        if (t < n_tokens) {
          while (t >= s_cu[b + 1]) ++b;
          const int len = s_len[b], x = len + t - s_cu[b], j = x >> p.page_shift, first = pages_of(len, p.page_shift);
          const int page = j < first ? p.table[static_cast<int64_t>(b) * p.columns + j] : p.free_pages[count - 1 - (s_pg[b] + j - first)];
          if (page >= 0 && page < p.pages) slot[i] = (page << p.page_shift) + (x & mask);
        }
      }
    }
    if (t0 + 4 <= p.tokens) {
      *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
      for (int i = 0; t0 + i < p.tokens; ++i) p.slots[t0 + i] = slot[i];
    }
  }
  for (int k = id; k < static_cast<int>(p_all); k += threads) {
    const int b = last_not_above(s_pg, p.streams, k);
    p.table[static_cast<int64_t>(b) * p.columns + pages_of(s_len[b], p.page_shift) + k - s_pg[b]] = p.free_pages[count - 1 - k];
  }
}

// The pages [jb, je) of a stream go, as far as they are there.
struct Going {
  int jb, je;
};
__device__ __forceinline__ Going going(const ReleaseParams& p, int b) {
  const int len = max(p.seqlens[b], 0), begin = max(p.begin[b], 0), end = p.end[b];
  Going g = {0, 0};
  if (begin >= end) return g;
  g.jb = pages_of(begin, p.page_shift);
  g.je = min(end >= len ? pages_of(len, p.page_shift) : end >> p.page_shift, p.columns);
  return g;
}

// A warp takes 256 entries of a stream at a time.  Counts first, then their prefix sums within the CTA and over the cluster, then the
// entries again with the places of those that go: in the order of streams and pages, whatever the number of CTAs.  (The list's order needs the sums
// over all streams, and a cluster has its barrier in hardware.)  Bound by latency: 96 streams of 1200 entries 9.3 us.
__global__ void __launch_bounds__(kReleaseThreads) release_pages_kernel(const ReleaseParams p, int pieces) {
  namespace cg = cooperative_groups;
  extern __shared__ int s_count[];       // [pieces of this CTA]
  __shared__ int s_warp[kReleaseThreads / 32], s_total;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kReleaseThreads / 32, kEntries = kReleaseColumns / 32;
  const int items = p.streams * pieces, per = (items + C - 1) / C;
  const int i0 = min(rank * per, items), n = min(per, items - i0);
  const int count = min(max(*p.free_count, 0), p.pages);
  auto entries = [&](int item, int& b, int& j0, uint32_t (&goes)[kEntries], int (&page)[kEntries], bool all) {
    b = item / pieces;
    j0 = item % pieces * kReleaseColumns;
    const Going g = going(p, b);
    int sum = 0;
    if (!all && (g.jb >= min(j0 + kReleaseColumns, p.columns) || g.je <= j0)) return 0;
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int j = j0 + i * 32 + lane;
      page[i] = -1;
      if (j < p.columns) page[i] = p.table[static_cast<int64_t>(b) * p.columns + j];
    }
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int j = j0 + i * 32 + lane;
      goes[i] = __ballot_sync(0xffffffffu, j >= g.jb && j < g.je && page[i] >= 0 && page[i] < p.pages);
      sum += __popc(goes[i]);
    }
    return sum;
  };
  uint32_t goes[kEntries];
  int page[kEntries], b, j0;
  for (int i = warp; i < n; i += kWarps) {
    const int sum = entries(i0 + i, b, j0, goes, page, false);
    if (lane == 0) s_count[i] = sum;
  }
  __syncthreads();
  // exclusive prefix sums, a run of pieces to a thread
  const int run = (n + kReleaseThreads - 1) / kReleaseThreads, r0 = min(static_cast<int>(threadIdx.x) * run, n), r1 = min(r0 + run, n);
  int sum = 0;
  for (int i = r0; i < r1; ++i) sum += s_count[i];
  const int inclusive = warp_inclusive(sum);
  if (lane == 31) s_warp[warp] = inclusive;
  __syncthreads();
  if (warp == 0) {
    const int mine = lane < kWarps ? s_warp[lane] : 0, upto = warp_inclusive(mine);
    if (lane < kWarps) s_warp[lane] = upto - mine;
    if (lane == kWarps - 1) s_total = upto;
  }
  __syncthreads();
  int at = s_warp[warp] + inclusive - sum;
  for (int i = r0; i < r1; ++i) {
    const int c = s_count[i];
    s_count[i] = at;
    at += c;
  }
  cluster.sync();
  int before = 0, all = 0;
  for (int r = 0; r < C; ++r) {
    const int t = *cluster.map_shared_rank(&s_total, r);
    if (r < rank) before += t;
    all += t;
  }
  cluster.sync();                        // nobody leaves while its shared memory is read; s_count is complete in this CTA
  const bool copies = p.table_out != p.table;
  for (int i = warp; i < n; i += kWarps) {
    if (!copies) {
      const int next = i + 1 < n ? s_count[i + 1] : s_total;
      if (next == s_count[i]) continue;
    }
    entries(i0 + i, b, j0, goes, page, true);
    int place = count + before + s_count[i];
#pragma unroll
    for (int e = 0; e < kEntries; ++e) {
      const int j = j0 + e * 32 + lane;
      const bool mine = (goes[e] >> lane) & 1;
      const int at_list = place + __popc(goes[e] & ((1u << lane) - 1u));
      if (mine && at_list < p.pages) p.free_pages[at_list] = page[e];
      if (j < p.columns && (mine || copies)) p.table_out[static_cast<int64_t>(b) * p.columns + j] = mine ? -1 : page[e];
      place += __popc(goes[e]);
    }
  }
  if (rank == 0) {
    for (int s = threadIdx.x; s < p.streams; s += kReleaseThreads) {
      const int len = p.seqlens[s], begin = max(p.begin[s], 0);
      p.seqlens_out[s] = p.end[s] >= len && begin < len ? begin : len;
    }
    if (threadIdx.x == 0) *p.count_out = min(count + all, p.pages);
  }
}

// A warp per token and tensor, 16 bytes to a lane and access, four of them under way.  HBM-bound: keys and values are read and written once
// (7219 tokens of 24 heads of 128: 31.6 us, 5.6 TB/s; 24 tokens of 8 heads 2.1, a launch).  What is written stays in L2, the attention behind it reads it.
__global__ void __launch_bounds__(kWriteThreads) write_pages_kernel(const WriteParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * (kWriteThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = w >> 1;
  if (t >= p.tokens) return;
  const int side = static_cast<int>(w & 1);
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.capacity) return;
  const uint16_t* src = (side ? p.src[1] : p.src[0]) + t * (side ? p.src_tok[1] : p.src_tok[0]);
  uint16_t* dst = (side ? p.dst[1] : p.dst[0]) + (slot >> p.page_shift) * (side ? p.dst_page[1] : p.dst_page[0]) +
                  (slot & ((1 << p.page_shift) - 1)) * (side ? p.dst_tok[1] : p.dst_tok[0]);
  const int64_t head = side ? p.dst_head[1] : p.dst_head[0];
  const int shift = p.head_shift - 3, n = p.heads << shift;
  for (int i0 = lane; i0 < n; i0 += 128) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + 32 * i < n) v[i] = ld_stream(src + (i0 + 32 * i) * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = i0 + 32 * i;
      if (at < n) *reinterpret_cast<uint4*>(dst + (at >> shift) * head + (at & ((1 << shift) - 1)) * 8) = v[i];
    }
  }
}

// More dynamic shared memory than 48 KB is asked for once per device.
static cudaError_t allow_shared(const void* kernel, int bytes, bool (&configured)[64], std::mutex& mu) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  if (!configured[dev & 63]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    configured[dev & 63] = true;
  }
  return cudaSuccess;
}

cudaError_t launch_extend_pages(const ExtendParams& p, int sm_count, cudaStream_t stream) {
  static bool configured[64] = {};
  static std::mutex mu;
  const int bytes = (3 * p.streams + 2) * 4;
  if (bytes > 48 * 1024 - 1024) {
    const cudaError_t e = allow_shared(reinterpret_cast<const void*>(extend_pages_kernel), (3 * kMostStreams + 2) * 4, configured, mu);
    if (e != cudaSuccess) return e;
  }
  const int64_t work = (static_cast<int64_t>(p.tokens) + 3) / 4;
  const int64_t blocks = (work + kExtendThreads - 1) / kExtendThreads;
  const unsigned grid = static_cast<unsigned>(blocks < 1 ? 1 : blocks > sm_count ? sm_count : blocks);
  extend_pages_kernel<<<grid, kExtendThreads, bytes, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_release_pages(const ReleaseParams& p, cudaStream_t stream) {
  static bool configured[64] = {};
  static std::mutex mu;
  const int pieces = (p.columns + kReleaseColumns - 1) / kReleaseColumns;
  const int64_t items = static_cast<int64_t>(p.streams) * pieces;
  const int C = items > kReleaseThreads / 32 ? kReleaseCtas : 1;
  const int64_t per = (items + C - 1) / C;
  if (per > kReleaseItems) return cudaErrorInvalidValue;
  const int bytes = static_cast<int>(per) * 4;
  if (bytes > 48 * 1024 - 1024) {
    const cudaError_t e = allow_shared(reinterpret_cast<const void*>(release_pages_kernel), kReleaseItems * 4, configured, mu);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(kReleaseThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, release_pages_kernel, p, pieces);
}

cudaError_t launch_write_pages(const WriteParams& p, cudaStream_t stream) {
  const int64_t warps = static_cast<int64_t>(p.tokens) * 2;
  write_pages_kernel<<<static_cast<unsigned>((warps * 32 + kWriteThreads - 1) / kWriteThreads), kWriteThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace dtb
