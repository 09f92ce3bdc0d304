"""Kernels compiled for the host: their threads as coroutines that meet at barriers, votes and shuffles.

`PREAMBLE` goes in front of a kernel's source; `launch_block(x, grid, threads, f)` runs f as every thread of block x.  Shared memory is
static, so blocks run one after another and find there what the one before has left, as they would on the device.  A block whose threads
wait for one another without end ends the program with an error."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ditango_b200", "csrc")

PREAMBLE = r"""
#include <ucontext.h>
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <set>
#include <tuple>
#include <type_traits>
#include <vector>
#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __grid_constant__
#define __launch_bounds__(...)
#define __shared__ static
#define __expf(x) std::exp(x)
#define __logf(x) std::log(x)
using std::max; using std::min;
#define CHECK(x) do { if (!(x)) { std::printf("failed: %s, line %d\n", #x, __LINE__); std::exit(1); } } while (0)
struct float2 { float x, y; };
struct alignas(16) float4 { float x, y, z, w; };
struct uint2 { uint32_t x, y; };
struct alignas(16) uint4 { uint32_t x, y, z, w; };
struct alignas(16) int4 { int x, y, z, w; };
inline float2 make_float2(float x, float y) { return {x, y}; }
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
inline uint2 make_uint2(uint32_t x, uint32_t y) { return {x, y}; }
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }
inline int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }
inline int __popc(uint32_t v) { return __builtin_popcount(v); }
inline int __float_as_int(float v) { int r; std::memcpy(&r, &v, 4); return r; }
inline float __int_as_float(int v) { float r; std::memcpy(&r, &v, 4); return r; }

struct Index { int x, y, z; };
Index threadIdx, blockIdx, gridDim, blockDim;
namespace host {
struct Thread { ucontext_t at; std::vector<char> stack; bool over; };
struct Meeting { int arrived = 0, turn = 0, any = 0, voted = 0; uint32_t votes = 0, vote_result = 0; };
std::vector<Thread> threads;
ucontext_t scheduler;
std::function<void()> body;
int now, alive;
uint64_t moves;                                  // meetings that came about, and threads that ended
std::map<std::pair<int, uint32_t>, Meeting> meetings;
uint64_t slots[1024];
inline void pause() { swapcontext(&threads[now].at, &scheduler); }
// All of `members` threads (0: all that are not over) come here.
inline Meeting& meet(int which, uint32_t mask, int members, int vote) {
  Meeting& m = meetings[{which, mask}];
  const int mine = m.turn;
  m.any |= vote != 0;
  if (vote) m.votes |= 1u << (now & 31);
  ++m.arrived;
  for (;;) {
    if (m.turn != mine) return m;
    if (m.arrived >= (members > 0 ? members : alive)) {
      m.voted = m.any, m.vote_result = m.votes;
      m.arrived = m.any = 0, m.votes = 0;
      ++m.turn, ++moves;
      return m;
    }
    pause();
  }
}
inline Meeting& warp(uint32_t mask, int vote) { return meet(100 + (now >> 5), mask, __builtin_popcount(mask), vote); }
inline void enter() { body(); threads[now].over = true; --alive; ++moves; pause(); }
}  // namespace host
inline void launch_block(int x, int grid, int n, std::function<void()> f) {
  using namespace host;
  blockIdx = {x, 0, 0}; gridDim = {grid, 1, 1}; blockDim = {n, 1, 1};
  body = std::move(f);
  threads.resize(n);
  meetings.clear();
  alive = n;
  for (Thread& t : threads) {
    if (t.stack.empty()) t.stack.resize(96 << 10);
    t.over = false;
    getcontext(&t.at);
    t.at.uc_stack.ss_sp = t.stack.data();
    t.at.uc_stack.ss_size = t.stack.size();
    t.at.uc_link = nullptr;
    makecontext(&t.at, enter, 0);
  }
  while (alive > 0) {
    const uint64_t before = moves;
    for (now = 0; now < n; ++now)
      if (!threads[now].over) { threadIdx = {now, 0, 0}; swapcontext(&scheduler, &threads[now].at); }
    if (moves == before) { std::printf("failed: block %d, %d threads wait for good\n", x, alive); std::exit(1); }
  }
}
inline void __syncthreads() { host::meet(0, 0, 0, 0); }
inline int __syncthreads_or(int v) { return host::meet(0, 0, 0, v).voted; }
inline void named_barrier(int which, int n) { host::meet(1 + which, 0, n, 0); }
inline void __syncwarp(uint32_t mask = 0xffffffffu) { host::warp(mask, 0); }
inline bool __any_sync(uint32_t mask, int v) { return host::warp(mask, v).vote_result != 0; }
inline uint32_t __ballot_sync(uint32_t mask, int v) { return host::warp(mask, v).vote_result; }
inline bool __all_sync(uint32_t mask, int v) { return host::warp(mask, !v).vote_result == 0; }
template <class T> inline T exchange(uint32_t mask, T v, int from) {
  static_assert(sizeof(T) <= 8, "");
  const int base = host::now & ~31;
  host::slots[host::now] = 0;
  std::memcpy(&host::slots[host::now], &v, sizeof(T));
  host::warp(mask, 0);
  T r;
  std::memcpy(&r, &host::slots[base + from], sizeof(T));
  host::warp(mask, 0);
  return r;
}
template <class T> inline T __shfl_up_sync(uint32_t mask, T v, int d) { const int l = threadIdx.x & 31; return exchange(mask, v, l >= d ? l - d : l); }
template <class T> inline T __shfl_xor_sync(uint32_t mask, T v, int d) { return exchange(mask, v, (threadIdx.x & 31) ^ d); }
template <class T> inline T __shfl_sync(uint32_t mask, T v, int from) { return exchange(mask, v, from); }
"""


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def cut(text, begin, end):
    """From `begin` up to, not with, the first `end` behind it."""
    at = text.index(begin)
    return text[at:text.index(end, at)]


def compiled(directory, text, **parts):
    """The program of `text`, with its @names@ filled in, behind the preamble; skips where there is no host compiler."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    for name, part in parts.items():
        text = text.replace(f"@{name}@", part)
    src, exe = str(directory / "kernel.cpp"), str(directory / "kernel")
    with open(src, "w") as f:
        f.write(PREAMBLE + text)
    # (whole numbers wrap around as on the device)
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-w", "-fwrapv", src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return exe


def output(exe, *args):
    r = subprocess.run([exe, *map(str, args)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (args, r.returncode, r.stdout[-2000:])
    return r.stdout
