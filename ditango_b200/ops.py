"""Tensor-level wrappers over the C ABI: torch tensors in, kernel launches on the current stream.

These are the only places arithmetic happens on the attention path; they raise when the
extension is missing or an argument is not a CUDA tensor of the expected kind.
"""
import ctypes
import functools
import math
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _capi
from ._capi import DTB_BF16, DTB_E4M3, DTB_F32, DTB_I8, LSE_BHS, LSE_BSH


class LaunchLog:
    """Optional accounting of kernel launches made through this module.  `count` always runs; with
    `events` enabled every flash launch is bracketed by two CUDA events on the launching stream so
    a benchmark can read per-launch device time and the FLOPs each launch executed.  (An event between two
    launches does not keep the second from overlapping the first; for a launch that overlaps its predecessor the
    pair then reads "end of the previous launch to end of this one", so the durations of a chain still add up to
    the chain's time.)"""
    count = 0
    events = None            # list of (start_event, end_event, flops) while enabled
    overlapped = 0           # flash launches made with overlap_previous

    @classmethod
    def reset(cls, with_events: bool = False):
        cls.count = 0
        cls.overlapped = 0
        cls.events = [] if with_events else None


# The raw handle of a device's current stream: building a Stream object around it costs several times the rest of a launch's
# Python.  The function is not part of torch's public interface; where a build lacks it, the Stream object is used.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr() -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise _capi.ExtensionError("ditango_b200 kernels take CUDA tensors only")


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch_stream(*tensors) -> int:
    """The current device's current stream, for a launch on `tensors` (None among them is skipped).  Those of another device are
    refused, not reached for."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        d = t.get_device()
        if d != dev:
            if d < 0:
                raise _capi.ExtensionError("ditango_b200 kernels take CUDA tensors only")
            if dev is not None or d != _current_device():
                raise _capi.ExtensionError(f"tensor on cuda:{d}, but the current device is cuda:{_current_device()}")
            dev = d
    return _stream_ptr() if _raw_stream is None else _raw_stream(dev)


def _empty(shape, dtype: torch.dtype, device) -> torch.Tensor:
    """torch.empty for a few axes, without the time that it takes to find its layout (1.6 us against 3.2)."""
    strides, n = [], 1
    for extent in reversed(shape):
        strides.append(n)
        n *= extent
    return torch.empty_strided(shape, strides[::-1], dtype=dtype, device=device)


def _empty_like(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous tensor of x's shape."""
    return torch.empty_like(x, dtype=dtype) if x.is_contiguous() else _empty(x.shape, dtype, x.device)


def _tok_stride(x: torch.Tensor) -> int:
    """Elements between consecutive tokens of a [..., H, D] tensor whose (H, D) block is dense and
    whose leading dims are laid out as one flat token axis."""
    if x.stride(-1) != 1 or x.stride(-2) != x.shape[-1]:
        raise _capi.ExtensionError("head and channel dims must be contiguous")
    ts = x.stride(-3)
    for d in range(x.dim() - 4, -1, -1):
        if x.shape[d] != 1 and x.stride(d) != x.stride(d + 1) * x.shape[d + 1]:
            raise _capi.ExtensionError("leading dims must flatten into one token axis")
    return ts


def read_status() -> int:
    """Synchronise the current stream and return (then clear) the device status word."""
    return _capi.load().dtb_read_status(_stream_ptr())


_STATUS_WATCH = {}      # device index -> [pinned int32 word, event behind the copy in flight or None, the event kept for it]


def poll_status():
    """Non-blocking look at the device status word, for the hot path.  Each call tests the copy of
    the word that the previous call queued (if it has landed) and queues the next copy behind the
    work already on the current stream; it raises ExtensionError when a kernel reported that a bounded
    wait ran out -- from that point on launches skip their work and results are not valid.  The
    report therefore comes at most one poll late.  `read_status()` clears the word."""
    lib = _capi.load()
    dev = torch.cuda.current_device()
    watch = _STATUS_WATCH.get(dev)
    if watch is None:
        watch = _STATUS_WATCH[dev] = [torch.zeros(1, dtype=torch.int32).pin_memory(), None, None]
    host, pending, _ = watch
    if pending is not None:
        if not pending.query():
            return                       # the earlier copy is still behind queued work
        watch[1] = None
        code = int(host[0])
        if code != 0:
            raise _capi.ExtensionError(
                f"a kernel gave up on a bounded wait (device status {code}); launches since then skipped "
                "their work -- results are not valid; read_status() clears the word")
    _capi.check(lib.dtb_peek_status_async(host.data_ptr(), _stream_ptr()), "dtb_peek_status_async")
    if watch[2] is None:
        watch[2] = torch.cuda.Event()
    watch[2].record()
    watch[1] = watch[2]


def post_status(code: int):
    """Set the device status word from the host (ordered on the current stream): kernels in flight give
    up their bounded waits and later launches skip their work until read_status() clears it."""
    _capi.check(_capi.load().dtb_post_status(int(code), _stream_ptr()), "dtb_post_status")


def flash_partial(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                  out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                  accumulate: bool = False, out_dtype: torch.dtype = torch.float32,
                  lse_layout: int = LSE_BHS, softmax_scale: Optional[float] = None,
                  cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
                  max_seqlen_q: Optional[int] = None, max_seqlen_k: Optional[int] = None,
                  overlap_previous: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention state of q against one KV chunk.

    Dense: q [B,Sq,H,D], k,v [B,Sk,H,D] bf16.  Packed (cu_seqlens given): q [Tq,H,D], k,v [Tk,H,D].
    Returns (out, lse); with accumulate=True the chunk's state is merged into the given fp32
    (out, lse) in place.  lse is [B,H,Sq] / [H,Tq] (LSE_BHS) or [B,Sq,H] / [Tq,H] (LSE_BSH).

    overlap_previous=True lets the launch start while the launch queued just before it on the current stream
    is finishing (DTB_LAUNCH_OVERLAP_PREVIOUS).  Only pass it when the last kernel or copy queued on the
    stream was another flash_partial call -- event waits and event records in between are fine, they neither
    write memory nor keep the launches from overlapping -- and when q, k, v, cu_seqlens were not written by
    that call; (out, lse) may be the state that call wrote.
    """
    lib = _capi.load()
    _need_cuda(q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k)
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise _capi.ExtensionError("q, k, v must be bfloat16")
    packed = cu_seqlens_q is not None
    H, D = q.shape[-2], q.shape[-1]
    if packed:
        if q.dim() != 3:
            raise _capi.ExtensionError("packed q must be [T,H,D]")
        Tq, Tk = q.shape[0], k.shape[0]
        nseg = cu_seqlens_q.numel() - 1
        sq = int(max_seqlen_q if max_seqlen_q is not None else Tq)
        sk = int(max_seqlen_k if max_seqlen_k is not None else Tk)
        if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_k.dtype != torch.int32:
            raise _capi.ExtensionError("cu_seqlens must be int32")
        lse_shape = (H, Tq) if lse_layout == LSE_BHS else (Tq, H)
    else:
        if q.dim() != 4:
            raise _capi.ExtensionError("dense q must be [B,S,H,D]")
        B, sq = q.shape[0], q.shape[1]
        sk = k.shape[1]
        nseg, Tq, Tk = B, B * sq, B * sk
        lse_shape = (B, H, sq) if lse_layout == LSE_BHS else (B, sq, H)
    if accumulate:
        if out is None or lse is None or out.dtype != torch.float32:
            raise _capi.ExtensionError("accumulate needs an existing fp32 (out, lse) state")
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
    if lse is None:
        lse = torch.empty(lse_shape, dtype=torch.float32, device=q.device)
    if tuple(lse.shape) != tuple(lse_shape) or not lse.is_contiguous() or lse.dtype != torch.float32:
        raise _capi.ExtensionError(f"lse must be a contiguous fp32 tensor of shape {lse_shape}")
    if out.shape != q.shape:
        raise _capi.ExtensionError("out must have q's shape")
    odt = DTB_F32 if out.dtype == torch.float32 else DTB_BF16
    if out.dtype not in (torch.float32, torch.bfloat16):
        raise _capi.ExtensionError("out must be float32 or bfloat16")
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    # dense: every query row meets every key row of its sequence; packed: upper bound by maxima
    flops = 4.0 * nseg * H * sq * sk * D
    ev = None
    if LaunchLog.events is not None:
        ev = (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
        ev[0].record()
    rc = lib.dtb_flash_fwd_ex(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _tok_stride(q), _tok_stride(k), _tok_stride(v),
        out.data_ptr(), odt, _tok_stride(out), lse.data_ptr(), lse_layout, int(accumulate),
        cu_seqlens_q.data_ptr() if packed else None, cu_seqlens_k.data_ptr() if packed else None,
        nseg, sq, sk, Tq, Tk, H, D, scale, _capi.LAUNCH_OVERLAP_PREVIOUS if overlap_previous else 0, _stream_ptr())
    _capi.check(rc, "dtb_flash_fwd_ex")
    LaunchLog.count += 1
    LaunchLog.overlapped += int(bool(overlap_previous))
    if ev is not None:
        ev[1].record()
        LaunchLog.events.append((ev[0], ev[1], flops))
    return out, lse


def _strides(x: torch.Tensor, shape) -> Tuple[int, int]:
    """(token, batch) strides in elements of a tensor [B,S,H,D], or packed [T,H,D], whose (H, D) block is dense; that of an axis of
    length 1, which nothing steps along, is given as a dense tensor's."""
    H, D = shape[-2], shape[-1]
    *outer, head, channel = x.stride()
    if channel != 1 or (head != D and H != 1):
        raise _capi.ExtensionError("head and channel dims must be contiguous")
    tok = outer[-1] if shape[-3] > 1 else H * D
    if len(shape) == 3:
        return tok, 0
    return tok, (outer[0] if shape[0] > 1 else tok * shape[1])


_FAR = 1 << 30           # (ctypes would cut off what an int does not hold)


def flash_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, left: int = -1, right: int = -1, sinks: int = 0,
                 q_start: Optional[int] = None, k_start: int = 0, seqlens_k: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, accumulate: bool = False,
                 out_dtype: torch.dtype = torch.float32, lse_layout: int = LSE_BHS, softmax_scale: Optional[float] = None,
                 cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
                 max_seqlen_q: Optional[int] = None, max_seqlen_k: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention state of q against one KV chunk with a sliding window and `sinks` first tokens that stay visible.

    The query at position x sees the key at position j when j <= x + right and (j >= x - left or j < sinks); -1 means no limit.
    Key j of a sequence is at position k_start + j.  Query i is at q_start + i; q_start=None puts the queries at the end of
    their sequence's keys (position i when there are as many queries as keys, the newest positions when the keys are a cache).

    Dense: q [B,Sq,H,D], k,v [B,Sk,Hk,D] bf16, any batch and token strides that are multiples of 8 and not below a token's heads
    (an expanded batch is refused); Hk divides H.  `seqlens_k`
    (int32 [B] on the device) gives the number of keys of each sequence, the rest of Sk may hold anything.  Packed
    (cu_seqlens given): q [Tq,H,D], k,v [Tk,Hk,D].  Returns (out, lse) as flash_partial does, mergeable with its states; with
    accumulate=True the state is merged into the given fp32 (out, lse) in place.  A row that sees no key has out 0 and lse -inf.
    Scores, sums and states are fp32; a weight is rounded to bf16 (2^-8 of itself at most) for the product with v, as in flash_partial.
    Keys and values that no query near by (in its 256) sees may hold anything, the others must be finite.  Few queries against many
    keys of a dense batch take two launches and scratch from the allocator of the current stream.
    """
    stream = _launch_stream(q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k, seqlens_k)
    at = 0 if q_start is None else q_start
    if not (-1 <= left <= _FAR and -1 <= right <= _FAR and 0 <= sinks <= _FAR and -_FAR <= k_start <= _FAR and -_FAR <= at <= _FAR):
        raise _capi.ExtensionError("left, right, sinks and positions are within 2^30")
    if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        raise _capi.ExtensionError("q, k, v must be bfloat16")
    packed = cu_seqlens_q is not None
    if packed != (cu_seqlens_k is not None):
        raise _capi.ExtensionError("cu_seqlens_q and cu_seqlens_k go together")
    shape, kshape = q.shape, k.shape
    if len(shape) != (3 if packed else 4) or len(kshape) != len(shape) or v.shape != kshape or kshape[-1] != shape[-1]:
        raise _capi.ExtensionError("q is [B,S,H,D] and k, v are [B,S,Hk,D], packed [T,H,D] and [T,Hk,D]")
    if packed:
        Tq, H, D = shape
        Tk, Hk, _ = kshape
        nseg = cu_seqlens_q.numel() - 1
        sq = min(Tq, int(max_seqlen_q)) if max_seqlen_q is not None else Tq
        sk = min(Tk, int(max_seqlen_k)) if max_seqlen_k is not None else Tk
        if any(c.dtype != torch.int32 or not c.is_contiguous() for c in (cu_seqlens_q, cu_seqlens_k)) or cu_seqlens_k.numel() != nseg + 1:
            raise _capi.ExtensionError("cu_seqlens must be contiguous int32, as many of q as of k")
        lse_shape = (H, Tq) if lse_layout == LSE_BHS else (Tq, H)
    else:
        nseg, sq, H, D = shape
        batch, sk, Hk, _ = kshape
        if batch != nseg:
            raise _capi.ExtensionError("q and k must have one batch size")
        Tq, Tk = nseg * sq, nseg * sk
        lse_shape = (nseg, H, sq) if lse_layout == LSE_BHS else (nseg, sq, H)
    if seqlens_k is not None and (packed or seqlens_k.dtype != torch.int32 or seqlens_k.numel() != nseg or not seqlens_k.is_contiguous()):
        raise _capi.ExtensionError("seqlens_k is contiguous int32 with one length per sequence of a dense batch")
    if accumulate and (out is None or lse is None or out.dtype != torch.float32):
        raise _capi.ExtensionError("accumulate needs an existing fp32 (out, lse) state")
    if out is None:
        if out_dtype not in _VALUES:
            raise _capi.ExtensionError("out must be float32 or bfloat16")
        out = _empty_like(q, out_dtype)
    elif out.shape != shape or not out.is_contiguous() or out.dtype not in _VALUES:
        raise _capi.ExtensionError("out must be contiguous float32 or bfloat16 of q's shape")
    if lse is None:
        lse = _empty(lse_shape, torch.float32, q.device)
    elif tuple(lse.shape) != lse_shape or not lse.is_contiguous() or lse.dtype != torch.float32:
        raise _capi.ExtensionError(f"lse must be a contiguous fp32 tensor of shape {lse_shape}")
    if q.numel() == 0:
        return out, lse
    # (an empty tensor has no address, and nothing is read)
    keys, values = k.data_ptr() or q.data_ptr(), v.data_ptr() or q.data_ptr()
    lib = _capi.load()
    scratch, scratch_bytes = None, 0
    if not packed and sq > 16:         # (fewer queries never have their keys split)
        scratch_bytes = lib.dtb_flash_window_scratch_bytes(nseg, sq, sk, H, Hk, D, left, right, sinks)
        if scratch_bytes < 0:
            _capi.check(scratch_bytes, "dtb_flash_window_scratch_bytes")
        if scratch_bytes:
            scratch = _empty((scratch_bytes,), torch.uint8, q.device)
    ev = None
    if LaunchLog.events is not None:
        ev = (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
        ev[0].record()
    rc = lib.dtb_flash_window(
        q.data_ptr(), keys, values, *_strides(q, shape), *_strides(k, kshape), *_strides(v, kshape),
        out.data_ptr(), _VALUES[out.dtype], lse.data_ptr(), lse_layout, accumulate,
        cu_seqlens_q.data_ptr() if packed else None, cu_seqlens_k.data_ptr() if packed else None,
        None if seqlens_k is None else seqlens_k.data_ptr(), nseg, sq, sk, Tq, Tk, H, Hk, D,
        D ** -0.5 if softmax_scale is None else softmax_scale, left, right, sinks,
        _capi.QUERIES_LAST if q_start is None else q_start, k_start, None if scratch is None else scratch.data_ptr(), scratch_bytes, stream)
    if rc:
        _capi.check(rc, "dtb_flash_window")
    LaunchLog.count += 1 if scratch is None else 2
    if ev is not None:
        ev[1].record()
        span = sk if left < 0 or right < 0 else min(sk, left + right + 1 + sinks)      # upper bound of a row's keys
        LaunchLog.events.append((ev[0], ev[1], 4.0 * nseg * H * sq * span * D))
    return out, lse


class PagePlan(NamedTuple):
    """What extend_pages found: `slots` [tokens] of the new tokens, `cu_seqlens` [streams + 1] among them, `seqlens` and `free_count` as they are
    now, and `missing` [1], 0 unless nothing was taken.  All int32 on the device."""
    slots: torch.Tensor
    cu_seqlens: torch.Tensor
    seqlens: torch.Tensor
    free_count: torch.Tensor
    missing: torch.Tensor


class PageRelease(NamedTuple):
    """The table, the streams' lengths and the number of free pages after release_pages."""
    table: torch.Tensor
    seqlens: torch.Tensor
    free_count: torch.Tensor


def _page_args(table, free, free_count, page_size, a, b, c):
    """Checks what the tables' two directions are given, a, b and c (or None) with a number per stream; returns (streams, columns, pages)."""
    i32 = torch.int32
    if not (table.dtype is i32 and free.dtype is i32 and free_count.dtype is i32 and a.dtype is i32 and b.dtype is i32 and (c is None or c.dtype is i32) and
            table.is_contiguous() and free.is_contiguous() and a.is_contiguous() and b.is_contiguous() and (c is None or c.is_contiguous())):
        raise _capi.ExtensionError("tables, lengths and pages are contiguous int32 tensors")
    shape = table.shape
    if len(shape) != 2 or free.dim() != 1 or free_count.numel() != 1 or not (a.numel() == b.numel() == shape[0] and (c is None or c.numel() == shape[0])):
        raise _capi.ExtensionError("a table is [streams, columns], with a number per stream; free pages are a list and their count")
    if shape[0] == 0:
        raise _capi.ExtensionError("a table without streams")
    if not 0 < page_size < 1 << 31:
        raise _capi.ExtensionError("a page size is a power of two from 16 to 2^20")
    return shape[0], shape[1], free.numel()


def extend_pages(table: torch.Tensor, seqlens: torch.Tensor, new_lens: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, page_size: int,
                 tokens: int) -> PagePlan:
    """Room in pages for new_lens [streams] tokens more behind the seqlens [streams] that each stream has.

    table [streams, columns] holds the streams' pages; entries for new ones are written in place.  The first free_count [1] of `free` are the
    numbers of pages that nobody holds, the last of those is taken first, and `free` has one entry per page of the pool.  `tokens`, known to
    the host, is the number of rows that the new keys and values come in: new_lens add up to it or less, and slots behind the last token
    are -1 (as is that of a token on a page that release_pages took from inside its stream).  All or nothing: with too few free pages `missing`
    says how many, with streams that outgrow their row or `tokens` it is -1, and then the table and the numbers stay as they are.  The results
    are new tensors, for the next step; one launch, no host round trip.  Up to 16384 streams."""
    streams, columns, pages = _page_args(table, free, free_count, page_size, seqlens, new_lens, None)
    if not 0 <= tokens < (1 << 31) - 4:
        raise _capi.ExtensionError("tokens is a number of rows")
    stream = _launch_stream(table, seqlens, new_lens, free, free_count)
    # (one allocation; slots begin it and so are 16-byte aligned)
    results = _empty((tokens + 2 * streams + 3,), torch.int32, table.device)
    slots = results.data_ptr()
    cu = slots + 4 * tokens
    lens = cu + 4 * streams + 4
    count = lens + 4 * streams
    rc = _capi.load().dtb_extend_pages(
        table.data_ptr(), seqlens.data_ptr(), new_lens.data_ptr(), free.data_ptr(), free_count.data_ptr(), streams, columns, pages, page_size,
        slots, tokens, cu, lens, count, count + 4, stream)
    if rc:
        _capi.check(rc, "dtb_extend_pages")
    LaunchLog.count += 1
    # (results are whole numbers: nothing is lost by parts that autograd does not know as views, and they are made in half the time)
    return PagePlan(*torch.unsafe_split_with_sizes(results, (tokens, streams + 1, streams, 1, 1)))


def release_pages(table: torch.Tensor, seqlens: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, begin: torch.Tensor, end: torch.Tensor,
                  page_size: int, *, out_table: Optional[torch.Tensor] = None) -> PageRelease:
    """Gives back the pages of each stream whose tokens all lie in [begin, end) [streams]: what a window has left behind (begin: the first tokens
    that stay), a stream that is over (0 and its length or more), or its newest tokens, where end is its length or more; it is then
    begin tokens long.  Their entries become -1, in place unless `out_table` takes the table as it is then; `free` gets them behind the others.  The
    numbers are new tensors; one launch."""
    streams, columns, pages = _page_args(table, free, free_count, page_size, seqlens, begin, end)
    if out_table is None:
        out_table = table
    elif out_table.dtype is not torch.int32 or out_table.shape != table.shape or not out_table.is_contiguous():
        raise _capi.ExtensionError("out_table is a contiguous int32 tensor of the table's shape")
    stream = _launch_stream(table, out_table, seqlens, free, free_count, begin, end)
    results = _empty((streams + 1,), torch.int32, table.device)
    lens = results.data_ptr()
    rc = _capi.load().dtb_release_pages(
        table.data_ptr(), out_table.data_ptr(), seqlens.data_ptr(), begin.data_ptr(), end.data_ptr(), free.data_ptr(), free_count.data_ptr(),
        streams, columns, pages, page_size, lens, lens + 4 * streams, stream)
    if rc:
        _capi.check(rc, "dtb_release_pages")
    LaunchLog.count += 1
    return PageRelease(out_table, *torch.unsafe_split_with_sizes(results, (streams, 1)))


def _pools(k: torch.Tensor, v: torch.Tensor):
    """Shape [pages, P, heads, D] of k_pages and v_pages, and the (page, token, head) strides of each; that of an axis of length 1, which nothing steps
    along, is given as if it lay behind the others."""
    shape, k_strides, v_strides = k.shape, k.stride(), v.stride()
    if not (k.dtype is v.dtype is torch.bfloat16 and len(shape) == 4 and v.shape == shape and k_strides[3] == v_strides[3] == 1):
        raise _capi.ExtensionError("pages are bfloat16 [pages, tokens, heads, D] with contiguous channels, of keys as of values")
    if shape[0] > 1 and shape[2] > 1:
        return shape, k_strides[:3], v_strides[:3]
    pages, P, heads, D = shape
    both = []
    for page, tok, head, _ in (k_strides, v_strides):
        if heads == 1:
            head = max(tok * P, D)
        if pages == 1:
            page = max(tok * P, head * heads)
        both.append((page, tok, head))
    return shape, *both


def write_pages(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor):
    """Keys and values k, v [..,Hk,D] bf16 of new tokens, any token stride, into the slots [tokens] (extend_pages) of k_pages and v_pages
    [pages, P, Hk, D], any strides.  A token whose slot is -1, or none of the pool's, is left out; slots are to differ from one another.
    One launch."""
    stream = _launch_stream(k, v, k_pages, v_pages, slots)
    shape, k_strides, v_strides = _pools(k_pages, v_pages)
    pages, P, Hk, D = shape
    kshape = k.shape
    if not (k.dtype is v.dtype is torch.bfloat16 and len(kshape) >= 3 and v.shape == kshape and kshape[-1] == D and kshape[-2] == Hk):
        raise _capi.ExtensionError("k and v are bfloat16 [..,Hk,D] with the pages' heads")
    if Hk * D == 0:
        return
    tokens = k.numel() // (Hk * D)
    if slots.dtype is not torch.int32 or slots.numel() != tokens or not slots.is_contiguous():
        raise _capi.ExtensionError("slots are contiguous int32, one per token")
    if tokens == 0:
        return
    rc = _capi.load().dtb_write_pages(
        k.data_ptr(), v.data_ptr(), _flat_tok_stride(k), _flat_tok_stride(v), tokens, slots.data_ptr(), k_pages.data_ptr(), *k_strides,
        v_pages.data_ptr(), *v_strides, pages, P, Hk, D, stream)
    if rc:
        _capi.check(rc, "dtb_write_pages")
    LaunchLog.count += 1


def _flat_tok_stride(x: torch.Tensor) -> int:
    """_tok_stride where the axes of one token, one head do not count."""
    if x.is_contiguous():
        return x.shape[-1] * x.shape[-2]
    if x.shape[-2] == 1 and x.stride(-1) == 1:
        x = x.as_strided(x.shape, (*x.stride()[:-2], x.shape[-1], 1))
    if x.numel() == x.shape[-1] * x.shape[-2]:
        x = x.as_strided(x.shape, (*(x.shape[-1] * x.shape[-2],) * (x.dim() - 2), *x.stride()[-2:]))
    return _tok_stride(x)


_PAGED_PLANS = {}         # (device, sequences, lengths, heads, D, packed) -> (bytes that flash_paged needs, its launches)


def flash_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, seqlens_k: torch.Tensor, *, left: int = -1,
                right: int = -1, sinks: int = 0, cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: Optional[int] = None,
                max_seqlen_k: Optional[int] = None, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                accumulate: bool = False, out_dtype: torch.dtype = torch.float32, lse_layout: int = LSE_BHS,
                softmax_scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention state of the newest tokens of sequences over their keys and values in pages: flash_window with a table.

    k_pages, v_pages [pages, P, Hk, D] bf16, any strides that are multiples of 8; table int32 [B, columns], entry j of a row is the page of the
    sequence's tokens [j P, (j + 1) P); seqlens_k int32 [B] keys of each, those of the queries included (write_pages goes before this).  The last
    query is at the last key's position; the query at position x sees key j when j <= x + right and (j >= x - left or j < sinks); -1
    means no limit (right=0: causal; -1: all tokens of a chunk see one another).

    Dense: q [B,Sq,H,D] bf16.  Packed: q [T,H,D] with cu_seqlens_q int32 [B + 1] on the device, up to max_seqlen_q (known to the host, T if not
    given) queries each; rows behind the last sequence, and behind the first max_seqlen_q of one, are left as they are.  Hk divides H.  max_seqlen_k is about the longest sequence's
    length, if the host knows it (the room in a row of the table if not): kernels and numbers of CTAs are chosen by it, and results depend on it by
    roundings alone.

    Returns (out, lse) as flash_window does, mergeable with its states and flash_partial's; with accumulate=True the state is merged into the given
    fp32 (out, lse) in place.  A row that sees no key has out 0 and lse -inf.  Entries of the table behind a sequence's last page or for pages that no
    query sees may be anything; where one that a query sees is not a page of the pool, its keys and values are 0.  Keys and values that
    no query near by (in its 256) sees may hold anything, the others must be finite.  Scratch comes from the allocator of the current stream."""
    stream = _launch_stream(q, k_pages, v_pages, table, seqlens_k, cu_seqlens_q, out, lse)
    if not (-1 <= left <= _FAR and -1 <= right <= _FAR and 0 <= sinks <= _FAR):
        raise _capi.ExtensionError("left, right and sinks are within 2^30")
    shape = q.shape
    (pages, P, Hk, D), k_strides, v_strides = _pools(k_pages, v_pages)
    packed = cu_seqlens_q is not None
    if q.dtype is not torch.bfloat16 or len(shape) != (3 if packed else 4) or shape[-1] != D:
        raise _capi.ExtensionError("q is bfloat16 [B,S,H,D], packed [T,H,D], with the pages' channels")
    tshape = table.shape
    if table.dtype is not torch.int32 or len(tshape) != 2 or not table.is_contiguous():
        raise _capi.ExtensionError("table is contiguous int32 [sequences, columns]")
    nseg, columns = tshape
    if seqlens_k.dtype is not torch.int32 or seqlens_k.numel() != nseg or not seqlens_k.is_contiguous():
        raise _capi.ExtensionError("seqlens_k is contiguous int32 with one length per sequence")
    if packed:
        T, H, _ = shape
        sq = min(T, int(max_seqlen_q)) if max_seqlen_q is not None else T
        if cu_seqlens_q.dtype is not torch.int32 or not cu_seqlens_q.is_contiguous() or cu_seqlens_q.numel() != nseg + 1:
            raise _capi.ExtensionError("cu_seqlens_q must be contiguous int32, one more than sequences")
        lse_shape = (H, T) if lse_layout == LSE_BHS else (T, H)
    else:
        batch, sq, H, _ = shape
        if batch != nseg:
            raise _capi.ExtensionError("q and the table must have one batch size")
        T = nseg * sq
        lse_shape = (nseg, H, sq) if lse_layout == LSE_BHS else (nseg, sq, H)
    sk = min(columns * P, _FAR - 1)
    if max_seqlen_k is not None:
        sk = max(0, min(sk, int(max_seqlen_k)))
    if left >= 0:
        sk = min(sk, left + sq + sinks)          # (the keys that a sequence's queries see together)
    if accumulate and (out is None or lse is None or out.dtype != torch.float32):
        raise _capi.ExtensionError("accumulate needs an existing fp32 (out, lse) state")
    if out is None:
        if out_dtype not in _VALUES:
            raise _capi.ExtensionError("out must be float32 or bfloat16")
        out = _empty_like(q, out_dtype)
    elif out.shape != shape or not out.is_contiguous() or out.dtype not in _VALUES:
        raise _capi.ExtensionError("out must be contiguous float32 or bfloat16 of q's shape")
    if lse is None:
        lse = _empty(lse_shape, torch.float32, q.device)
    elif tuple(lse.shape) != lse_shape or not lse.is_contiguous() or lse.dtype != torch.float32:
        raise _capi.ExtensionError(f"lse must be a contiguous fp32 tensor of shape {lse_shape}")
    if T * H * D == 0 or sq <= 0:
        return out, lse
    lib = _capi.load()
    key = (q.get_device(), nseg, sq, sk, T, H, Hk, D, packed)
    plan = _PAGED_PLANS.get(key)
    if plan is None:
        plan = lib.dtb_flash_paged_scratch_bytes(nseg, sq, sk, T, H, Hk, D), lib.dtb_flash_paged_launches(nseg, sq, sk, T, packed, H, Hk, D)
        if min(plan) < 0:
            _capi.check(min(plan), "dtb_flash_paged")
        if len(_PAGED_PLANS) >= 4096:
            _PAGED_PLANS.clear()
        _PAGED_PLANS[key] = plan
    need, launches = plan
    scratch = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=q.device) if need else None
    q_strides = (H * D, 0 if packed else sq * H * D) if q.is_contiguous() else _strides(q, shape)
    ev = None
    if LaunchLog.events is not None:
        ev = (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
        ev[0].record()
    rc = lib.dtb_flash_paged(
        q.data_ptr(), *q_strides, k_pages.data_ptr(), *k_strides, v_pages.data_ptr(), *v_strides, pages, P, table.data_ptr(), columns,
        seqlens_k.data_ptr(), cu_seqlens_q.data_ptr() if packed else None, out.data_ptr(), _VALUES[out.dtype], lse.data_ptr(), lse_layout, accumulate,
        nseg, sq, sk, T, H, Hk, D, D ** -0.5 if softmax_scale is None else softmax_scale, left, right, sinks, None if scratch is None else scratch.data_ptr(), need, stream)
    if rc:
        _capi.check(rc, "dtb_flash_paged")
    LaunchLog.count += launches
    if ev is not None:
        ev[1].record()
        span = sk if left < 0 or right < 0 else min(sk, left + right + 1 + sinks)      # upper bound of a row's keys
        LaunchLog.events.append((ev[0], ev[1], 4.0 * T * H * span * D))
    return out, lse


class QuantizedRows(NamedTuple):
    """Values of a state in 8 bits: codes [..,H,D] (int8 or float8_e4m3fn) and one exponent byte b per row [..,H]; a value is
    code * 2^(b - 127).  b = 255 marks a row with an infinity or a NaN, which reads back as NaN."""
    values: torch.Tensor
    exponents: torch.Tensor

    @property
    def shape(self):
        return self.values.shape

    @property
    def dtype(self):
        return self.values.dtype

    @property
    def device(self):
        return self.values.device

    @property
    def nbytes(self) -> int:
        return self.values.nbytes + self.exponents.nbytes


_CODES = {torch.int8: DTB_I8, torch.float8_e4m3fn: DTB_E4M3}
_VALUES = {torch.float32: DTB_F32, torch.bfloat16: DTB_BF16}


def _new_rows(device, shape, dtype: torch.dtype) -> QuantizedRows:
    if dtype not in _CODES:
        raise _capi.ExtensionError(f"rows are kept in int8 or float8_e4m3fn, not {dtype}")
    return QuantizedRows(_empty(shape, dtype, device), _empty(shape[:-1], torch.uint8, device))


def _check_rows(rows: QuantizedRows, shape):
    values, exponents = rows
    if (values.dtype not in _CODES or exponents.dtype != torch.uint8 or values.shape != shape or exponents.shape != shape[:-1] or
            not values.is_contiguous() or not exponents.is_contiguous()):
        raise _capi.ExtensionError("rows are contiguous int8 or float8_e4m3fn codes with one contiguous uint8 exponent per row")


def _check_result(out, dtype, shape):
    if out.dtype != dtype or out.shape != shape or not out.is_contiguous():
        raise _capi.ExtensionError(f"a result must be a contiguous {dtype} tensor of the states' shape")


def quantize_rows(out: torch.Tensor, dtype: torch.dtype = torch.int8, *, rows: Optional[QuantizedRows] = None) -> QuantizedRows:
    """The values [..,H,D] of a state (fp32 or bf16, contiguous) in 8 bits, each row by its own power of two; into `rows` where
    given.  One launch."""
    shape = out.shape
    if out.dtype not in _VALUES or not out.is_contiguous():
        raise _capi.ExtensionError("a state's values are contiguous float32 or bfloat16")
    if rows is None:
        stream = _launch_stream(out)
        rows = _new_rows(out.device, shape, dtype)
    else:
        stream = _launch_stream(out, *rows)
        _check_rows(rows, shape)
    n = out.numel()
    if n:                      # (an empty tensor has no address)
        rc = _capi.load().dtb_quantize_rows(out.data_ptr(), _VALUES[out.dtype], rows.values.data_ptr(), _CODES[rows.values.dtype],
                                            rows.exponents.data_ptr(), n // shape[-1], shape[-1], stream)
        if rc:
            _capi.check(rc, "dtb_quantize_rows")
        LaunchLog.count += 1
    return rows


def dequantize_rows(rows: QuantizedRows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `rows` stand for, as fp32 or bf16 (exact in both).  One launch."""
    if dtype not in _VALUES:
        raise _capi.ExtensionError("rows are read back as float32 or bfloat16")
    values, exponents = rows
    shape = values.shape
    stream = _launch_stream(values, exponents)
    _check_rows(rows, shape)
    out = torch.empty_like(values, dtype=dtype)
    n = values.numel()
    if n:
        rc = _capi.load().dtb_dequantize_rows(values.data_ptr(), _CODES[values.dtype], exponents.data_ptr(), out.data_ptr(), _VALUES[dtype],
                                              n // shape[-1], shape[-1], stream)
        if rc:
            _capi.check(rc, "dtb_dequantize_rows")
        LaunchLog.count += 1
    return out


# for n states: types of one array that holds their values', exponents' and lse's addresses, one of their types and layouts
_ARRAYS = {n: (ctypes.c_void_p * (3 * n), ctypes.c_int * (2 * n)) for n in range(1, _capi.MERGE_MAX_STATES + 1)}


def _merge_rows(states, shape, out, lse_out, lse_out_layout, out_bf16, out_rows):
    """Launch of dtb_merge_rows; states[i] = (values tensor or QuantizedRows, lse, layout)."""
    n = len(states)
    if len(shape) not in (3, 4) or n not in _ARRAYS:
        raise _capi.ExtensionError(f"1 to {_capi.MERGE_MAX_STATES} states of [B,S,H,D] or [T,H,D]")
    B, S, H, D = (1, *shape) if len(shape) == 3 else shape
    rows, row_shape = B * S * H, shape[:-1]
    tensors, (pointers, ints) = [out, out_bf16, lse_out], _ARRAYS[n]
    addresses, kinds = pointers(), ints()
    for i, (o, l, lay) in enumerate(states):
        if type(o) is QuantizedRows:
            v, e = o
            if e.dtype != torch.uint8 or e.shape != row_shape or not e.is_contiguous():
                raise _capi.ExtensionError("exponents are contiguous uint8, one per row")
            tensors += (v, e, l)
            addresses[n + i] = e.data_ptr()
            dtype = _CODES.get(v.dtype)
        else:
            v = o
            tensors += (v, l)
            dtype = _VALUES.get(v.dtype)
        if dtype is None or v.shape != shape or not v.is_contiguous():
            raise _capi.ExtensionError("states must be contiguous, of one shape, and fp32, bf16 or QuantizedRows")
        if l.dtype != torch.float32 or l.numel() != rows or not l.is_contiguous():
            raise _capi.ExtensionError("lse must be contiguous fp32 with B*S*H entries")
        addresses[i] = v.data_ptr()
        addresses[2 * n + i] = l.data_ptr()
        kinds[i] = dtype
        kinds[n + i] = lay
    if out is not None:
        _check_result(out, torch.float32, shape)
    if out_bf16 is not None:
        _check_result(out_bf16, torch.bfloat16, shape)
    if lse_out is not None and (lse_out.dtype != torch.float32 or lse_out.numel() != rows or not lse_out.is_contiguous()):
        raise _capi.ExtensionError("lse_out must be contiguous fp32 with B*S*H entries")
    codes, code, exponents = None, 0, None
    if out_rows is not None:
        _check_rows(out_rows, shape)
        codes, exponents = out_rows
        tensors += out_rows
        code = _CODES[codes.dtype]
    stream = _launch_stream(*tensors)
    if rows * D == 0:
        return
    at, kinds_at = ctypes.addressof(addresses), ctypes.addressof(kinds)
    rc = _capi.load().dtb_merge_rows(
        n, at, kinds_at, at + 8 * n, at + 16 * n, kinds_at + 4 * n, None if out is None else out.data_ptr(),
        None if lse_out is None else lse_out.data_ptr(), lse_out_layout, None if out_bf16 is None else out_bf16.data_ptr(),
        None if codes is None else codes.data_ptr(), code, None if exponents is None else exponents.data_ptr(), B, S, H, D, stream)
    if rc:
        _capi.check(rc, "dtb_merge_rows")
    LaunchLog.count += 1


def merge_states(states: Sequence[Tuple[Union[torch.Tensor, QuantizedRows], torch.Tensor, int]], *,
                 out: Optional[torch.Tensor] = None, lse_out: Optional[torch.Tensor] = None,
                 lse_out_layout: int = LSE_BSH, out_bf16: Optional[torch.Tensor] = None,
                 want_lse: bool = True, fp32_out: bool = True,
                 out_rows: Union[QuantizedRows, torch.dtype, None] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """One-pass merge of partial states.  states[i] = (out_i [B,S,H,D] fp32|bf16 contiguous or QuantizedRows,
    lse_i fp32 contiguous, layout_i).  Returns (out fp32 [B,S,H,D], lse_out or None).  With
    fp32_out=False only the bf16 copy `out_bf16` is written and returned in place of `out`.  `out_rows`
    (QuantizedRows to fill) has the result written in 8 bits too; with fp32_out=False and no `out_bf16`
    that is what is returned, and a type (torch.int8, torch.float8_e4m3fn) asks for new ones."""
    if out_rows is not None or QuantizedRows in [type(o) for o, _, _ in states]:
        shape, device = states[0][0].shape, states[0][1].device
        if isinstance(out_rows, torch.dtype):
            if fp32_out or out_bf16 is not None:
                raise _capi.ExtensionError("out_rows is a type only where its rows are what is returned: fp32_out=False and no out_bf16")
            out_rows = _new_rows(device, shape, out_rows)
        if not fp32_out:
            out = None
            if out_bf16 is None and out_rows is None:
                raise _capi.ExtensionError("fp32_out=False needs out_bf16 or out_rows")
        elif out is None:
            out = _empty(shape, torch.float32, device)
        if not want_lse:
            lse_out = None
        elif lse_out is None:
            lead, s, h = tuple(shape[:-3]), shape[-3], shape[-2]
            lse_out = _empty(lead + ((s, h) if lse_out_layout == LSE_BSH else (h, s)), torch.float32, device)
        _merge_rows(states, shape, out, lse_out, lse_out_layout, out_bf16, out_rows)
        return (out if out is not None else out_bf16 if out_bf16 is not None else out_rows), lse_out
    lib = _capi.load()
    n = len(states)
    o0 = states[0][0]
    if o0.dim() == 3:
        B, (S, H, D) = 1, o0.shape
    else:
        B, S, H, D = o0.shape
    outs = (ctypes.c_void_p * n)()
    lses = (ctypes.c_void_p * n)()
    dts = (ctypes.c_int * n)()
    lays = (ctypes.c_int * n)()
    for i, (o, l, lay) in enumerate(states):
        _need_cuda(o, l)
        if not o.is_contiguous() or not l.is_contiguous() or o.shape != o0.shape:
            raise _capi.ExtensionError("states must be contiguous and of one shape")
        if l.dtype != torch.float32 or l.numel() != B * S * H:
            raise _capi.ExtensionError("lse must be fp32 with B*S*H entries")
        outs[i], lses[i] = o.data_ptr(), l.data_ptr()
        dts[i] = DTB_F32 if o.dtype == torch.float32 else DTB_BF16
        lays[i] = lay
    if not fp32_out:
        if out_bf16 is None:
            raise _capi.ExtensionError("fp32_out=False needs out_bf16")
        out = None
    elif out is None:
        out = torch.empty(o0.shape, dtype=torch.float32, device=o0.device)
    if out_bf16 is not None and (out_bf16.dtype != torch.bfloat16 or out_bf16.shape != o0.shape
                                 or not out_bf16.is_contiguous()):
        raise _capi.ExtensionError("out_bf16 must be a contiguous bfloat16 tensor of the states' shape")
    if not want_lse:
        lse_out = None
    if want_lse and lse_out is None:
        shape = ((B, S, H) if lse_out_layout == LSE_BSH else (B, H, S)) if o0.dim() == 4 else \
                ((S, H) if lse_out_layout == LSE_BSH else (H, S))
        lse_out = torch.empty(shape, dtype=torch.float32, device=o0.device)
    rc = lib.dtb_merge_states(
        n, outs, dts, lses, lays, out.data_ptr() if out is not None else None,
        lse_out.data_ptr() if lse_out is not None else None,
        lse_out_layout, out_bf16.data_ptr() if out_bf16 is not None else None, B, S, H, D, _stream_ptr())
    _capi.check(rc, "dtb_merge_states")
    LaunchLog.count += 1
    return (out if out is not None else out_bf16), lse_out


def copy_chunks(pairs: Sequence[Tuple[torch.Tensor, torch.Tensor]], chunk_bytes: int,
                extents: Tuple[int, int, int], src_strides: Tuple[int, int, int],
                dst_strides: Tuple[int, int, int]):
    """Strided chunk copy src -> dst for up to four tensor pairs in one launch (byte strides)."""
    lib = _capi.load()
    n = len(pairs)
    srcs = (ctypes.c_void_p * n)()
    dsts = (ctypes.c_void_p * n)()
    for i, (s, d) in enumerate(pairs):
        _need_cuda(s, d)
        srcs[i], dsts[i] = s.data_ptr(), d.data_ptr()
    rc = lib.dtb_copy_chunks(n, srcs, dsts, chunk_bytes, *extents, *src_strides, *dst_strides, _stream_ptr())
    _capi.check(rc, "dtb_copy_chunks")
    LaunchLog.count += 1


def norm_rope(q: torch.Tensor, k: torch.Tensor, q_norm: Tuple[torch.Tensor, torch.Tensor, float],
              k_norm: Tuple[torch.Tensor, torch.Tensor, float], cos: torch.Tensor, sin: torch.Tensor,
              text_len: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Layer norm over D of q, k [B,S,H,D] bf16 (norms as (weight, bias, eps)), then rotary embedding (interleaved
    pairs, cos / sin fp32 [S - text_len, D]) of the tokens behind the first text_len; new tensors, one launch."""
    lib = _capi.load()
    _need_cuda(q, k, q_norm[0], q_norm[1], k_norm[0], k_norm[1], cos, sin)
    B, S, H, D = q.shape
    for x in (q, k, q_norm[0], q_norm[1], k_norm[0], k_norm[1]):
        if x.dtype != torch.bfloat16 or not x.is_contiguous():
            raise _capi.ExtensionError("norm_rope takes contiguous bfloat16 tensors")
    for x in (cos, sin):
        if x.dtype != torch.float32 or not x.is_contiguous() or tuple(x.shape) != (S - text_len, D):
            raise _capi.ExtensionError("cos and sin must be contiguous fp32 tensors of shape [S - text_len, D]")
    if k.shape != q.shape or any(x.numel() != D for x in (q_norm[0], q_norm[1], k_norm[0], k_norm[1])):
        raise _capi.ExtensionError("q and k must have one shape; weights and biases hold D elements")
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rc = lib.dtb_norm_rope(
        q.data_ptr(), qo.data_ptr(), q_norm[0].data_ptr(), q_norm[1].data_ptr(), float(q_norm[2]),
        k.data_ptr(), ko.data_ptr(), k_norm[0].data_ptr(), k_norm[1].data_ptr(), float(k_norm[2]),
        cos.data_ptr(), sin.data_ptr(), B, S, text_len, H, D, _stream_ptr())
    _capi.check(rc, "dtb_norm_rope")
    LaunchLog.count += 1
    return qo, ko


class GridRope(NamedTuple):
    """Rotary positions of tokens that are places of a (time, height, width) grid, in row-major order.  An axis with d of a head's
    channels turns its pair i by (origin + step * index) * base^(-2 i / d).  The places lie in `shards` pieces as split_tensor_uneven
    makes them, padding included, and `first` is the number of a sequence's first video token among those: 0 for all pieces one
    after another, r * ceil(places / shards) for rank r's.  Tokens behind the last piece are padding too."""
    grid: Tuple[int, int, int]
    axes: Tuple[int, int, int]
    base: float = 10000.0
    origin: Tuple[float, float, float] = (0.0, 0.0, 0.0)
    step: Tuple[float, float, float] = (1.0, 1.0, 1.0)
    first: int = 0
    shards: int = 1


@functools.lru_cache(maxsize=64)
def _rope_arrays(grid, axes, base, origin, step):
    """What the C interface reads of a GridRope (host arrays, read at the launch)."""
    if not all(0 <= n < 1 << 31 for n in (*grid, *axes)):
        raise _capi.ExtensionError("a grid's extents and an axis's channels are not negative and below 2^31")
    return (ctypes.c_int * 3)(*grid), (ctypes.c_int * 3)(*axes), (ctypes.c_double * 7)(base, *origin, *step)


Norm = Tuple[torch.Tensor, Optional[torch.Tensor], float]


def _grid_rope_args(q, k, norms, rope, text_len, video_len):
    """Checks what both passes are given; returns (shapes, element type, arguments from `grid` on)."""
    shape, kshape, dtype = q.shape, k.shape, q.dtype
    if len(shape) != 4 or len(kshape) != 4 or shape[:2] != kshape[:2] or shape[3] != kshape[3]:
        raise _capi.ExtensionError("q and k are [B,S,H,D] and [B,S,Hk,D]")
    B, S, H, D = shape
    video_len = S - text_len if video_len is None else video_len
    if text_len < 0 or video_len < 0 or text_len + video_len > S:
        raise _capi.ExtensionError("text and video tokens lie within the sequence")
    if dtype not in _VALUES or k.dtype != dtype:
        raise _capi.ExtensionError("q and k must be bfloat16 or float32 alike")
    for w, b, _ in norms:
        for x in (w,) if b is None else (w, b):
            if x.dtype != dtype or x.numel() != D or not x.is_contiguous():
                raise _capi.ExtensionError("weights and biases hold D contiguous elements of q's type")
    grid, axes, base, origin, step, first, shards = rope
    if not 0 < shards < 1 << 31 or not 0 <= first < 1 << 62:
        raise _capi.ExtensionError("shards and first are positions among the pieces")
    # (as plain numbers: what is kept goes by their values, and a tensor among them would be known by its identity)
    arrays = _rope_arrays(tuple(grid), tuple(axes), float(base), tuple(map(float, origin)), tuple(map(float, step)))
    return shape, kshape, _VALUES[dtype], (*arrays, first, shards, B, S, text_len, video_len, H, kshape[2], D)


def norm_rope_grid(q: torch.Tensor, k: torch.Tensor, q_norm: Norm, k_norm: Norm, rope: GridRope, *, text_len: int = 0,
                   video_len: Optional[int] = None, rms: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Layer norm (RMS norm with `rms`) over D of q [B,S,H,D] and k [B,S,Hk,D], bf16 or fp32, norms as (weight, bias or None, eps);
    then rotary positions of the `video_len` tokens (None: all) behind the first `text_len`, from their place in rope's grid.
    Any token and batch strides that are multiples of 16 bytes; new contiguous tensors, one launch.  Padding behind the grid's
    last place comes out as 0, as with zero-padded tables."""
    (qw, qb, q_eps), (kw, kb, k_eps) = q_norm, k_norm
    stream = _launch_stream(q, k, qw, qb, kw, kb)
    shape, kshape, dtype, rest = _grid_rope_args(q, k, (q_norm, k_norm), rope, text_len, video_len)
    qo, ko = _empty_like(q, q.dtype), _empty_like(k, k.dtype)
    if q.numel() == 0 and k.numel() == 0:
        return qo, ko
    rc = _capi.load().dtb_norm_rope_grid(
        q.data_ptr(), *_strides(q, shape), qo.data_ptr(), qw.data_ptr(), None if qb is None else qb.data_ptr(), q_eps,
        k.data_ptr(), *_strides(k, kshape), ko.data_ptr(), kw.data_ptr(), None if kb is None else kb.data_ptr(), k_eps,
        dtype, rms, *rest, stream)
    if rc:
        _capi.check(rc, "dtb_norm_rope_grid")
    LaunchLog.count += 1
    return qo, ko


_ROPE_SCRATCH = {}        # (device, D) -> bytes that the backward pass needs


def norm_rope_grid_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, q_norm: Norm, k_norm: Norm, rope: GridRope, *,
                            text_len: int = 0, video_len: Optional[int] = None, rms: bool = False) -> Tuple[Optional[torch.Tensor], ...]:
    """Gradients of norm_rope_grid's inputs from those of its results, dq and dk: (q's, k's, q_norm's weight and bias, k_norm's
    weight and bias), None for a bias that is None.  Two launches; the sums for the weights are taken in a fixed order."""
    (qw, qb, q_eps), (kw, kb, k_eps) = q_norm, k_norm
    stream = _launch_stream(dq, dk, q, k, qw, qb, kw, kb)
    shape, kshape, dtype, rest = _grid_rope_args(q, k, (q_norm, k_norm), rope, text_len, video_len)
    if dq.shape != shape or dk.shape != kshape or dq.dtype != q.dtype or dk.dtype != q.dtype:
        raise _capi.ExtensionError("dq and dk have the shapes and the type of q and k")
    gq, gk = _empty_like(q, q.dtype), _empty_like(k, k.dtype)
    sums = [None if x is None else torch.empty_like(x) for x in (qw, qb, kw, kb)]
    if q.numel() == 0 and k.numel() == 0:
        return (gq, gk, *(None if x is None else x.zero_() for x in sums))
    lib = _capi.load()
    key = (q.get_device(), shape[3])
    need = _ROPE_SCRATCH.get(key)
    if need is None:
        need = lib.dtb_norm_rope_grid_scratch_bytes(shape[3])
        if need < 0:
            _capi.check(need, "dtb_norm_rope_grid_scratch_bytes")
        _ROPE_SCRATCH[key] = need
    scratch = _empty((need,), torch.uint8, q.device)
    rc = lib.dtb_norm_rope_grid_backward(
        dq.data_ptr(), *_strides(dq, shape), dk.data_ptr(), *_strides(dk, kshape),
        q.data_ptr(), *_strides(q, shape), qw.data_ptr(), q_eps, k.data_ptr(), *_strides(k, kshape), kw.data_ptr(), k_eps,
        gq.data_ptr(), gk.data_ptr(), *[None if x is None else x.data_ptr() for x in sums], dtype, rms, *rest,
        scratch.data_ptr(), need, stream)
    if rc:
        _capi.check(rc, "dtb_norm_rope_grid_backward")
    LaunchLog.count += 2
    return (gq, gk, *sums)


MOD_MAX_DIM = 3072


def _check_streams(video, text, *others):
    _need_cuda(video, text, *others)
    B, Sv, dim = video.shape
    if text.dim() != 3 or text.shape[0] != B or text.shape[2] != dim:
        raise _capi.ExtensionError("video and text must be [B, S, dim] tensors of one batch and width")
    for x in (video, text, *others):
        if x.dtype != torch.bfloat16 or not x.is_contiguous():
            raise _capi.ExtensionError("contiguous bfloat16 tensors expected")
    return B, Sv, text.shape[1], dim


def ln_modulate(video: torch.Tensor, text: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float,
                mod: torch.Tensor) -> torch.Tensor:
    """Layer norm of both streams, modulated by `mod` [B, 6 dim] (shift, scale, gate of video, then of text): the joint
    tensor [B, text + video, dim], text first, in one launch."""
    B, Sv, St, dim = _check_streams(video, text, weight, bias, mod)
    if weight.numel() != dim or bias.numel() != dim or tuple(mod.shape) != (B, 6 * dim):
        raise _capi.ExtensionError("weight and bias hold dim elements, mod is [B, 6 dim]")
    out = torch.empty(B, St + Sv, dim, dtype=torch.bfloat16, device=video.device)
    rc = _capi.load().dtb_ln_modulate(video.data_ptr(), text.data_ptr(), weight.data_ptr(), bias.data_ptr(), float(eps),
                                      mod.data_ptr(), out.data_ptr(), B, Sv, St, dim, _stream_ptr())
    _capi.check(rc, "dtb_ln_modulate")
    LaunchLog.count += 1
    return out


def gate_add(video: torch.Tensor, text: torch.Tensor, a: torch.Tensor, mod: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(video, text) + gate * (their parts of the joint tensor a [B, text + video, dim]), gates from `mod` as in
    ln_modulate; new tensors, one launch."""
    B, Sv, St, dim = _check_streams(video, text, a, mod)
    if tuple(a.shape) != (B, St + Sv, dim) or tuple(mod.shape) != (B, 6 * dim):
        raise _capi.ExtensionError("a is [B, text + video, dim], mod is [B, 6 dim]")
    vo, to = torch.empty_like(video), torch.empty_like(text)
    rc = _capi.load().dtb_gate_add(video.data_ptr(), text.data_ptr(), a.data_ptr(), mod.data_ptr(), vo.data_ptr(), to.data_ptr(),
                                   B, Sv, St, dim, _stream_ptr())
    _capi.check(rc, "dtb_gate_add")
    LaunchLog.count += 1
    return vo, to


_DRIFT_SCRATCH = {}


def drift_accumulate(cur: torch.Tensor, prev: torch.Tensor, accum: torch.Tensor,
                     scratch: Optional[torch.Tensor] = None):
    """accum (one fp32 element on the device) += relative L1 drift of `cur` against `prev`
    (fp32, same number of elements), without a host round trip.  `scratch` defaults to a per-device
    buffer kept by this module and grown on demand."""
    lib = _capi.load()
    _need_cuda(cur, prev, accum, scratch)
    if cur.dtype != torch.float32 or prev.dtype != torch.float32 or accum.dtype != torch.float32:
        raise _capi.ExtensionError("drift_accumulate takes fp32 tensors")
    if cur.numel() != prev.numel() or accum.numel() != 1:
        raise _capi.ExtensionError("cur and prev must have equal sizes; accum must hold one element")
    cur, prev = cur.contiguous(), prev.contiguous()
    n = cur.numel()
    need = lib.dtb_drift_scratch_bytes(n)
    if scratch is None:
        key = cur.device
        scratch = _DRIFT_SCRATCH.get(key)
        if scratch is None or scratch.numel() < need:
            scratch = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=cur.device)
            _DRIFT_SCRATCH[key] = scratch
    rc = lib.dtb_drift_accumulate(cur.data_ptr(), prev.data_ptr(), n, accum.data_ptr(), scratch.data_ptr(),
                                  scratch.numel(), _stream_ptr())
    _capi.check(rc, "dtb_drift_accumulate")
    LaunchLog.count += 1
