"""Keys and values of streams that grow, all layers of all streams in one pool of pages.

Where proCache keeps attention states between denoising steps, this keeps keys and values between chunks of a stream: latent frames
generated one after another behind their text, each attending what came before it, whole or through a sliding window with first tokens that
stay visible.  (The reference has no counterpart; its sequences are attended as a whole.)  Streams of one batch may have any lengths; what a
window leaves behind goes back to the pool.  Tables, lengths and the list of free pages stay on the device, and a step needs no host
round trip: the host knows how many rows of new tokens it hands over, nothing else."""
from typing import Optional, Tuple

import torch

from .. import ops as _engine
from .._capi import ExtensionError, LSE_BHS


class StreamCache:
    """`streams` streams of up to `max_tokens` tokens each share `num_pages` pages of `page_size` tokens (a power of two from 16), each page
    with a place in every one of `layers` layers.  `left` and `sinks`: keys visible before a query's own position (-1: all) and first tokens
    that stay visible, as in ops.flash_window; `right` of each call says what a chunk's tokens see behind themselves.

    A step: `extend`, then `attend` once per layer, then, with a window, `slide`.  All calls of one cache go on one stream, and can be captured
    into a CUDA graph together (numbers are updated in place)."""

    def __init__(self, layers: int, streams: int, num_pages: int, kv_heads: int, head_dim: int, max_tokens: int, *, page_size: int = 64, left: int = -1,
                 sinks: int = 0, device: Optional[torch.device] = None):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"page_size is a power of two from 16, not {page_size}")
        if min(layers, streams, num_pages, kv_heads, max_tokens) < 1 or head_dim not in (64, 128) or left < -1 or sinks < 0:
            raise ValueError("sizes are positive, head_dim is 64 or 128, left is -1 or more and sinks 0 or more")
        columns = -(-max_tokens // page_size)
        room = columns * page_size
        if (page_size > 1 << 20 or room >= 1 << 30 or max(streams * room, num_pages * page_size) >= 1 << 31 or max(left, sinks) > 1 << 30 or
                streams > 16384 or streams * -(-columns // 256) > 1 << 18):
            raise ValueError("pages hold up to 2^20 tokens, a stream fewer than 2^30, all streams and all pages fewer than 2^31 each; up to 16384 streams, "
                             "and 2^18 runs of 256 pages in their table")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if device.type != "cuda":
            raise ExtensionError("ditango_b200 kernels take CUDA tensors only")
        self.layers, self.streams, self.num_pages, self.page_size = layers, streams, num_pages, page_size
        self.left, self.sinks = left, sinks
        # the tokens of a page's head one after another: what attention reads of it is one run of memory
        self.pages = torch.empty(layers, 2, num_pages, kv_heads, page_size, head_dim, dtype=torch.bfloat16, device=device)
        self.max_tokens = room

        def ints(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device=device)
        self.table = ints(streams, columns, fill=-1)
        self.seqlens = ints(streams)
        self.free = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = ints(1, fill=num_pages)
        self.missing = ints(1)                # of the last extend: 0, or why nothing was taken (ops.extend_pages)
        self._zero, self._sinks = ints(streams), ints(streams, fill=sinks)
        self.plan: Optional[_engine.PagePlan] = None

    def keys(self, layer: int) -> torch.Tensor:
        """The keys' pages of a layer, [pages, page_size, heads, head_dim]."""
        return self.pages[layer, 0].transpose(1, 2)

    def values(self, layer: int) -> torch.Tensor:
        return self.pages[layer, 1].transpose(1, 2)

    def extend(self, new_lens: torch.Tensor, tokens: int) -> _engine.PagePlan:
        """Room for new_lens (int32 [streams]) tokens of each stream, which come as `tokens` rows, stream after stream, rows behind the last
        token being padding.  Without enough pages, or where a stream outgrows max_tokens, nothing happens to any stream, `missing` says so,
        and `attend` writes and returns nothing."""
        plan = _engine.extend_pages(self.table, self.seqlens, new_lens, self.free, self.free_count, self.page_size, tokens)
        self._keep(plan.seqlens, plan.free_count)
        self.missing.copy_(plan.missing)
        self.plan = plan
        return plan

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, right: int = 0, max_new: Optional[int] = None,
               max_len: Optional[int] = None, out_dtype: torch.dtype = torch.bfloat16, lse_layout: int = LSE_BHS,
               softmax_scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Writes the new tokens' k, v [tokens, kv_heads, head_dim] into the layer's pages and attends q [tokens, heads, head_dim] over them:
        (out, lse) of ops.flash_paged, packed, rows of padding left unwritten.  `max_new` is the largest of new_lens (`tokens` if not
        given), `max_len` about the longest stream's length, if the host knows them: kernels are chosen by both, and a token of each of many streams
        takes up to 1.7 times as long without `max_new`."""
        plan = self.plan
        if plan is None:
            raise ExtensionError("attend comes behind extend")
        if q.shape[0] != plan.slots.shape[0]:
            raise ExtensionError(f"q has {q.shape[0]} rows, extend was told of {plan.slots.shape[0]}")
        keys, values = self.keys(layer), self.values(layer)
        _engine.write_pages(k, v, keys, values, plan.slots)
        return _engine.flash_paged(q, keys, values, self.table, self.seqlens, left=self.left, right=right, sinks=self.sinks, cu_seqlens_q=plan.cu_seqlens,
                                   max_seqlen_q=max_new, max_seqlen_k=max_len, out_dtype=out_dtype, lse_layout=lse_layout, softmax_scale=softmax_scale)

    def slide(self):
        """Gives back the pages that no later token sees: behind the first tokens and before the window of the next one."""
        if self.left < 0:
            return
        # (a stream's last token stays: what ends at its end would count as cut short)
        end = (self.seqlens - max(self.left, 1)).clamp_(min=0)
        self._release(torch.minimum(self._sinks, end), end)

    def finish(self, over: torch.Tensor):
        """Streams where `over` (bool [streams]) are empty again."""
        self._release(self._zero, torch.where(over, self.seqlens, self._zero))

    def truncate(self, lengths: torch.Tensor):
        """Drops the tokens of each stream from lengths (int32 [streams]) on; a stream that is no longer than that stays as it is.  With a window only
        tokens since the last `slide` can be dropped: it has given back what a window that ends before them would see."""
        self._release(torch.minimum(lengths, self.seqlens), self.seqlens)

    def _release(self, begin: torch.Tensor, end: torch.Tensor):
        left = _engine.release_pages(self.table, self.seqlens, self.free, self.free_count, begin, end, self.page_size)
        self._keep(left.seqlens, left.free_count)

    def _keep(self, seqlens: torch.Tensor, free_count: torch.Tensor):
        self.seqlens.copy_(seqlens)
        self.free_count.copy_(free_count)
