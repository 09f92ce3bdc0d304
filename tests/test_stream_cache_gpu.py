"""Streams through StreamCache: extended, written, attended, their windows slid, cut short and ended, against attention in 64 bits over all that
each stream has been given (tolerances: tests/test_flash_window_gpu.py)."""
import random

import pytest
import torch

from tests.test_flash_window_gpu import _check, _exact, _rand, _visible

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class _Streams:
    """A cache and, per layer and stream, what it has been given."""

    def __init__(self, cache, H, seed=0):
        self.cache, self.H, self.n = cache, H, 0
        _, _, _, self.Hk, _, self.D = cache.pages.shape
        self.kv = [[[torch.zeros(0, self.Hk, self.D, dtype=torch.bfloat16) for _ in range(2)] for _ in range(cache.streams)] for _ in range(cache.layers)]

    def lens(self):
        return [self.kv[0][b][0].shape[0] for b in range(self.cache.streams)]

    def step(self, new, right=0, spare=0, **kw):
        from ditango_b200 import ops
        c = self.cache
        T = sum(new) + spare
        c.extend(_i(new), T)
        for layer in range(c.layers):
            self.n += 3
            q, k, v = _rand((T, self.H, self.D), self.n), _rand((T, self.Hk, self.D), self.n + 1), _rand((T, self.Hk, self.D), self.n + 2)
            out, lse = c.attend(layer, q.cuda(), k.cuda(), v.cuda(), right=right, max_new=max(new) or None, lse_layout=ops.LSE_BSH, **kw)
            at = 0
            for b, n in enumerate(new):
                rows = slice(at, at + n)
                at += n
                given = self.kv[layer][b]
                given[0], given[1] = torch.cat([given[0], k[rows]]), torch.cat([given[1], v[rows]])
                total = given[0].shape[0]
                seen = _visible(n, total, c.left, right, c.sinks, total - n, 0) if c.left >= 0 or right >= 0 else torch.ones(n, total, dtype=torch.bool)
                _check(out[rows], lse[rows], *_exact(q[rows], *given, seen))
        assert c.seqlens.tolist() == self.lens() and c.missing.item() == 0 and ops.read_status() == 0

    def pages_held(self):
        held = [p for row in self.cache.table.tolist() for p in row if p >= 0]
        free = self.cache.free.tolist()[:self.cache.free_count.item()]
        assert sorted(held + free) == list(range(self.cache.num_pages))
        return len(held)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,sinks,P", [(-1, 0, 16), (90, 21, 16), (128, 0, 64), (1, 5, 32), (0, 0, 16)])
def test_streams_of_frames_and_tokens(left, sinks, P, D):
    from ditango_b200.core.stream_cache import StreamCache
    cache = StreamCache(2, 4, 400, 2, D, 3000, page_size=P, left=left, sinks=sinks)
    s = _Streams(cache, 4)
    rng = random.Random(left + P)
    s.step([30, 0, 7, 300])                            # the text
    for i in range(6):
        s.step([rng.choice((0, 1, 1, 45, 200)) for _ in range(4)], right=rng.choice((0, -1, 30)), spare=rng.choice((0, 3)))
        cache.slide()
        held = s.pages_held()
        if left >= 0:                                  # no more than first tokens, window and a page at either end of each
            assert held <= sum(min(-(-n // P), -(-sinks // P) + -(-max(left, 1) // P) + 2) for n in s.lens())
    s.step([5, 5, 5, 5])                               # (of which three are dropped: what was there before them may be gone)
    # the third stream ends and begins anew in other pages; the second loses its newest tokens
    cache.finish(torch.tensor([False, False, True, False], device="cuda"))
    for layer in s.kv:
        layer[2] = [x[:0] for x in layer[2]]
    keep = max(0, s.lens()[1] - 3)
    cache.truncate(_i([10 ** 6, keep, 10 ** 6, 10 ** 6]))
    for layer in s.kv:
        layer[1] = [x[:keep] for x in layer[1]]
    assert cache.seqlens.tolist() == s.lens()
    s.pages_held()
    s.step([2, 5, 40, 1])
    cache.finish(torch.ones(4, dtype=torch.bool, device="cuda"))
    assert s.pages_held() == 0 and cache.seqlens.tolist() == [0] * 4


def test_a_pool_that_is_full_leaves_every_stream_as_it_was():
    from ditango_b200.core.stream_cache import StreamCache
    cache = StreamCache(1, 2, 4, 1, 64, 1000, page_size=16)
    s = _Streams(cache, 1)
    s.step([20, 10])
    cache.extend(_i([5, 25]), 30)                      # 1 + 2 + 2 pages
    assert cache.missing.item() == 1 and cache.seqlens.tolist() == [20, 10] and cache.free_count.item() == 1
    q = torch.randn(30, 1, 64, device="cuda").to(torch.bfloat16)
    before = cache.pages.clone()
    cache.attend(0, q, q, q, max_new=25)
    assert torch.equal(cache.pages.view(torch.int16), before.view(torch.int16))
    s.step([1, 6])
    cache.extend(_i([0, 990]), 990)                    # 16 + 990 tokens in 63 pages, one of them held, one free
    assert cache.missing.item() == 61
    cache.extend(_i([0, 993]), 993)                    # a row of 63 pages has room for 1008
    assert cache.missing.item() == -1 and cache.max_tokens == 1008


@pytest.mark.parametrize("left", [-1, 70])
def test_steps_replayed_from_a_graph(left):
    """One captured step of single tokens, with the window's slide, replayed: lengths, tables and the free list move on by themselves."""
    from ditango_b200 import ops
    from ditango_b200.core.stream_cache import StreamCache
    cache = StreamCache(2, 3, 60, 2, 64, 700, page_size=16, left=left, sinks=5)
    s = _Streams(cache, 4)
    s.step([100, 3, 31])
    new, T = _i([1, 1, 1]), 3
    q, k, v = (torch.zeros(2, T, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2))

    def step():
        cache.extend(new, T)
        got = [cache.attend(layer, q[layer], k[layer], v[layer], max_new=1, max_len=200, lse_layout=ops.LSE_BSH) for layer in range(2)]
        cache.slide()
        return got
    kept = [x.clone() for x in (cache.table, cache.seqlens, cache.free, cache.free_count, cache.pages)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip((cache.table, cache.seqlens, cache.free, cache.free_count, cache.pages), kept):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for i in range(40):
        fresh = [_rand((2, T, h, 64), 500 + 3 * i + j) for j, h in enumerate((4, 2, 2))]
        for dst, src in zip((q, k, v), fresh):
            dst.copy_(src)
        graph.replay()
        for layer, (out, lse) in enumerate(results):
            for b in range(3):
                given = s.kv[layer][b]
                for x in range(2):
                    given[x] = torch.cat([given[x], fresh[1 + x][layer, b:b + 1]])
                if i % 13 == 0 or i == 39:
                    total = given[0].shape[0]
                    _check(out[b:b + 1], lse[b:b + 1], *_exact(fresh[0][layer, b:b + 1], *given, _visible(1, total, left, 0, 5, total - 1, 0)))
    assert cache.seqlens.tolist() == s.lens() and cache.missing.item() == 0 and ops.read_status() == 0
    s.pages_held()


def test_refusals():
    from ditango_b200._capi import ExtensionError
    from ditango_b200.core.stream_cache import StreamCache
    cache = StreamCache(1, 2, 4, 1, 64, 100, page_size=16)
    q = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ExtensionError):
        cache.attend(0, q, q, q)
    cache.extend(_i([1, 1]), 2)
    with pytest.raises(ExtensionError):
        cache.attend(0, q, q, q)
    with pytest.raises(ExtensionError):
        cache.extend(_i([1]), 2)
