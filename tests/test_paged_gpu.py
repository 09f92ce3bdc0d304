"""Keys and values in pages: tables, writes and attention over them, against the definitions (attention in 64 bits).

Tolerances of the attention are those of tests/test_flash_window_gpu.py: 2^-8 of each weight for its rounding to bf16, 1e-4 for the
scores, 2^-8 of a bf16 result.  Tables, slots and written pages are compared exactly."""
import math
import random

import pytest
import torch

from tests.test_flash_window_gpu import SCORE, _check, _exact, _rand, _visible

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ tables and slots
def _extend(table, lens, new, free, count, P, tokens):
    """(table, slots, cu, lens, count, missing) of plain lists."""
    table, M = [list(r) for r in table], len(table[0])
    need = sum(-(-(a + n) // P) - -(-a // P) for a, n in zip(lens, new))
    bad = any(a < 0 or n < 0 or a + n > M * P for a, n in zip(lens, new)) or sum(new) > tokens or not 0 <= count <= len(free)
    if bad or need > count:
        return table, [-1] * tokens, [0] * (len(lens) + 1), list(lens), count, -1 if bad else need - count
    slots, cu = [], [0]
    for b, n in enumerate(new):
        for x in range(lens[b], lens[b] + n):
            if x % P == 0:
                count -= 1
                table[b][x // P] = free[count]
            page = table[b][x // P]              # (-1 where a stream that was cut short had given its last page back before)
            slots.append(page * P + x % P if page >= 0 else -1)
        cu.append(len(slots))
    return table, slots + [-1] * (tokens - len(slots)), cu, [a + n for a, n in zip(lens, new)], count, 0


def _release(table, lens, free, count, begin, end, P):
    table, free, left = [list(r) for r in table], list(free), []
    for b, n in enumerate(lens):
        for j in range(len(table[0])):
            last = min((j + 1) * P, n) - 1
            goes = j * P < n and j * P >= begin[b] and (last < end[b] if end[b] >= n else (j + 1) * P <= end[b])
            if goes and table[b][j] >= 0:
                free[count], table[b][j] = table[b][j], -1
                count += 1
        left.append(max(begin[b], 0) if end[b] >= n and begin[b] < n else n)
    return table, left, free, count


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class _Pages:
    """Streams on the device, and the same as lists."""

    def __init__(self, lens, P, columns, spare, seed=0):
        self.P, self.pages = P, sum(-(-n // P) for n in lens) + spare
        order = list(range(self.pages))
        random.Random(seed).shuffle(order)
        self.lens, self.table = list(lens), []
        at = 0
        for n in lens:
            used = -(-n // P)
            self.table.append(order[at:at + used] + [-1] * (columns - used))
            at += used
        self.free, self.count = order[at:] + order[:at], self.pages - at
        self.load()

    def load(self):
        self.g = [_i(x) for x in (self.table, self.lens, self.free, [self.count])]

    def extend(self, new, tokens):
        from ditango_b200 import ops
        table, lens, free, count = self.g
        plan = ops.extend_pages(table, lens, _i(new), free, count, self.P, tokens)
        want = _extend(self.table, self.lens, new, self.free, self.count, self.P, tokens)
        got = (table.tolist(), plan.slots.tolist(), plan.cu_seqlens.tolist(), plan.seqlens.tolist(), plan.free_count.item(), plan.missing.item())
        assert got == want and lens.tolist() == self.lens and count.item() == self.count
        self.table, _, _, self.lens, self.count, _ = want
        self.g[1], self.g[3] = plan.seqlens, plan.free_count
        return plan

    def release(self, begin, end, in_place):
        from ditango_b200 import ops
        table, lens, free, count = self.g
        out = None if in_place else torch.empty_like(table)
        got = ops.release_pages(table, lens, free, count, _i(begin), _i(end), self.P, out_table=out)
        want = _release(self.table, self.lens, self.free, self.count, begin, end, self.P)
        assert got.table is (table if in_place else out) and (in_place or table.tolist() == self.table)
        assert (got.table.tolist(), got.seqlens.tolist(), free.tolist(), got.free_count.item()) == want
        self.table, self.lens, self.free, self.count = want
        self.g = [got.table, got.seqlens, free, got.free_count]


@pytest.mark.parametrize("P", [16, 64, 1024])
@pytest.mark.parametrize("streams", [1, 3, 70, 600])
def test_streams_that_come_grow_and_go(streams, P):
    rng = random.Random(streams * P)
    pages = _Pages([rng.choice((0, 1, P - 1, P, P + 1, rng.randrange(5 * P))) for _ in range(streams)], P, 12, 7 * streams + 3, seed=streams)
    for step in range(12):
        new = [rng.choice((0, 1, 1, P, rng.randrange(2 * P))) for _ in range(streams)]
        if rng.random() < 0.3:
            new = [1] * streams
        pages.extend(new, sum(new) + rng.choice((0, 0, 1, 50)))
        if step % 2:
            begin = [rng.choice((0, 0, rng.randrange(3 * P))) for _ in range(streams)]
            end = [rng.choice((0, rng.randrange(6 * P), 10 ** 6, n, n - 1)) for n in pages.lens]
            pages.release(begin, end, step % 4 == 1)
    held = [p for row in pages.table for p in row if p >= 0]
    assert sorted(held + pages.free[:pages.count]) == list(range(pages.pages))


def test_long_rows_and_many_pages():
    pages = _Pages([70000, 0, 33, 51200], 16, 6000, 9000)
    pages.extend([5000, 20000, 1, 44800], 70000)
    pages.release([40, 0, 0, 16 * 256], [60000, 10, 33, 16 * 4000], False)
    pages.release([0, 0, 0, 0], [10 ** 9] * 4, True)
    assert pages.count == pages.pages and pages.lens == [0] * 4
    pages.extend([1, 0, 0, 17], 18)


def test_what_cannot_be_had_takes_nothing():
    pages = _Pages([20, 3, 64], 16, 8, 2)
    pages.extend([12, 12, 33], 60)                         # 0 + 0 + 3 pages, two are free
    assert pages.lens == [20, 3, 64] and pages.count == 2
    pages.extend([1, 2 ** 31 - 1, 1], 100)
    pages.extend([1, 126, 1], 200)                         # a row of 8 pages holds 128
    pages.extend([1, -1, 1], 200)
    pages.extend([3, 3, 3], 8)                             # more than the rows that there are
    pages.extend([0, 0, 0], 0)
    pages.extend([12, 13, 32], 57)
    assert pages.count == 0 and pages.lens == [32, 16, 96]
    pages.lens[1], pages.count = -5, 9
    pages.load()
    pages.extend([1, 1, 1], 3)


def test_a_list_that_is_full_is_not_written_past_its_end():
    """Pages that were given back already, by numbers that are not right."""
    from ditango_b200 import ops
    guard = torch.full((64,), 77, dtype=torch.int32, device="cuda")
    free = guard[16:24]
    free.copy_(torch.arange(8))
    table = _i([[0, 1, 2, 3]])
    got = ops.release_pages(table, _i([64]), free, _i([6]), _i([0]), _i([64]), 16)
    assert free.tolist() == [0, 1, 2, 3, 4, 5, 0, 1] and got.free_count.item() == 8 and got.seqlens.item() == 0
    assert (guard[:16] == 77).all() and (guard[24:] == 77).all()


# ------------------------------------------------------------------------------------------------ writes
def _pool(pages, P, Hk, D, layout, seed=3):
    """[pages, P, Hk, D]: heads of a token together ("token"), tokens of a head together ("head"), keys and values in one tensor ("both")."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "token":
        return [torch.randn(pages, P, Hk, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    if layout == "head":
        return [torch.randn(pages, Hk, P, D, generator=g, device="cuda").to(torch.bfloat16).transpose(1, 2) for _ in range(2)]
    both = torch.randn(pages, 2, Hk, P, D + 8, generator=g, device="cuda").to(torch.bfloat16)
    return [both[:, i, :, :, :D].transpose(1, 2) for i in range(2)]


@pytest.mark.parametrize("layout", ["token", "head", "both"])
@pytest.mark.parametrize("T,Hk,D,P", [(1, 1, 64, 16), (7, 3, 128, 16), (300, 8, 64, 64), (33, 24, 128, 128), (1000, 5, 64, 256)])
def test_writes_go_to_their_slots_and_nowhere_else(T, Hk, D, P, layout):
    from ditango_b200 import ops
    pages = T // P + 5
    k_pages, v_pages = _pool(pages, P, Hk, D, layout)
    slots = torch.randperm(pages * P, generator=torch.Generator().manual_seed(T))[:T].int()
    slots[::5] = -1
    slots[3::11] = torch.tensor([pages * P, -7, 2 ** 31 - 1], dtype=torch.int32).repeat(T)[:slots[3::11].numel()]
    x = torch.randn(T, 3, Hk, D, device="cuda").to(torch.bfloat16)
    for k, v in ((x[:, 0].contiguous(), x[:, 1].contiguous()), (x[:, 1], x[:, 2])):
        want = []
        for pool, new in ((k_pages, k), (v_pages, v)):
            flat = pool.reshape(pages * P, Hk, D).clone()
            there = (slots >= 0) & (slots < pages * P)
            flat[slots[there].long().cuda()] = new[there.cuda()]
            want.append(flat.view(pages, P, Hk, D))
        ops.write_pages(k, v, k_pages, v_pages, slots.cuda())
        assert torch.equal(k_pages, want[0]) and torch.equal(v_pages, want[1])


def test_a_batch_and_a_pool_beyond_32_bits():
    from ditango_b200 import ops
    pages, P, Hk, D = 2 ** 16, 32, 16, 128                  # 2^32 elements and a page
    both = torch.zeros(pages + 1, 2, P, Hk, D, dtype=torch.bfloat16, device="cuda")
    k_pages, v_pages = both[:, 0], both[:, 1]
    x = torch.randn(2, 3, Hk, D, device="cuda").to(torch.bfloat16)
    slots = _i([5, pages * P + 31, (pages - 1) * P, pages // 2 * P + 1, 0, pages * P])
    ops.write_pages(x, 2 * x, k_pages, v_pages, slots)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(k_pages[s // P, s % P], x.flatten(0, 1)[i]) and torch.equal(v_pages[s // P, s % P], 2 * x.flatten(0, 1)[i])
    assert both.count_nonzero().item() <= 2 * x.numel()
    # ... and read again, as one key and value of a sequence whose page lies behind 2^32 elements
    q = torch.randn(1, 1, Hk, D, device="cuda").to(torch.bfloat16)
    out, lse = ops.flash_paged(q, k_pages, v_pages, _i([[pages]]), _i([32]), left=0, right=0)
    # (its weight is 2 to a difference of two products rounded apart, not 1, and is rounded to bf16 where the sum is not: 2^-8, as everywhere)
    value = 2 * x[0, 1].float()
    assert ((out[0, 0] - value).abs() <= 2.0 ** -8 * value.abs()).all()
    assert (lse[0, :, 0].double() - (q[0, 0].double() * x[0, 1].double()).sum(-1) / math.sqrt(D)).abs().max() < SCORE
    q = torch.randn(1, 300, Hk, D, device="cuda").to(torch.bfloat16)
    out, _ = ops.flash_paged(q, k_pages, v_pages, _i([[pages] * 10]), _i([320]), left=0, right=0)
    assert ((out[0, 299] - value).abs() <= 2.0 ** -8 * value.abs()).all() and torch.equal(out[0, 298], torch.zeros_like(out[0, 298]))
    assert ops.read_status() == 0


# ------------------------------------------------------------------------------------------------ attention
class _Cache:
    """Sequences' keys and values, dense on the host and in pages on the device; what no sequence holds is NaN."""

    def __init__(self, lens, Hk, D, P, layout="head", seed=0, spare_columns=1, anything=()):
        self.k, self.v = ([_rand((n, Hk, D), 100 * seed + 2 * b + i) for b, n in enumerate(lens)] for i in range(2))
        self.lens, self.P = lens, P
        used = [-(-n // P) for n in lens]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.k_pages, self.v_pages = _pool(pages, P, Hk, D, layout)
        self.k_pages.fill_(math.nan)
        self.v_pages.fill_(math.nan)
        table = torch.full((len(lens), max(used) + spare_columns), -1, dtype=torch.int32)
        behind = (-1, pages, 2 ** 31 - 1, -2 ** 31, order[-1])                # what a row holds behind its last page
        for b, n in enumerate(used):
            mine, order = order[:n], order[n:]
            table[b] = torch.tensor([behind[(b + j) % 5] for j in range(table.shape[1])], dtype=torch.int32)
            table[b, :n] = torch.tensor(mine, dtype=torch.int32)
            for dst, src in ((self.k_pages, self.k[b]), (self.v_pages, self.v[b])):
                for j, page in enumerate(mine):
                    part = src[j * P:(j + 1) * P].cuda()
                    dst[page, :part.shape[0]] = part
        self.table, self.seqlens = table.cuda(), _i(lens)


def _attend(cache, q, new, *, left=-1, right=-1, sinks=0, packed=True, **kw):
    """Checks the sequences' results; q [T,H,D] on the host."""
    from ditango_b200 import ops
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    kw.setdefault("lse_layout", ops.LSE_BSH)
    gq = q.cuda()
    if packed:
        kw.update(cu_seqlens_q=_i(cu))
        kw.setdefault("max_seqlen_q", max(new))
    else:
        gq = gq.view(len(new), new[0], *q.shape[1:])
    out, lse = ops.flash_paged(gq, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, left=left, right=right, sinks=sinks, **kw)
    flat_out, flat_lse = (out, lse) if packed else (out.flatten(0, 1), lse.flatten(0, 1))
    for b, (n, total) in enumerate(zip(new, cache.lens)):
        seen = _visible(n, total, left, right, sinks, total - n, 0)
        if left < 0 and right < 0:
            seen = torch.ones(n, total, dtype=torch.bool)
        _check(flat_out[cu[b]:cu[b + 1]], flat_lse[cu[b]:cu[b + 1]], *_exact(q[cu[b]:cu[b + 1]], cache.k[b], cache.v[b], seen))
    assert ops.read_status() == 0
    return out, lse


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (-1, 40, 9), (0, 0, 3), (37, 0, 0), (100, 60, 21), (200, 0, 300), (2 ** 30, 2 ** 30, 2 ** 30)]
# queries, lengths, heads, key heads: rows from 1 to 64 and more, lengths of zero and one, around tiles of 64 and 128
TOKENS = [([1], [1], 1, 1), ([1], [700], 3, 3), ([1, 1, 1], [1300, 0, 64], 8, 1), ([2, 0, 5], [515, 33, 5], 8, 2), ([17], [1000], 4, 4),
          ([8], [2111], 8, 1), ([1, 16, 3, 1, 0, 9], [127, 129, 1, 2000, 0, 448], 8, 2), ([33], [300], 2, 1), ([4, 100], [2, 60], 6, 3)]
CHUNKS = [([257], [257], 2, 2), ([200, 1, 700], [900, 333, 700], 4, 2), ([300, 130], [1111, 64], 3, 1), ([129, 513, 0, 2, 150], [129, 1000, 40, 0, 149], 2, 2)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("P", [16, 32, 128])
@pytest.mark.parametrize("new,lens,H,Hk", TOKENS)
def test_tokens_match_the_definition(new, lens, H, Hk, P, left, right, sinks, D):
    cache = _Cache(lens, Hk, D, P, layout=("head", "token", "both")[len(new) % 3])
    dtype = torch.bfloat16 if (sum(new) + left) % 2 else torch.float32
    _attend(cache, _rand((sum(new), H, D), 50), new, left=left, right=right, sinks=sinks, out_dtype=dtype)


# rows of a key head from 33 to 96: one block of 48, or two
ROWS48 = [([5, 2, 0], [900, 70, 9], 16, 2), ([3], [2111], 48, 3), ([33], [1290], 2, 2), ([12, 1, 9], [3000, 64, 500], 8, 1), ([9, 11, 0, 5], [9, 4000, 3, 129], 16, 2),
          ([24, 17, 2], [1000, 17, 65], 4, 1), ([48, 50, 1], [48, 2000, 700], 3, 3)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("new,lens,H,Hk", ROWS48)
def test_rows_in_blocks_of_48(new, lens, H, Hk, left, right, sinks, D):
    cache = _Cache(lens, Hk, D, 32, layout=("head", "token", "both")[len(new) % 3], seed=15)
    _attend(cache, _rand((sum(new) + 1, H, D), 69), new, left=left, right=right, sinks=sinks, out_dtype=torch.bfloat16 if H % 4 else torch.float32)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("new,lens,H,Hk", CHUNKS)
def test_chunks_match_the_definition(new, lens, H, Hk, P, left, right, sinks, D):
    cache = _Cache(lens, Hk, D, P, layout=("head", "token", "both")[len(new) % 3], seed=1)
    dtype = torch.bfloat16 if (sum(new) + left) % 2 else torch.float32
    _attend(cache, _rand((sum(new), H, D), 51), new, left=left, right=right, sinks=sinks, out_dtype=dtype)


# few blocks against many keys (all split), a last round of blocks that is mostly empty (some split), both among short sequences, more sequences
# than blocks are planned for, lengths that a plan has to order
SPLITS = [([300], [6000], 2, 1, -1, 0, 0), ([140, 1, 600], [9000, 4000, 700], 2, 2, -1, 0, 0), ([129], [5000], 1, 1, 900, 0, 70), ([1000], [1200], 40, 1, -1, -1, 0),
          ([700, 300, 900], [800, 4000, 900], 24, 1, -1, 0, 0), ([600], [2500], 60, 1, 500, 100, 30), ([200, 1, 130] * 100, [220, 90, 140] * 100, 2, 2, -1, 0, 0),
          ([130, 260, 0, 513] * 5, [140, 3000, 77, 1500] * 5, 2, 1, -1, 10, 0), ([129] * 3, [0, 5, 4000], 4, 4, -1, 0, 0)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,lens,H,Hk,left,right,sinks", SPLITS)
def test_blocks_whose_keys_are_split(new, lens, H, Hk, left, right, sinks, D):
    """(the kernel of few rows takes up to 64 / (H / Hk) queries)"""
    cache = _Cache(lens, Hk, D, 64, seed=9)
    q = _rand((sum(new), H, D), 61)
    _attend(cache, q, new, left=left, right=right, sinks=sinks, out_dtype=torch.bfloat16 if H % 4 else torch.float32)


# heads that share the rows of a tile: powers of two of them, and the power of two in other numbers; tokens around the ends of blocks
SHARED = [([65], [700], 8, 8), ([33, 40], [500, 41], 16, 8), ([9, 17, 100, 1], [300, 17, 1000, 5], 16, 2), ([3, 70], [400, 300], 48, 2), ([2, 3], [129, 700], 64, 1),
          ([1, 2, 5], [60, 2, 900], 128, 1), ([30], [2000], 12, 1), ([64, 65, 31], [64, 400, 333], 24, 6), ([40, 200], [40, 777], 5, 1), ([129], [1500], 6, 2)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (-1, -1, 0), (90, 20, 33), (3, 0, 0)])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("new,lens,H,Hk", SHARED)
def test_heads_that_share_tiles(new, lens, H, Hk, packed, left, right, sinks, D):
    if not packed:
        new = [max(new)] * len(new)
    cache = _Cache(lens, Hk, D, 32, layout="token" if H % 3 else "head", seed=14)
    dtype = torch.bfloat16 if (H + left) % 2 else torch.float32
    _attend(cache, _rand((sum(new), H, D), 68), new, left=left, right=right, sinks=sinks, packed=packed, out_dtype=dtype)


@pytest.mark.parametrize("D", [64, 128])
def test_split_blocks_fold_into_a_state(D):
    from ditango_b200 import ops
    new, lens, H = [200, 140], [5000, 300], 4
    cache = _Cache(lens, 2, D, 16, seed=10)
    T = sum(new) + 3
    q = _rand((T, H, D), 62)
    old_k, old_v = _rand((40, 2, D), 63), _rand((40, 2, D), 64)
    out, lse = ops.flash_window(q[None].cuda(), old_k[None].cuda(), old_v[None].cuda())
    out, lse = out[0].contiguous(), lse[0].contiguous()
    before = out.clone(), lse.clone()
    cu = [0, 200, 340]
    ops.flash_paged(q.cuda(), cache.k_pages, cache.v_pages, cache.table, cache.seqlens, left=2000, right=0, sinks=9, cu_seqlens_q=_i(cu), max_seqlen_q=200, out=out, lse=lse,
                    accumulate=True)
    assert torch.equal(out[340:], before[0][340:]) and torch.equal(lse[:, 340:], before[1][:, 340:])
    for b, n in enumerate(new):
        seen = torch.cat([torch.ones(n, 40, dtype=torch.bool), _visible(n, lens[b], 2000, 0, 9, lens[b] - n, 0)], 1)
        want, want_lse, spread = _exact(q[cu[b]:cu[b + 1]], torch.cat([old_k, cache.k[b]]), torch.cat([old_v, cache.v[b]]), seen)
        _check(out[cu[b]:cu[b + 1]], lse.t()[cu[b]:cu[b + 1]], want, want_lse, 1.01 * spread)
    assert ops.read_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 5, 70, 300])
def test_dense_queries_and_both_layouts_of_lse(n, D):
    from ditango_b200 import ops
    lens = [n, 500, 0, 1029]
    cache = _Cache(lens, 2, D, 32, seed=2)
    q = _rand((4 * n, 6, D), 52)
    out, lse = _attend(cache, q, [n] * 4, right=0, packed=False)
    again, bhs = ops.flash_paged(q.cuda().view(4, n, 6, D), cache.k_pages, cache.v_pages, cache.table, cache.seqlens, right=0)
    assert torch.equal(bhs, lse.transpose(1, 2)) and torch.equal(again, out)
    for hint in (1, 77, 10 ** 6):              # (about the longest length: other numbers of CTAs, and so other roundings)
        _attend(cache, q, [n] * 4, right=0, packed=False, max_seqlen_k=hint)
    fused = torch.randn(4, n, 3, 6, D, device="cuda").to(torch.bfloat16)
    fused[:, :, 1] = q.cuda().view(4, n, 6, D)
    view, _ = ops.flash_paged(fused[:, :, 1], cache.k_pages, cache.v_pages, cache.table, cache.seqlens, right=0)
    assert torch.equal(view, out)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [[1, 3, 0], [200, 3, 300]])
def test_states_merge_with_those_of_other_kernels_and_rows_behind_the_last_stay(new, D):
    """The window's state folded into that of other keys; rows that no sequence has are not touched."""
    from ditango_b200 import ops
    lens, H, T = [900, 64, 333], 4, sum(new) + 5
    cache = _Cache(lens, 2, D, 16, seed=3)
    q = _rand((T, H, D), 53)
    old_k, old_v = _rand((50, 2, D), 54), _rand((50, 2, D), 55)
    out, lse = ops.flash_window(q[None].cuda(), old_k[None].cuda(), old_v[None].cuda(), lse_layout=ops.LSE_BSH)
    out, lse = out[0].contiguous(), lse[0].contiguous()
    before = out.clone(), lse.clone()
    cu = [sum(new[:b]) for b in range(4)]
    got = ops.flash_paged(q.cuda(), cache.k_pages, cache.v_pages, cache.table, cache.seqlens, right=0, cu_seqlens_q=_i(cu), max_seqlen_q=max(new), out=out, lse=lse,
                          accumulate=True, lse_layout=ops.LSE_BSH)
    assert got[0] is out and got[1] is lse
    assert torch.equal(out[cu[-1]:], before[0][cu[-1]:]) and torch.equal(lse[cu[-1]:], before[1][cu[-1]:])
    for b, n in enumerate(new):
        seen = torch.cat([torch.ones(n, 50, dtype=torch.bool), _visible(n, lens[b], -1, 0, 0, lens[b] - n, 0)], 1)
        want, want_lse, spread = _exact(q[cu[b]:cu[b + 1]], torch.cat([old_k, cache.k[b]]), torch.cat([old_v, cache.v[b]]), seen)
        # (two states and their merge: weights rounded once each)
        _check(out[cu[b]:cu[b + 1]], lse[cu[b]:cu[b + 1]], want, want_lse, 1.01 * spread)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 20, 140, 600])
@pytest.mark.parametrize("P", [16, 64, 128])
def test_keys_and_pages_that_nobody_sees_may_be_anything(n, P, D):
    """Keys between the first tokens and the windows hold infinities and NaN, and pages of them alone are gone from the table."""
    left, sinks, total = 133, 21, 2000
    cache = _Cache([total], 2, D, P, seed=4)
    hidden = ~_visible(n, total, left, 0, sinks, total - n, 0).any(0)
    for j in range(-(-total // P)):
        page, part = cache.table[0, j].item(), hidden[j * P:(j + 1) * P]
        cache.k_pages[page, :part.numel()][part.cuda()] = math.inf
        cache.v_pages[page, :part.numel()][part.cuda()] = math.nan
        if part.all():
            cache.table[0, j] = (-1, 2 ** 30, -5)[j % 3]
    _attend(cache, _rand((n, 4, D), 56), [n], left=left, right=0, sinks=sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 30, 200])
def test_a_page_outside_the_pool_is_one_of_zeros(n, D):
    cache = _Cache([700, 90], 2, D, 16, seed=5)
    for b, j, page in ((0, 3, -1), (0, 30, 10 ** 6), (1, 0, -2 ** 31)):
        cache.table[b, j] = page
        cache.k[b][16 * j:16 * j + 16] = 0
        cache.v[b][16 * j:16 * j + 16] = 0
    _attend(cache, _rand((2 * n, 4, D), 57), [n, n], right=0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_a_nan_that_is_seen_shows_and_stays_in_its_rows(n, D):
    from ditango_b200 import ops
    cache = _Cache([640, 640], 2, D, 64, seed=6)
    page = cache.table[1, 9].item()
    cache.k_pages[page, 63, 1, 5] = math.nan                # the second sequence's last key, second key head: its last query alone sees it
    q = _rand((2 * n, 4, D), 58)
    out, lse = ops.flash_paged(q.cuda(), cache.k_pages, cache.v_pages, cache.table, cache.seqlens, right=0, cu_seqlens_q=_i([0, n, 2 * n]), max_seqlen_q=n,
                               lse_layout=ops.LSE_BSH)
    nan = torch.zeros(2 * n, 4, dtype=torch.bool)
    nan[-1, 2:] = True
    assert torch.equal(lse.isnan().cpu(), nan) and torch.equal(out.isnan().all(-1).cpu(), nan) and torch.equal(out.isnan().any(-1).cpu(), nan)


@pytest.mark.parametrize("D", [64, 128])
def test_growing_scores(D):
    """Keys whose scores grow all along the sequence, so that references move many times, and far."""
    for n in (1, 20, 260):
        cache = _Cache([1500], 1, D, 32, seed=7)
        q = _rand((n, 2, D), 59)
        ramp = torch.linspace(0.1, 12, 1500)[:, None, None]
        cache.k[0] = (cache.k[0].float().abs() * ramp).to(torch.bfloat16)
        q = q.abs()
        for j in range(-(-1500 // 32)):
            part = cache.k[0][j * 32:(j + 1) * 32].cuda()
            cache.k_pages[cache.table[0, j].item(), :part.shape[0]] = part
        from ditango_b200 import ops
        out, lse = ops.flash_paged(q.cuda()[None], cache.k_pages, cache.v_pages, cache.table, cache.seqlens, right=0, lse_layout=ops.LSE_BSH)
        want, want_lse, spread = _exact(q, cache.k[0], cache.v[0], _visible(n, 1500, -1, 0, 0, 1500 - n, 0))
        # a score is a sum of D products in fp32: off by D 2^-24 of their sizes, here up to 12 * 4 * 4 each
        score = D * 2.0 ** -24 * D * 12 * 16 / math.sqrt(D)
        assert ((lse[0].cpu().double() - want_lse).abs() <= SCORE + score).all()
        assert ((out[0].cpu().double() - want).abs() <= (2.0 ** -8 + 2 * (SCORE + score)) * spread + 1e-30).all()


def test_results_are_the_same_on_every_run_and_stream():
    from ditango_b200 import ops
    lens = [20000, 17, 3000, 9999]
    cache = _Cache(lens, 2, 128, 16, seed=8)
    new = [1, 1, 3, 2]
    q = _rand((7, 8, 128), 60).cuda()
    kw = dict(right=0, cu_seqlens_q=_i([0, 1, 2, 5, 7]), max_seqlen_q=3)
    first = ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, **kw)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    others = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            others.append(ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, **kw))
    torch.cuda.synchronize()
    for o in others:
        assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])
    assert new and ops.read_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [3, 7, 20, 48, 65, 128, 200])
def test_any_number_of_heads_to_a_key_head(group, D):
    for new, lens, Hk in (([2, 1], [300, 1], 2), ([3], [2500], 1), ([1, 5, 0, 2], [64, 1000, 0, 2], 1)):
        cache = _Cache(lens, Hk, D, 16, seed=16)
        _attend(cache, _rand((sum(new), group * Hk, D), 70), new, right=0, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("hint", [0, 1, 100, 4000, 2 ** 31 - 1])
@pytest.mark.parametrize("new,lens,H,Hk", [([1], [3000], 8, 1), ([1] * 40, [700] * 39 + [20], 8, 2), ([70], [5000], 2, 2), ([300, 2], [9000, 2], 4, 2)])
def test_a_wrong_guess_of_the_lengths_does_no_harm(new, lens, H, Hk, hint):
    cache = _Cache(lens, Hk, 64, 32, seed=19)
    for left in (-1, 500):
        _attend(cache, _rand((sum(new), H, 64), 72), new, left=left, right=0, max_seqlen_k=hint)


def test_two_graphs_at_once():
    """(each has scratch of its own)"""
    from ditango_b200 import ops
    caches = [_Cache([3000, 40], 2, 64, 16, seed=17), _Cache([9000, 500, 7], 4, 128, 32, seed=18)]
    graphs, results, expected = [], [], []
    for cache, new, H in ((caches[0], [1, 1], 8), (caches[1], [5, 200, 2], 8), (caches[1], [1, 1, 1], 32), (caches[0], [300, 20], 4)):
        q, cu = _rand((sum(new), H, cache.k_pages.shape[-1]), 71).cuda(), _i([sum(new[:i]) for i in range(len(new) + 1)])

        def call():
            return ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, right=0, cu_seqlens_q=cu, max_seqlen_q=max(new))
        expected.append([x.clone() for x in call()])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(call())
        graphs[-1].inputs = q, cu
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for out, lse in results:
            out.zero_()
            lse.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert ops.read_status() == 0
        for got, want in zip(results, expected):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("n", [1, 4, 300])
def test_a_step_in_a_graph(n):
    """Pages, writes and attention of one step captured; lengths, tables and tokens of each replay are read from the device."""
    from ditango_b200 import ops
    P, Hk, H, D, B = 16, 2, 4, 64, 3
    pages = _Pages([5, 0, 300], P, 100, 200)
    table, lens, free, count = pages.g
    k_pages, v_pages = _pool(pages.pages, P, Hk, D, "head")
    dense = [[torch.zeros(0, Hk, D, dtype=torch.bfloat16) for _ in range(B)] for _ in range(2)]
    for b in range(B):
        x = [_rand((pages.lens[b], Hk, D), 70 + b), _rand((pages.lens[b], Hk, D), 80 + b)]
        slots = [pages.table[b][i // P] * P + i % P for i in range(pages.lens[b])]
        ops.write_pages(x[0].cuda(), x[1].cuda(), k_pages, v_pages, _i(slots))
        dense[0][b], dense[1][b] = x
    T = B * n
    q, k, v = (torch.zeros(T, h, D, dtype=torch.bfloat16, device="cuda") for h in (H, Hk, Hk))
    new = _i([n] * B)

    def step():
        plan = ops.extend_pages(table, lens, new, free, count, P, T)
        ops.write_pages(k, v, k_pages, v_pages, plan.slots)
        out, lse = ops.flash_paged(q, k_pages, v_pages, table, plan.seqlens, right=0, cu_seqlens_q=plan.cu_seqlens, max_seqlen_q=n, lse_layout=ops.LSE_BSH)
        lens.copy_(plan.seqlens)
        count.copy_(plan.free_count)
        return out, lse
    kept = [x.clone() for x in (table, lens, free, count)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip((table, lens, free, count), kept):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    total = list(pages.lens)
    for i in range(3):
        fresh = [_rand((T, h, D), 90 + 3 * i + j) for j, h in enumerate((H, Hk, Hk))]
        for dst, src in zip((q, k, v), fresh):
            dst.copy_(src)
        graph.replay()
        for b in range(B):
            rows = slice(b * n, (b + 1) * n)
            total[b] += n
            dense[0][b], dense[1][b] = torch.cat([dense[0][b], fresh[1][rows]]), torch.cat([dense[1][b], fresh[2][rows]])
            _check(out[rows], lse[rows], *_exact(fresh[0][rows], dense[0][b], dense[1][b], _visible(n, total[b], -1, 0, 0, total[b] - n, 0)))
    assert lens.tolist() == total and ops.read_status() == 0


@pytest.mark.parametrize("n", [1, 300])
def test_a_posted_status_keeps_results_from_being_written(n):
    from ditango_b200 import ops
    cache = _Cache([2000, 333], 2, 64, 16, seed=11)
    q = _rand((2 * n, 4, 64), 65).cuda()
    out, lse = torch.full((2 * n, 4, 64), 7.0, device="cuda"), torch.full((4, 2 * n), 7.0, device="cuda")
    kw = dict(right=0, cu_seqlens_q=_i([0, n, 2 * n]), max_seqlen_q=n)
    torch.cuda.synchronize()
    ops.post_status(5)
    ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, out=out, lse=lse, **kw)
    assert ops.read_status() == 5 and (out == 7).all() and (lse == 7).all()
    _attend(cache, q.cpu(), [n, n], right=0)


@pytest.mark.parametrize("n", [2, 200])
def test_offsets_beyond_the_rows_are_not_followed(n):
    """Offsets of the queries that end behind the rows, begin before them or fall: nothing outside the rows is read or written."""
    from ditango_b200 import ops
    cache = _Cache([500, 400, 300], 1, 64, 16, seed=12)
    guard = torch.full((n + 40, 2, 64), 7.0, device="cuda")
    lse_guard = torch.full((n + 40, 2), 7.0, device="cuda")
    q = _rand((n, 2, 64), 66).cuda()
    for cu in ([0, n // 2, n + 30, n + 60], [-20, n, n, n], [n, 0, n // 2, 2 * n], [2 ** 31 - 1, -2 ** 31, n, n]):
        guard.fill_(7.0)
        lse_guard.fill_(7.0)
        ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, right=0, cu_seqlens_q=_i(cu), max_seqlen_q=n, out=guard[20:20 + n], lse=lse_guard[20:20 + n],
                        lse_layout=ops.LSE_BSH)
        assert ops.read_status() == 0
        for x in (guard, lse_guard):
            assert (x[:20] == 7).all() and (x[20 + n:] == 7).all()


def test_launches_are_counted():
    # (the nodes of a captured call: it has no others than kernels)
    import ctypes

    from ditango_b200 import ops
    nodes = ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes
    nodes.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_size_t)]
    cache = _Cache([3000, 40], 2, 64, 16, seed=13)
    for new in ([1, 1], [300, 1], [300, 300]):
        q = _rand((sum(new), 4, 64), 67).cuda()
        kw = dict(right=0, cu_seqlens_q=_i([0, new[0], sum(new)]), max_seqlen_q=max(new))
        ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, **kw)
        torch.cuda.synchronize()
        before = ops.LaunchLog.count
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, **kw)
        n = ctypes.c_size_t()
        assert nodes(graph.raw_cuda_graph(), None, ctypes.byref(n)) == 0
        assert n.value == ops.LaunchLog.count - before


def test_other_devices_and_types_are_refused():
    from ditango_b200 import ops
    from ditango_b200._capi import ExtensionError
    cache = _Cache([40], 1, 64, 16)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.flash_paged(q.cpu(), cache.k_pages, cache.v_pages, cache.table, cache.seqlens),
                 lambda: ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table.cpu(), cache.seqlens),
                 lambda: ops.flash_paged(q, cache.k_pages, cache.v_pages.float(), cache.table, cache.seqlens),
                 lambda: ops.flash_paged(q.half(), cache.k_pages, cache.v_pages, cache.table, cache.seqlens),
                 lambda: ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens.long()),
                 lambda: ops.flash_paged(q, cache.k_pages[..., :32], cache.v_pages[..., :32], cache.table, cache.seqlens)):
        with pytest.raises(ExtensionError):
            call()
