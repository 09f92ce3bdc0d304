"""Keys and values in pages at the ends of what the calls take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("free", [6, 1])                 # room for the three pages, and not
def test_rows_up_to_the_largest_number(free):
    """Slots of 2^31 - 5 rows, with rows of another's in front of them and behind."""
    from ditango_b200 import _capi
    tokens, guard = 2 ** 31 - 5, 1 << 20
    slots = torch.full((guard + tokens + guard,), 7, dtype=torch.int32, device="cuda")
    table, lens, new, pages, count = _i([[0, -1, -1, -1], [-1] * 4]), _i([16, 0]), _i([20, 3]), _i([7, 6, 5, 4, 3, 2, 1, 0]), _i([free])
    cu, out, left, missing = _i([9] * 3), _i([9, 9]), _i([9]), _i([9])
    rc = _capi.load().dtb_extend_pages(table.data_ptr(), lens.data_ptr(), new.data_ptr(), pages.data_ptr(), count.data_ptr(), 2, 4, 8, 16,
                                       slots.data_ptr() + 4 * guard, tokens, cu.data_ptr(), out.data_ptr(), left.data_ptr(), missing.data_ptr(),
                                       torch.cuda.current_stream().cuda_stream)
    _capi.check(rc, "dtb_extend_pages")
    assert bool((slots[:guard] == 7).all()) and bool((slots[guard + tokens:] == 7).all())
    rows = slots[guard:guard + tokens]
    if free == 6:
        assert rows[:23].tolist() == [32 + i for i in range(16)] + [48 + i for i in range(4)] + [64 + i for i in range(3)]
        assert (missing.item(), left.item(), out.tolist(), cu.tolist()) == (0, 3, [36, 3], [0, 20, 23])
        rows = rows[23:]
    else:
        assert (missing.item(), left.item(), out.tolist(), cu.tolist()) == (2, 1, [16, 0], [0, 0, 0])
    for part in rows.split(1 << 28):
        assert bool((part == -1).all())


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("lens,n", [([2000, 333], 1), ([60000], 1), ([9000, 40, 3000], 9), ([5000], 1000), ([20000, 100], 300)])
def test_after_a_failure_nothing_is_stored_until_the_word_is_clear(lens, n, accumulate):
    """By every kernel: clusters, shares, tiles, tiles whose keys are split, and the launches that join."""
    from ditango_b200 import ops
    from tests.test_flash_window_gpu import _rand
    from tests.test_paged_gpu import _attend, _Cache
    cache = _Cache(lens, 2, 64, 16, seed=21)
    T = n * len(lens)
    q = _rand((T, 8, 64), 66).cuda()
    out, lse = torch.full((T, 8, 64), 7.0, device="cuda"), torch.full((8, T), 7.0, device="cuda")
    kw = dict(right=0, cu_seqlens_q=_i([n * i for i in range(len(lens) + 1)]), max_seqlen_q=n, accumulate=accumulate)
    torch.cuda.synchronize()
    ops.post_status(5)
    for _ in range(3):
        ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, out=out, lse=lse, **kw)
    assert ops.read_status() == 5 and bool((out == 7).all()) and bool((lse == 7).all())
    _attend(cache, q.cpu(), [n] * len(lens), right=0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (-1, -1, 0), (300, 20, 33)])
@pytest.mark.parametrize("hints", [True, False])
@pytest.mark.parametrize("new,lens", [([1500] + [1] * 299, [2000] + [70] * 299), ([2] * 150 + [0, 900] + [1] * 150, [50] * 150 + [0, 900] + [1] * 150), ([40] * 260, [100] * 260)])
def test_a_long_chunk_among_hundreds_of_streams(new, lens, hints, left, right, sinks, D):
    from tests.test_flash_window_gpu import _rand
    from tests.test_paged_gpu import _attend, _Cache
    cache = _Cache(lens, 2, D, 16, seed=22)
    q = _rand((sum(new), 8, D), 71)
    _attend(cache, q, new, left=left, right=right, sinks=sinks, **({} if hints else dict(max_seqlen_q=None)))


def test_as_many_streams_as_there_can_be_and_a_chunk_of_any_length():
    """Rows of one sequence times sequences are more than 2^31; the rows that there are, are not."""
    from ditango_b200 import ops
    streams, T, H, D, P = 65535, 262145, 32, 64, 16
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(T, H, D, device="cuda", generator=g).to(torch.bfloat16)
    k_pages, v_pages = (torch.randn(8, P, H, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    at = 40000                                            # the stream with all but one of the others' rows
    new = torch.ones(streams, dtype=torch.int64)
    new[at] = T - streams + 1
    table = (torch.arange(streams, dtype=torch.int32, device="cuda") % 8)[:, None].contiguous()
    lens = (torch.arange(streams, dtype=torch.int32, device="cuda") % 5 + 1).contiguous()
    lens[at] = 16
    cu = torch.zeros(streams + 1, dtype=torch.int32)
    cu[1:] = new.cumsum(0)
    for right in (-1, 0):
        out, lse = ops.flash_paged(q, k_pages, v_pages, table, lens, right=right, cu_seqlens_q=cu.cuda(), lse_layout=ops.LSE_BSH)
        assert ops.read_status() == 0
        owner = torch.repeat_interleave(torch.arange(streams, device="cuda"), new.cuda())
        i = torch.arange(T, device="cuda") - cu.cuda()[owner]
        x = lens[owner] - new.cuda()[owner] + i
        for a in range(0, T, 1 << 15):
            rows = slice(a, min(a + (1 << 15), T))
            k, v = (pages.float()[owner[rows] % 8] for pages in (k_pages, v_pages))                      # [rows, P, H, D]
            j = torch.arange(P, device="cuda")
            seen = (j < lens[owner[rows], None]) & (torch.ones_like(x[rows, None], dtype=torch.bool) if right < 0 else j <= x[rows, None])
            s = torch.einsum("thd,tphd->thp", q[rows].float(), k).masked_fill(~seen[:, None], float("-inf")) / 8
            top = torch.logsumexp(s, -1)
            w = torch.where(top[..., None] == float("-inf"), 0.0, (s - top[..., None]).exp())
            want, spread = torch.einsum("thp,tphd->thd", w, v), torch.einsum("thp,tphd->thd", w, v.abs())
            assert bool(((out[rows] - want).abs() <= (2.0 ** -8 + 3e-4) * spread + 1e-6).all())
            assert torch.equal(top == float("-inf"), lse[rows] == float("-inf"))
            assert bool(((lse[rows] - top).abs()[top > float("-inf")] <= 2e-4).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (50, 7, 20), (-1, -1, 0)])
@pytest.mark.parametrize("most", [1, 3, 40, 150, 300])
def test_of_sequences_longer_than_said_the_first_rows_are_as_they_were(most, left, right, sinks, D):
    from ditango_b200 import ops
    from tests.test_flash_window_gpu import _rand
    from tests.test_paged_gpu import _Cache
    new, lens = [400, 2, 170], [900, 60, 200]
    cache = _Cache(lens, 2, D, 16, seed=23)
    q = _rand((sum(new), 4, D), 72).cuda()
    cu = [0, 400, 402, 572]
    call = lambda **kw: ops.flash_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.seqlens, left=left, right=right, sinks=sinks, cu_seqlens_q=_i(cu),
                                        lse_layout=ops.LSE_BSH, **kw)
    whole, whole_lse = call()
    out, lse = torch.full_like(whole, 7.0), torch.full_like(whole_lse, 7.0)
    call(out=out, lse=lse, max_seqlen_q=most)
    assert ops.read_status() == 0
    for b, n in enumerate(new):
        kept = min(n, most)
        a, z = cu[b] + kept, cu[b + 1]
        assert bool((out[a:z] == 7).all()) and bool((lse[a:z] == 7).all())
        # (another kernel may have them: two results, each off by 2^-8 of its weights and 1e-4 for the scores)
        rows = slice(cu[b], a)
        assert bool((out[rows] - whole[rows]).abs().max() <= 2 * (2.0 ** -8 + 2e-4) * max(1.0, cache.v[b].abs().max().item()))
        same = (lse[rows] == whole_lse[rows]) | ((lse[rows] - whole_lse[rows]).abs() <= 2e-4)
        assert bool(same.all())


def test_tables_of_as_many_streams_as_there_can_be():
    import random

    from tests.test_paged_gpu import _Pages
    rng, P, streams = random.Random(5), 16, 16384
    pages = _Pages([rng.choice((0, 1, P, rng.randrange(3 * P))) for _ in range(streams)], P, 5, 3 * streams, seed=6)
    pages.extend([1] * streams, streams + 7)
    pages.extend([rng.choice((0, 0, 1, rng.randrange(P))) for _ in range(streams)], streams * P)
    pages.release([0] * streams, [rng.choice((0, P, n)) for n in pages.lens], True)
    pages.release([rng.choice((0, 5)) for _ in range(streams)], [10 ** 6] * streams, False)
    pages.extend([2] * streams, 2 * streams)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -20, 8.0])
@pytest.mark.parametrize("lens,n", [([700], 1), ([60000], 1), ([9000, 40, 3000], 9), ([5000], 300)])
def test_scales_from_the_smallest(lens, n, scale, accumulate):
    """Clusters, shares, tiles whose keys are split: with a scale of nearly 0 the mean of the values, and the logarithm of their number."""
    from ditango_b200 import ops
    from tests.test_flash_window_gpu import SCORE, _exact, _rand
    from tests.test_paged_gpu import _Cache
    cache = _Cache(lens, 2, 64, 16, seed=24)
    q = _rand((n * len(lens), 4, 64), 73)
    out, lse = (torch.zeros(q.shape, device="cuda"), torch.full(q.shape[:2], float("-inf"), device="cuda")) if accumulate else (None, None)
    out, lse = ops.flash_paged(q.cuda(), cache.k_pages, cache.v_pages, cache.table, cache.seqlens, cu_seqlens_q=_i([n * i for i in range(len(lens) + 1)]), max_seqlen_q=n,
                               softmax_scale=scale, lse_layout=ops.LSE_BSH, out=out, lse=lse, accumulate=accumulate)
    assert ops.read_status() == 0
    for b, total in enumerate(lens):
        rows = slice(n * b, n * (b + 1))
        want, top, spread = _exact(q[rows], cache.k[b], cache.v[b], torch.ones(n, total, dtype=torch.bool), scale)
        # scores are off by 2^-21 of |q||k|, which 8 makes 64 times what 1/8 makes of it: the weights by as much more than SCORE says
        score = SCORE * max(1.0, scale * 8)
        assert bool(((out[rows].cpu().double() - want).abs() <= (2.0 ** -8 + 2 * score) * spread + 1e-30).all())
        assert bool(((lse[rows].cpu().double() - top).abs() <= score).all())
