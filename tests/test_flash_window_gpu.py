"""Attention with a sliding window and first tokens that stay visible, against the definition in 64 bits.

Tolerances.  The weights are rounded to bf16 for the product with V (half a step is 2^-8 of a weight), the result once more if it is
bf16: 2^-8 sum_j p_j |v_j| (+ 2^-8 |out|).  A score is a sum of D products in fp32, off by at most D 2^-24 sum |q k| scale, which for
the normal inputs here stays below 1e-4; that is what lse may be off by, and what moves a weight by 1e-4 of itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCORE = 1e-4


def _rand(shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _visible(Sq, Sk, left, right, sinks, q_at, k_at):
    x, j = torch.arange(Sq)[:, None] + q_at, torch.arange(Sk)[None] + k_at
    seen = (j <= x + right) if right >= 0 else torch.ones(Sq, Sk, dtype=torch.bool)
    return seen & ((j >= x - left) | (j < sinks)) if left >= 0 else seen


def _exact(q, k, v, seen, scale=None):
    """One sequence: q [Sq,H,D], k, v [Sk,Hk,D], seen [Sq,Sk] -> (out, lse [Sq,H], sum p |v|) in 64 bits."""
    group = q.shape[1] // k.shape[1]
    q, k, v = (x.double().transpose(0, 1) for x in (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)))
    s = (q @ k.transpose(1, 2) * (scale or 1 / math.sqrt(q.shape[-1]))).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else s.new_full(s.shape[:-1], -math.inf)
    p = torch.where(lse[..., None] == -math.inf, torch.zeros_like(s), (s - lse[..., None]).exp())
    hidden = ~seen.any(0)
    v = v.masked_fill(hidden[None, :, None], 0.0)
    return (p @ v).transpose(0, 1), lse.transpose(0, 1), (p @ v.abs()).transpose(0, 1)


def _check(out, lse, want, want_lse, spread):
    """out, spread [Sq,H,D], lse [Sq,H]"""
    most = (2.0 ** -8 + 2 * SCORE) * spread + (2.0 ** -8 * want.abs() if out.dtype == torch.bfloat16 else 0) + 1e-30
    assert ((out.cpu().double() - want).abs() <= most).all()
    empty = want_lse == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty) and ((lse.cpu().double() - want_lse)[~empty].abs() <= SCORE).all()


def _run_and_check(q, k, v, *, left, right, sinks, q_start=None, k_start=0, lens=None, gpu=None, **kw):
    from ditango_b200 import ops
    B, Sq = q.shape[:2]
    gq, gk, gv = gpu or (q.cuda(), k.cuda(), v.cuda())
    sl = torch.tensor(lens, dtype=torch.int32).cuda() if lens is not None else None
    out, lse = ops.flash_window(gq, gk, gv, left=left, right=right, sinks=sinks, q_start=q_start, k_start=k_start, seqlens_k=sl,
                                lse_layout=ops.LSE_BSH, **kw)
    for b in range(B):
        n = lens[b] if lens is not None else k.shape[1]
        at = k_start + n - Sq if q_start is None else q_start
        _check(out[b], lse[b], *_exact(q[b], k[b, :n], v[b, :n], _visible(Sq, n, left, right, sinks, at, k_start)))
    assert ops.read_status() == 0
    return out, lse


# Sq, Sk, H, Hk: single tokens, tokens that share key heads, odd lengths around the tiles of 16, 128 and 256
SIZES = [(1, 1, 1, 1), (1, 700, 3, 3), (1, 1300, 8, 1), (3, 515, 8, 2), (5, 17, 4, 4), (16, 129, 2, 2), (100, 100, 6, 2), (127, 383, 2, 1),
         (128, 128, 1, 1), (255, 900, 2, 2), (257, 257, 3, 1), (300, 1111, 4, 2), (700, 700, 2, 2)]
WINDOWS = [(0, 0, 0), (0, 0, 5), (7, 0, 3), (63, 20, 0), (100, 100, 130), (128, 127, 128), (300, 0, 17), (-1, 0, 0), (-1, 50, 9), (40, -1, 300),
           (-1, -1, 0), (5000, 5000, 5000)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("Sq,Sk,H,Hk", SIZES)
def test_window_matches_the_definition(Sq, Sk, H, Hk, left, right, sinks, D):
    B = 2 if Sq * Sk < 10 ** 5 else 1
    q, k, v = _rand((B, Sq, H, D), Sq), _rand((B, Sk, Hk, D), Sk), _rand((B, Sk, Hk, D), Sk + 1)
    dtype = torch.bfloat16 if (Sq + left) % 2 else torch.float32
    _run_and_check(q, k, v, left=left, right=right, sinks=sinks, out_dtype=dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 9, 200, 600])
@pytest.mark.parametrize("q_start,k_start,left,right,sinks", [
    (0, 0, 50, 50, 10), (1000, 900, 50, 0, 950), (1000, 900, 50, 0, 20), (0, 400, 100, 100, 0), (0, 400, 100, 500, 405), (400, 0, 150, 0, 0),
    (-50, 0, 20, 10, 4), (2 ** 30 - 700, 2 ** 30 - 500, 300, 20, 0), (5000, 0, 10, 10, 3), (100, 0, 2 ** 30, 2 ** 30, 2 ** 30)])
def test_chunks_at_other_positions(Sq, q_start, k_start, left, right, sinks, D):
    """Keys of a chunk that starts elsewhere: windows that miss it in part or whole, first tokens in it, behind it, none."""
    q, k, v = _rand((1, Sq, 2, D), 1), _rand((1, 450, 2, D), 2), _rand((1, 450, 2, D), 3)
    _run_and_check(q, k, v, left=left, right=right, sinks=sinks, q_start=q_start, k_start=k_start)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 2, 33, 150, 400])
def test_caches_of_different_lengths_with_anything_behind_them(Sq, D):
    lens = [0, 1, Sq, 600, 477, 129]
    q, k, v = _rand((6, Sq, 4, D), 4), _rand((6, 600, 2, D), 5), _rand((6, 600, 2, D), 6)
    for b, n in enumerate(lens):
        k[b, n:], v[b, n:] = math.nan, math.inf
    _run_and_check(q, k, v, left=90, right=0, sinks=7, lens=lens)
    _run_and_check(q, k, v, left=90, right=40, sinks=0, lens=lens, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 11, 128, 300])
def test_keys_that_nobody_sees_may_hold_anything(Sq, D):
    """Between the first tokens and the windows, before the first window and behind the last one."""
    Sk, left, right, sinks, at = 1500, 130, 30, 21, 700
    q, k, v = _rand((1, Sq, 2, D), 7), _rand((1, Sk, 2, D), 8), _rand((1, Sk, 2, D), 9)
    seen = _visible(Sq, Sk, left, right, sinks, at, 0).any(0)
    k[:, ~seen], v[:, ~seen] = math.inf, math.nan
    _run_and_check(q, k, v, left=left, right=right, sinks=sinks, q_start=at)


@pytest.mark.parametrize("D", [64, 128])
def test_strides_of_fused_projections_and_sequence_first_tensors(D):
    B, S, H = 2, 333, 3
    x = _rand((B, S, 3, H, D), 10)
    gx = x.cuda()
    q, k, v = x.unbind(2)
    _run_and_check(q, k, v, left=60, right=10, sinks=4, gpu=gx.unbind(2))
    y = _rand((S, B, 3, H, D), 11)
    gy = y.cuda()
    _run_and_check(*(t.transpose(0, 1) for t in y.unbind(2)), left=60, right=10, sinks=4, gpu=tuple(t.transpose(0, 1) for t in gy.unbind(2)))
    # queries behind the text of a joint sequence, keys of the whole
    _run_and_check(q[:, 26:], k, v, left=60, right=60, sinks=26, gpu=(gx[:, 26:, 0], gx[:, :, 1], gx[:, :, 2]))


@pytest.mark.parametrize("D", [64, 128])
def test_packed_sequences_leave_the_rows_behind_them_alone(D):
    from ditango_b200 import ops
    qs, ks = [0, 300, 300, 301, 561], [0, 300, 340, 640, 640]       # one without queries, one with more keys, one without keys
    q, k, v = _rand((580, 4, D), 12), _rand((700, 2, D), 13), _rand((700, 2, D), 14)
    k[640:], v[640:] = math.nan, math.nan
    out = torch.full((580, 4, D), 7.0, device="cuda")
    lse = torch.full((580, 4), 7.0, device="cuda")
    ops.flash_window(q.cuda(), k.cuda(), v.cuda(), left=70, right=70, sinks=9, out=out, lse=lse, lse_layout=ops.LSE_BSH,
                     cu_seqlens_q=torch.tensor(qs, dtype=torch.int32).cuda(), cu_seqlens_k=torch.tensor(ks, dtype=torch.int32).cuda(),
                     max_seqlen_q=300, max_seqlen_k=300)
    assert (out[561:] == 7).all() and (lse[561:] == 7).all()
    for a, b, c, d in zip(qs, qs[1:], ks, ks[1:]):
        if b > a:
            seen = _visible(b - a, d - c, 70, 70, 9, (d - c) - (b - a), 0)
            _check(out[a:b], lse[a:b], *_exact(q[a:b], k[c:d], v[c:d], seen))
    assert ops.read_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 13, 260])
@pytest.mark.parametrize("layout", [0, 1])
def test_chunks_folded_into_a_state_are_the_whole(Sq, D, layout):
    """Five chunks of keys accumulated one after another, some of which some rows or none see.  Each adds its rounding of the weights."""
    from ditango_b200 import ops
    Sk, left, right, sinks, at = 1000, 250, 30, 40, 600
    q, k, v = _rand((2, Sq, 3, D), 15), _rand((2, Sk, 3, D), 16), _rand((2, Sk, 3, D), 17)
    gq, gk, gv = q.cuda(), k.cuda(), v.cuda()
    state, cuts = None, [0, 30, 300, 301, 700, 1000]
    for a, b in zip(cuts, cuts[1:]):
        kw = dict(left=left, right=right, sinks=sinks, q_start=at, k_start=a, lse_layout=layout)
        if state is None:
            state = ops.flash_window(gq, gk[:, a:b], gv[:, a:b], **kw)
        else:
            again = ops.flash_window(gq, gk[:, a:b], gv[:, a:b], out=state[0], lse=state[1], accumulate=True, **kw)
            assert again[0] is state[0] and again[1] is state[1]
    out, lse = state[0], state[1] if layout == 1 else state[1].transpose(1, 2)
    for b in range(2):
        _check(out[b], lse[b], *_exact(q[b], k[b], v[b], _visible(Sq, Sk, left, right, sinks, at, 0)))
    # a chunk that no row sees changes nothing
    before = state[0].clone(), state[1].clone()
    ops.flash_window(gq, gk, gv, left=5, right=5, q_start=10 ** 6, out=state[0], lse=state[1], accumulate=True, lse_layout=layout)
    assert torch.equal(state[0], before[0]) and torch.equal(state[1], before[1])


def test_states_merge_with_those_of_full_attention():
    """Text queries and keys by flash_partial, the video's window beside it: merge_states joins them."""
    from ditango_b200 import ops
    q, k, v = _rand((1, 300, 2, 64), 18), _rand((1, 700, 2, 64), 19), _rand((1, 700, 2, 64), 20)
    gq, gk, gv = q.cuda(), k.cuda(), v.cuda()
    a = ops.flash_partial(gq, gk[:, :100].contiguous(), gv[:, :100].contiguous(), lse_layout=ops.LSE_BSH)
    b = ops.flash_window(gq, gk[:, 100:], gv[:, 100:], left=120, right=0, q_start=400, k_start=100, lse_layout=ops.LSE_BSH)
    out, lse = ops.merge_states([(*a, ops.LSE_BSH), (*b, ops.LSE_BSH)])
    _check(out[0], lse[0], *_exact(q[0], k[0], v[0], _visible(300, 700, 120, 0, 100, 400, 0)))


@pytest.mark.parametrize("Sq", [1, 300])
def test_large_scores_and_a_maximum_that_keeps_growing(Sq):
    """Scores up to a few hundred, the largest in the last keys: the running maximum moves at every tile.  The scores are small whole
    multiples, so that they are exact in fp32."""
    D, Sk = 128, 900
    q = torch.zeros(1, Sq, 2, D)
    k = torch.zeros(1, Sk, 2, D)
    q[..., 0] = 16.0
    k[..., 0] = (torch.arange(Sk) // 4).float()[None, :, None]
    q, k, v = q.to(torch.bfloat16), k.to(torch.bfloat16), _rand((1, Sk, 2, D), 21)
    _run_and_check(q, k, v, left=400, right=0, sinks=5)


@pytest.mark.parametrize("Sq", [1, 40, 400])
def test_captured_replayed_and_beside_another_stream(Sq):
    from ditango_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(2, s, 4, 64, generator=g, device="cuda").to(torch.bfloat16) for s in (Sq, 800, 800))
    kw = dict(left=200, right=0, sinks=8, out_dtype=torch.bfloat16)
    lens = torch.tensor([800, 500], dtype=torch.int32, device="cuda")
    ops.flash_window(q, k, v, seqlens_k=lens, **kw)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.flash_window(q, k, v, seqlens_k=lens, **kw)
        graphs.append((graph, got))
    q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
    lens.copy_(torch.tensor([450, 777], dtype=torch.int32))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for (graph, _), s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    want = ops.flash_window(q, k, v, seqlens_k=lens, **kw)
    for _, got in graphs:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_cache_past_32_bit_offsets():
    from ditango_b200 import ops
    Sk = 2 ** 31 // (24 * 128) + 3000
    k = torch.zeros(1, Sk, 24, 128, dtype=torch.bfloat16, device="cuda")
    k[:, -2000:].normal_()
    q = torch.randn(1, 300, 24, 128, device="cuda").to(torch.bfloat16)
    tail = k[:, -2000:].contiguous()
    for rows in (1, 300):
        got = ops.flash_window(q[:, :rows], k, k, left=1000, right=0)
        want = ops.flash_window(q[:, :rows], tail, tail, left=1000, right=0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_nothing_to_do():
    from ditango_b200 import ops
    e = torch.empty(2, 0, 4, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(2, 5, 4, 64, device="cuda").to(torch.bfloat16)
    assert ops.flash_window(e, x, x)[0].shape == (2, 0, 4, 64)
    for q in (x, torch.randn(2, 300, 4, 64, device="cuda").to(torch.bfloat16)):
        out, lse = ops.flash_window(q, e, e)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_results_do_not_change_from_run_to_run():
    from ditango_b200 import ops
    for Sq in (1, 700):
        q, k, v = (x.cuda() for x in (_rand((1, Sq, 24, 128), 1), _rand((1, 3000, 24, 128), 2), _rand((1, 3000, 24, 128), 3)))
        a, al = ops.flash_window(q, k, v, left=2500, right=0, sinks=100)
        for _ in range(3):
            b, bl = ops.flash_window(q, k, v, left=2500, right=0, sinks=100)
            assert torch.equal(a, b) and torch.equal(al, bl)


def test_a_posted_status_keeps_results_from_being_written():
    from ditango_b200 import ops
    for Sq in (1, 300):
        q, k = _rand((1, Sq, 2, 64), 1).cuda(), _rand((1, 500, 2, 64), 2).cuda()
        out, lse = torch.full((1, Sq, 2, 64), 3.0, device="cuda"), torch.full((1, 2, Sq), 3.0, device="cuda")
        try:
            ops.post_status(77)
            ops.flash_window(q, k, k, left=100, right=0, out=out, lse=lse)
        finally:
            assert ops.read_status() == 77
        assert (out == 3).all() and (lse == 3).all()
        ops.flash_window(q, k, k, left=100, right=0, out=out, lse=lse)
        assert not (out == 3).any()


def _check_on_gpu(out, lse, q, k, v, b, *, left, right, sinks, at, heads, k_start=0):
    """Some heads of one sequence against 64 bits on the device."""
    group = q.shape[2] // k.shape[2]
    seen = _visible(q.shape[1], k.shape[1], left, right, sinks, at, k_start)
    for h in heads:
        want = _exact(*(x.double() for x in (q[b, :, h:h + 1], k[b, :, h // group:h // group + 1], v[b, :, h // group:h // group + 1])), seen.cuda())
        _check(out[b, :, h:h + 1], lse[b, :, h:h + 1], *(x.cpu() for x in want))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("accumulate", [False, True])
def test_many_blocks_of_rows_that_see_nothing(D, accumulate):
    """Sequences without a key, one after another, between those that have some: more of their blocks than a CTA has blocks under way."""
    from ditango_b200 import ops
    B, Sq, Sk, H = 9, 600, 700, 40
    q, k, v = (_rand((B, n, H, D), n + D).cuda() for n in (Sq, Sk, Sk))
    v[:] = v.flip(1)
    lens = [Sk, 0, 0, 0, 0, 0, 333, 0, 17]
    sl = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = ops.flash_window(q, k, v, left=150, right=90, sinks=70, q_start=0, seqlens_k=sl, lse_layout=ops.LSE_BSH)
    assert ops.read_status() == 0
    if accumulate:
        ops.flash_window(q, k, v, left=150, right=90, sinks=70, q_start=0, seqlens_k=sl, lse_layout=ops.LSE_BSH, out=out, lse=lse, accumulate=True)
        lse -= math.log(2.0)                    # the same state twice
    for b, n in enumerate(lens):
        if n:
            _check_on_gpu(out, lse, q, k[:, :n], v[:, :n], b, left=150, right=90, sinks=70, at=0, heads=(0, H - 1))
        else:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
    assert ops.read_status() == 0


# Launches large enough for the tiles of 128 rows, whole or with their keys split into parts (which takes scratch): B, Sq, Sk, H, Hk, window
LARGE = {"whole": (1, 700, 1500, 32, 8, dict(left=500, right=60, sinks=30)), "parts": (1, 200, 4500, 24, 6, dict(left=4000, right=0, sinks=70)),
         "two": (3, 300, 4500, 12, 12, dict(left=4100, right=130, sinks=140))}
large = pytest.mark.parametrize("kind,D", [(kind, D) for kind in LARGE for D in (64, 128)])


def _large(kind, D, seed=0):
    B, Sq, Sk, H, Hk, window = LARGE[kind]
    g = torch.Generator(device="cuda").manual_seed(seed + D)
    return *(torch.randn(B, n, h, D, generator=g, device="cuda").to(torch.bfloat16) for n, h in ((Sq, H), (Sk, Hk), (Sk, Hk))), window


def _heads(q):
    return 0, 5, q.shape[2] - 1


@large
def test_only_launches_that_leave_sms_idle_are_split(kind, D):
    from ditango_b200 import _capi
    B, Sq, Sk, H, Hk, w = LARGE[kind]
    lib = _capi.load()
    size = lib.dtb_flash_window_scratch_bytes(B, Sq, Sk, H, Hk, D, w["left"], w["right"], w["sinks"])
    state = B * Sq * H * (D + 1) * 4
    assert size % state == 0 and (size >= 2 * state) == (kind != "whole")
    assert lib.dtb_flash_window_scratch_bytes(B, 16, Sk, H, Hk, D, w["left"], w["right"], w["sinks"]) == 0


@large
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, -77, 9000])
def test_large_launches_match_the_definition(kind, D, dtype, shift):
    """At the end of their keys, a little before it, and far behind it, where only the first tokens are seen."""
    from ditango_b200 import ops
    q, k, v, w = _large(kind, D)
    at = k.shape[1] - q.shape[1] + shift
    out, lse = ops.flash_window(q, k, v, **w, q_start=at, out_dtype=dtype, lse_layout=ops.LSE_BSH)
    out2, lse2 = ops.flash_window(q, k, v, **w, q_start=at, out_dtype=dtype)
    assert torch.equal(out, out2) and torch.equal(lse, lse2.transpose(1, 2))
    for b in range(q.shape[0]):
        _check_on_gpu(out, lse, q, k, v, b, **w, at=at, heads=_heads(q))
    assert ops.read_status() == 0


@large
def test_large_launches_of_different_lengths(kind, D):
    from ditango_b200 import ops
    q, k, v, w = _large(kind, D)
    lens = [1, 999, 0] if len(q) == 3 else [999]
    for b, n in enumerate(lens):
        k[b, n:], v[b, n:] = math.nan, math.inf
    out, lse = ops.flash_window(q, k, v, **w, seqlens_k=torch.tensor(lens, dtype=torch.int32).cuda(), lse_layout=ops.LSE_BSH)
    for b, n in enumerate(lens):
        _check_on_gpu(out, lse, q, k[:, :n], v[:, :n], b, **w, at=n - q.shape[1], heads=_heads(q))
    assert ops.read_status() == 0


@large
def test_keys_that_no_large_launch_sees_may_hold_anything(kind, D):
    from ditango_b200 import ops
    q, k, v, w = _large(kind, D)
    w = dict(w, left=w["left"] // 2)
    at = 2 * k.shape[1] // 3 - q.shape[1]
    seen = _visible(q.shape[1], k.shape[1], *w.values(), at, 0).any(0).cuda()
    assert not seen.all()
    k[:, ~seen], v[:, ~seen] = math.inf, math.nan
    out, lse = ops.flash_window(q, k, v, **w, q_start=at, lse_layout=ops.LSE_BSH)
    k[:, ~seen], v[:, ~seen] = 0, 0
    _check_on_gpu(out, lse, q, k, v, 0, **w, at=at, heads=_heads(q))


@large
@pytest.mark.parametrize("layout", [0, 1])
def test_large_chunks_folded_into_a_state_are_the_whole(kind, D, layout):
    from ditango_b200 import ops
    q, k, v, w = _large(kind, D)
    at, cut = k.shape[1] - q.shape[1], k.shape[1] // 2 + 13
    out, lse = ops.flash_window(q, k[:, :cut], v[:, :cut], **w, q_start=at, lse_layout=layout)
    again = ops.flash_window(q, k[:, cut:], v[:, cut:], **w, q_start=at, k_start=cut, out=out, lse=lse, accumulate=True, lse_layout=layout)
    assert again[0] is out and again[1] is lse
    _check_on_gpu(out, lse if layout else lse.transpose(1, 2), q, k, v, 0, **w, at=at, heads=_heads(q))
    before = out.clone(), lse.clone()
    ops.flash_window(q, k, v, left=w["left"], right=w["right"], q_start=10 ** 6, out=out, lse=lse, accumulate=True, lse_layout=layout)
    assert torch.equal(out, before[0]) and torch.equal(lse, before[1])
    assert ops.read_status() == 0


@large
def test_large_launches_on_views_of_one_projection(kind, D):
    """Queries and keys as slices of a tensor with other things beside them, batch or sequence first."""
    from ditango_b200 import ops
    q, k, v, w = _large(kind, D)
    H, Hk, S = q.shape[2], k.shape[2], k.shape[1]
    for first in (True, False):
        x = torch.full((q.shape[0], S, H + 2 * Hk + 1, D) if first else (S, q.shape[0], H + 2 * Hk + 1, D), math.nan, dtype=torch.bfloat16, device="cuda")
        y = x if first else x.transpose(0, 1)
        views = y[:, S - q.shape[1]:, :H], y[:, :, H:H + Hk], y[:, :, H + Hk:H + 2 * Hk]
        for to, of in zip(views, (q, k, v)):
            to.copy_(of)
        want, got = ops.flash_window(q, k, v, **w), ops.flash_window(*views, **w)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@large
def test_large_launches_captured_twice_beside_others(kind, D):
    """Graphs replayed at once on two streams have scratch of their own, and a launch between them too."""
    from ditango_b200 import ops
    (q, k, v, w), (q2, _, _, _) = _large(kind, D), _large(kind, D, seed=1)
    queries = q.clone(), q2.clone()
    want = [ops.flash_window(x, k, v, **w) for x in queries]
    graphs = []
    for x in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.flash_window(x, k, v, **w), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        between = ops.flash_window(q, k, v, **w)
    torch.cuda.synchronize()
    assert torch.equal(between[0], want[0][0])
    for (_, got, _), x in zip(graphs, want):
        assert torch.equal(got[0], x[0]) and torch.equal(got[1], x[1])


@large
def test_large_launches_after_a_failure_write_nothing(kind, D):
    from ditango_b200 import ops
    q, k, v, w = _large(kind, D)
    out, lse = torch.full(q.shape, 3.0, device="cuda"), torch.full((q.shape[0], q.shape[2], q.shape[1]), 3.0, device="cuda")
    try:
        ops.post_status(77)
        ops.flash_window(q, k, v, **w, out=out, lse=lse)
    finally:
        assert ops.read_status() == 77
    assert (out == 3).all() and (lse == 3).all()


@pytest.mark.parametrize("D", [64, 128])
def test_large_packed_sequences(D):
    from ditango_b200 import ops
    q, k, v, w = _large("whole", D)
    q, k, v = q[0], k[0], v[0]
    qs, ks = [0, 300, 300, 301, 561, 690], [0, 300, 340, 640, 640, 1400]
    k[1400:], v[1400:] = math.nan, math.nan
    out, lse = torch.full(q.shape, 7.0, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")
    ops.flash_window(q, k, v, **w, out=out, lse=lse, lse_layout=ops.LSE_BSH, cu_seqlens_q=torch.tensor(qs, dtype=torch.int32).cuda(),
                     cu_seqlens_k=torch.tensor(ks, dtype=torch.int32).cuda())
    assert (out[690:] == 7).all() and (lse[690:] == 7).all()
    for a, b, c, d in zip(qs, qs[1:], ks, ks[1:]):
        if b > a:
            _check_on_gpu(*(x[None] for x in (out[a:b], lse[a:b], q[a:b], k[c:d], v[c:d])), 0, **w, at=(d - c) - (b - a), heads=_heads(q[None]))
    assert ops.read_status() == 0


def test_scratch_that_is_too_small_is_refused():
    from ditango_b200 import _capi
    q, k, v, w = _large("parts", 64)
    (B, Sq, Sk, H, Hk, _), lib = LARGE["parts"], _capi.load()
    out, lse, scratch = torch.full(q.shape, 3.0, device="cuda"), torch.full((B, H, Sq), 3.0, device="cuda"), torch.empty(1024, dtype=torch.uint8, device="cuda")
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), H * 64, 0, Hk * 64, 0, Hk * 64, 0, out.data_ptr(), 0, lse.data_ptr(), 0, 0, None, None, None, B, Sq, Sk,
            Sq, Sk, H, Hk, 64, 0.125, w["left"], w["right"], w["sinks"], _capi.QUERIES_LAST, 0)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.dtb_flash_window(*args, scratch.data_ptr(), 1024, stream) == -1 and "scratch" in lib.dtb_last_error().decode()
    torch.cuda.synchronize()
    assert (out == 3).all() and (lse == 3).all()
    assert lib.dtb_flash_window(*args, None, 0, stream) == 0            # without scratch the keys stay whole
    _check_on_gpu(out, lse.transpose(1, 2), q, k, v, 0, **w, at=Sk - Sq, heads=_heads(q))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["few", *LARGE])
def test_a_nan_among_the_scores_shows(kind, D):
    """In the rows that see it, and as lse too, and when the state is folded into another; other rows are what they were."""
    from ditango_b200 import ops
    q, k, v, w = _large("parts" if kind == "few" else kind, D)
    if kind == "few":
        q = q[:, :9]
    Sq, Sk = q.shape[1], k.shape[1]
    w = dict(w, left=w["left"] // 2 if kind != "whole" else 100, sinks=0)
    want = ops.flash_window(q, k, v, **w, lse_layout=ops.LSE_BSH)
    j = Sk - Sq - w["left"] + Sq // 2                   # seen by the rows in front of the middle
    k[0, j, 0] = math.nan
    seen = _visible(Sq, Sk, *w.values(), Sk - Sq, 0)[:, j].cuda()
    assert seen.any() and not seen.all()
    group = q.shape[2] // k.shape[2]
    for state in (None, tuple(x.clone() for x in want)):
        kw = {} if state is None else dict(out=state[0], lse=state[1], accumulate=True)
        out, lse = ops.flash_window(q, k, v, **w, lse_layout=ops.LSE_BSH, **kw)
        assert out[0, seen, :group].isnan().all() and lse[0, seen, :group].isnan().all()
        assert not out[0, ~seen].isnan().any() and not out[:, :, group:].isnan().any() and not lse[0, ~seen].isnan().any()
        if state is None:
            assert torch.equal(out[0, ~seen], want[0][0, ~seen]) and torch.equal(lse[:, :, group:], want[1][:, :, group:])
    assert ops.read_status() == 0


@pytest.mark.parametrize("kw", [dict(left=2 ** 32), dict(right=-2 ** 32 - 1), dict(sinks=2 ** 32 + 1), dict(q_start=2 ** 32), dict(k_start=-2 ** 33)])
def test_numbers_that_an_int_does_not_hold_are_refused(kw):
    from ditango_b200 import _capi, ops
    x = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_capi.ExtensionError):
        ops.flash_window(x, x, x, **kw)


@pytest.mark.parametrize("Sq,H", [(1, 2), (40, 2), (300, 24)])
@pytest.mark.parametrize("left,right,sinks,q_start,k_start", [
    (-1, 0, 0, 2 ** 30, 0), (-1, 5, 0, 2 ** 30, -2 ** 30), (-1, -1, 0, 2 ** 30, -2 ** 30), (-1, -1, 0, -2 ** 30, 2 ** 30), (40, -1, 0, -2 ** 30, 0),
    (40, -1, 0, 2 ** 30, -2 ** 30), (2 ** 30, 2 ** 30, 0, 2 ** 30, -2 ** 30)])
def test_no_limit_is_none_at_any_position(Sq, H, left, right, sinks, q_start, k_start):
    """At the ends of the positions that are accepted, where a limit of 2^30 does hide keys."""
    q, k, v = _rand((1, Sq, H, 64), 1), _rand((1, 450, H, 64), 2), _rand((1, 450, H, 64), 3)
    _run_and_check(q, k, v, left=left, right=right, sinks=sinks, q_start=q_start, k_start=k_start)
