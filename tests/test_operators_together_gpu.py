"""Norm and positions, windowed attention chunk by chunk, states kept in 8 bits and merged, as the cached ring runs them, against 64 bits.

Tolerances, for one row.  Attention of a chunk: its weights are rounded to bf16 (2^-8 of sum p |v|), its scores off by SCORE; a merge is
a convex combination whose weights are off by SCORE at most twice, of states no larger than A, the row's largest value in any
state.  A state kept in 8 bits is off by half a step: A / 127 in int8 (the step is below 2 A / 127), 2^-4 A in e4m3; each is kept once,
and two of them once more, merged.  Against the inputs before norm and positions: q and k have been rounded to bf16, 2^-8 of each
value, which moves a score by d = 2.05 * 2^-8 * scale * sum |q k| at most, a weight by e^(2 d) - 1 of itself and lse by d."""
import math

import pytest
import torch

from tests.test_flash_window_gpu import SCORE, _exact as _attention, _visible
from tests.test_norm_rope_grid_gpu import _angles, _cuda, _exact as _positions, _inputs, _rope

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.int8: 1 / 127, torch.float8_e4m3fn: 2.0 ** -4}


def _run(q, k, v, norms, rope, text, window, cuts, code):
    from ditango_b200 import ops
    q, k = ops.norm_rope_grid(q, k, *norms, rope, text_len=text)
    states = []
    for a, b in zip(cuts, cuts[1:]):
        out, lse = ops.flash_window(q, k[:, a:b], v[:, a:b], left=window, right=window, sinks=text, q_start=0, k_start=a, lse_layout=ops.LSE_BSH)
        states.append((ops.quantize_rows(out, code), lse, ops.LSE_BSH))
    both, lse = ops.merge_states(states[:2], out_rows=code, fp32_out=False)
    out, lse = ops.merge_states([(both, lse, ops.LSE_BSH)] + states[2:])
    return q, k, out, lse


# B, text, grid, H, Hk, window, where the chunks begin: some rows see nothing of some of them
@pytest.mark.parametrize("B,text,grid,H,Hk,window,cuts", [(2, 7, (3, 4, 5), 4, 2, 20, [0, 7, 8, 50, 67]), (1, 40, (6, 12, 16), 24, 8, 300, [0, 298, 596, 894, 1192]),
                                                          (1, 0, (7, 9, 11), 3, 3, 0, [0, 100, 400, 693])])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_as_the_cached_ring_runs_them(B, text, grid, H, Hk, window, cuts, D, code):
    from ditango_b200 import ops
    tokens = math.prod(grid)
    S = text + tokens
    q, k, norms, g = _inputs(B, S, H, Hk, D, torch.bfloat16, True, S)
    v = torch.randn(B, S, Hk, D, generator=g).to(torch.bfloat16)
    rope = _rope(grid, D)
    args = q.cuda(), k.cuda(), v.cuda(), _cuda(norms), rope, text, window, cuts, code
    rq, rk, out, lse = (x.cpu() for x in _run(*args))
    assert ops.read_status() == 0
    ang = _angles(rope, tokens)
    eq, ek = (_positions(x.double(), w.double(), b.double(), e, ang, text, False) for x, (w, b, e) in zip((q, k), norms))
    seen = _visible(S, S, window, window, text, 0, 0)
    for b in range(B):
        # from q and k as the kernel gave them
        want, want_lse, spread = _attention(rq[b], rk[b], v[b], seen)
        top = torch.stack([_attention(rq[b], rk[b, x:y], v[b, x:y], seen[:, x:y])[0].abs().amax(-1) for x, y in zip(cuts, cuts[1:])]).amax(0)[..., None]
        most = (2.0 ** -8 + 2 * SCORE) * spread + (2 * HALF_STEP[code] * 1.02 + 4 * SCORE) * top
        assert ((out[b] - want).abs() <= most).all() and ((lse[b] - want_lse).abs() <= 2 * SCORE).all()
        # from the inputs
        want, want_lse, spread = _attention(eq[b], ek[b], v[b], seen)
        s = (eq[b].abs().transpose(0, 1) @ ek[b].repeat_interleave(H // Hk, 1).abs().permute(1, 2, 0)).masked_fill(~seen, 0.0).amax(-1).T
        d = (2.05 * 2.0 ** -8 * s / math.sqrt(D) + SCORE)[..., None]
        assert ((out[b] - want).abs() <= most * (2 * d).exp() + spread * (2 * d).expm1()).all()
        assert ((lse[b] - want_lse).abs() <= d[..., 0] + 2 * SCORE).all()


def test_captured_and_replayed_on_other_inputs():
    from ditango_b200 import ops
    text, grid, window, cuts = 40, (6, 12, 16), 300, [0, 298, 596, 894, 1192]
    q, k, norms, g = _inputs(1, 1192, 24, 8, 64, torch.bfloat16, True, 3)
    v = torch.randn(1, 1192, 8, 64, generator=g).to(torch.bfloat16)
    q, k, v, norms, rope = q.cuda(), k.cuda(), v.cuda(), _cuda(norms), _rope(grid, 64)
    args = (norms, rope, text, window, cuts, torch.int8)
    _run(q, k, v, *args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(q, k, v, *args)
    for _ in range(2):
        q.normal_(), k.normal_(), v.normal_()
        graph.replay()
        want = _run(q, k, v, *args)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert ops.read_status() == 0
