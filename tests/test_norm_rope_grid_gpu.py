"""Norm and rotary positions on three axes, forward and backward, against the same steps in 64 bits.

Tolerances: the arithmetic is fp32, some twenty roundings of 2^-24 and a reciprocal root of 2^-22 relative to a row's largest value:
2^-18 of it.  A bf16 result adds half a step, 2^-8 of itself.  The sums for weights and biases are sums of fp32 terms in three stages of
at most a few hundred additions each: 1000 * 2^-24 of the sum of the terms' magnitudes."""
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

ROW = 2.0 ** -18
SUM = 1000 * 2.0 ** -24


def _angles(rope, tokens):
    """[tokens, D / 2] in 64 bits; NaN at padding."""
    t, h, w = rope.grid
    places, out = t * h * w, torch.full((tokens, sum(rope.axes) // 2), math.nan, dtype=torch.float64)
    size, rest = divmod(places, rope.shards)
    length = size + (rest > 0)
    for i in range(tokens):
        shard, at = divmod(rope.first + i, length) if length else (rope.shards, 0)
        if shard >= rope.shards or at >= size + (shard < rest):
            continue
        n = shard * size + min(shard, rest) + at
        pos = (n // (h * w), n // w % h, n % w)
        out[i] = torch.cat([(o + s * x) * rope.base ** (-torch.arange(0, d, 2, dtype=torch.float64) / max(d, 1))
                            for x, d, o, s in zip(pos, rope.axes, rope.origin, rope.step)])
    return out


def _exact(x, w, b, eps, ang, text_len, rms):
    """x, w, b in 64 bits."""
    xc = x if rms else x - x.mean(-1, keepdim=True)
    y = xc * torch.rsqrt(xc.square().mean(-1, keepdim=True) + eps) * w + (0 if b is None else b)
    n = ang.shape[0]
    front, video, behind = y.split([text_len, n, y.shape[1] - text_len - n], dim=1)
    pad = ang.isnan().any(-1)
    ang = ang.masked_fill(pad[:, None], 0.0)[None, :, None]
    re, im = video[..., 0::2], video[..., 1::2]
    video = torch.stack([re * ang.cos() - im * ang.sin(), im * ang.cos() + re * ang.sin()], dim=-1).flatten(-2)
    return torch.cat([front, video.masked_fill(pad[None, :, None, None], 0.0), behind], dim=1)


def _inputs(B, S, H, Hk, D, dtype, bias, seed):
    g = torch.Generator().manual_seed(seed)
    q, k = ((torch.randn(B, S, h, D, generator=g) * 2 + 0.5).to(dtype) for h in (H, Hk))
    norms = [((1 + 0.3 * torch.randn(D, generator=g)).to(dtype), torch.randn(D, generator=g).to(dtype) if bias else None, e) for e in (1e-6, 1e-3)]
    return q, k, norms, g


def _cuda(norms):
    return [(w.cuda(), None if b is None else b.cuda(), e) for w, b, e in norms]


def _rope(grid, D, **kw):
    from ditango_b200 import ops
    axes = {64: (16, 24, 24), 128: (44, 42, 42)}[D]
    return ops.GridRope(grid, axes, **kw)


# B, text, grid, tokens behind the text, tokens behind the video, H, Hk
CASES = [(1, 0, (1, 1, 1), 1, 0, 1, 1), (2, 5, (2, 3, 4), 24, 0, 3, 3), (1, 0, (3, 4, 5), 70, 0, 48, 48), (2, 7, (3, 5, 7), 105, 9, 24, 8),
         (1, 33, (1, 2, 2), 0, 0, 7, 1), (3, 1, (4, 6, 9), 211, 2, 2, 5), (1, 0, (0, 5, 5), 3, 0, 4, 4), (1, 226, (5, 17, 23), 1955, 0, 50, 50)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rms,bias", [(False, True), (True, False), (False, False), (True, True)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,text,grid,video,behind,H,Hk", CASES)
def test_forward_and_backward_match_exact(B, text, grid, video, behind, H, Hk, D, rms, bias, dtype):
    from ditango_b200 import ops
    S = text + video + behind
    q, k, norms, g = _inputs(B, S, H, Hk, D, dtype, bias, S)
    rope = _rope(grid, D, first=2 if video > 100 else 0, origin=(0.0, -3.5, 100.0), step=(1.0, 0.5, 1.0))
    ang = _angles(rope, video)
    kw = dict(text_len=text, video_len=video, rms=rms)
    outs = ops.norm_rope_grid(q.cuda(), k.cuda(), *_cuda(norms), rope, **kw)
    dz = [torch.randn(x.shape, generator=g).to(dtype) for x in (q, k)]
    grads = ops.norm_rope_grid_backward(dz[0].cuda(), dz[1].cuda(), q.cuda(), k.cuda(), *_cuda(norms), rope, **kw)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    for i, (x, (w, b, eps)) in enumerate(zip((q, k), norms)):
        leaves = [t.double().requires_grad_() for t in ((x, w) if b is None else (x, w, b))]
        want = _exact(*leaves[:2], leaves[2] if bias else None, eps, ang, text, rms)
        assert outs[i].dtype == dtype and outs[i].is_contiguous()
        most = half * want.abs() + ROW * 4 * want.abs().amax(-1, keepdim=True)
        assert ((outs[i].cpu().double() - want).abs() <= most).all()
        got = torch.autograd.grad(want, leaves, dz[i].double())
        mine = [grads[i], grads[2 + 2 * i]] + ([grads[3 + 2 * i]] if bias else [])
        assert bias or grads[3 + 2 * i] is None
        row = got[0].abs().amax(-1, keepdim=True) + 1e-12
        # (a small row's rstd multiplies what cancels in g - mean - x^ mean: the largest |rstd g| of the row counts)
        xc = x.double() if rms else x.double() - x.double().mean(-1, keepdim=True)
        scale = torch.rsqrt(xc.square().mean(-1, keepdim=True) + eps) * dz[i].double().abs().amax(-1, keepdim=True) * w.double().abs().max() * 4
        assert ((mine[0].cpu().double() - got[0]).abs() <= half * got[0].abs() + ROW * torch.maximum(row, scale)).all()
        terms = dz[i].double().abs().amax(-1, keepdim=True) * 1.5
        bounds = [(terms * (xc * torch.rsqrt(xc.square().mean(-1, keepdim=True) + eps)).abs()).sum((0, 1, 2)), terms.expand_as(x).sum((0, 1, 2))]
        for a, e, bound in zip(mine[1:], got[1:], bounds):
            assert a.dtype == dtype and ((a.cpu().double() - e).abs() <= half * e.abs() + (SUM + 2 * ROW) * bound + 1e-30).all()


def test_gradients_against_differences():
    """Central differences of the 64-bit definition along random directions."""
    from ditango_b200 import ops
    q, k, norms, g = _inputs(1, 20, 2, 2, 64, torch.float32, True, 3)
    rope = _rope((2, 3, 3), 64)
    ang = _angles(rope, 18)
    dz = torch.randn(q.shape, generator=g)
    grads = ops.norm_rope_grid_backward(dz.cuda(), dz.cuda(), q.cuda(), k.cuda(), *_cuda(norms), rope, text_len=2)
    (w, b, eps), h = norms[0], 1e-5
    for leaf, grad in zip((q, w, b), (grads[0], grads[2], grads[3])):
        d = torch.randn(leaf.shape, generator=g).double()

        def f(s):
            args = [t.double() + s * d if t is leaf else t.double() for t in (q, w, b)]
            return (_exact(*args, eps, ang, 2, False) * dz.double()).sum()
        slope = float((f(h) - f(-h)) / (2 * h))
        assert abs(slope - float((grad.cpu().double() * d).sum())) <= 1e-4 * float((grad.cpu().double() * d).abs().sum())


def test_far_positions_keep_their_angles():
    """Positions of a few million, where an angle in fp32 would be off by a tenth of a turn and more."""
    from ditango_b200 import ops
    q, k, norms, _ = _inputs(1, 60, 2, 2, 64, torch.float32, True, 4)
    rope = _rope((3, 4, 5), 64, origin=(3.0e6, 5.5e6, 1.0e7), step=(1.0, 1000.0, 7.0))
    outs = ops.norm_rope_grid(q.cuda(), k.cuda(), *_cuda(norms), rope)
    want = _exact(q.double(), norms[0][0].double(), norms[0][1].double(), norms[0][2], _angles(rope, 60), 0, False)
    # the angle's product and reduction in 64 bits: 1e7 * 2^-52 of a radian
    assert ((outs[0].cpu().double() - want).abs() <= 4 * ROW * want.abs().amax(-1, keepdim=True)).all()


def test_strides_of_a_fused_projection():
    from ditango_b200 import ops
    B, S, H, D = 2, 31, 3, 128
    x = torch.randn(B, S, 3, H, D, device="cuda").to(torch.bfloat16)
    y = torch.randn(S, B, 2, H, D, device="cuda").to(torch.bfloat16)
    norms = _cuda(_inputs(1, 1, 1, 1, D, torch.bfloat16, True, 5)[2])
    rope = _rope((2, 3, 5), D)
    q, k = x[:, :, 0], x[:, :, 1]
    dq, dk = y[:, :, 0].transpose(0, 1), y[:, :, 1].transpose(0, 1)
    c = lambda t: t.contiguous()
    for a, b in zip(ops.norm_rope_grid(q, k, *norms, rope, text_len=1), ops.norm_rope_grid(c(q), c(k), *norms, rope, text_len=1)):
        assert torch.equal(a, b)
    for a, b in zip(ops.norm_rope_grid_backward(dq, dk, q, k, *norms, rope, text_len=1),
                    ops.norm_rope_grid_backward(c(dq), c(dk), c(q), c(k), *norms, rope, text_len=1)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("world,grid", [(4, (3, 5, 7)), (3, (2, 2, 2)), (8, (1, 2, 3))])
def test_shards_and_their_padding_are_those_of_the_tables(world, grid):
    """Each rank's piece, and all pieces one after another, get the rows that split tables give them; what padding holds does not matter."""
    from ditango_b200 import ops
    from ditango_b200.executor.cogvideox_dit import grid_tables
    from ditango_b200.utils import split_tensor_uneven
    n = grid[0] * grid[1] * grid[2]
    rope = _rope(grid, 64, shards=world)
    whole = [split_tensor_uneven(x, world, dim=0) for x in grid_tables(rope._replace(shards=1), n, "cpu")]
    length = whole[0][0].shape[0]
    q, k, norms, _ = _inputs(1, world * length + 2, 3, 3, 64, torch.float32, True, 6)
    ang = _angles(rope, world * length)
    real = ~ang.isnan().any(-1)
    assert int(real.sum()) == n
    q[:, 2:][:, ~real] = math.nan
    full = ops.norm_rope_grid(q.cuda(), k.cuda(), *_cuda(norms), rope, text_len=2)
    assert (full[0][:, 2:].cpu()[:, ~real] == 0).all() and full[0].isfinite().all()
    dz = torch.ones_like(q)
    grads = ops.norm_rope_grid_backward(dz.cuda(), dz.cuda(), q.cuda(), k.cuda(), *_cuda(norms), rope, text_len=2)
    assert (grads[0][:, 2:].cpu()[:, ~real] == 0).all() and all(g.isfinite().all() for g in grads)
    for r in range(world):
        cut = slice(2 + r * length, 2 + (r + 1) * length)
        piece = ops.norm_rope_grid(q[:, cut].cuda(), k[:, cut].cuda(), *_cuda(norms), rope._replace(first=r * length))
        assert torch.equal(piece[0], full[0][:, cut]) and torch.equal(piece[1], full[1][:, cut])
        cos, sin = grid_tables(rope._replace(first=r * length), length, "cpu")
        assert torch.equal(cos, whole[0][r]) and torch.equal(sin, whole[1][r])


def test_autograd_of_the_block_step_and_its_general_path():
    """The kernels' gradients against those of the separate operations on tables, through modules; a hook keeps the separate ones."""
    from ditango_b200 import ops
    from ditango_b200.executor.cogvideox_dit import norm_and_rotate_grid
    torch.manual_seed(0)
    rope = _rope((2, 3, 4), 64)
    x = torch.randn(2, 30, 3, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    k = torch.randn(2, 30, 3, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    nq, nk = (nn.LayerNorm(64, eps=1e-6).cuda().to(torch.bfloat16) for _ in range(2))
    nq.weight.data.normal_()
    leaves = [x, k, *nq.parameters(), *nk.parameters()]
    dz = [torch.randn(2, 30, 3, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]

    def run():
        n0 = ops.LaunchLog.count
        outs = norm_and_rotate_grid(x, k, nq, nk, rope, 4, 24)
        return outs, torch.autograd.grad(outs, leaves, dz), ops.LaunchLog.count - n0
    outs, grads, launches = run()
    nq.register_forward_hook(lambda m, i, o: None)
    want, want_grads, general = run()
    assert (launches, general) == (3, 0)
    for a, b in zip((*outs, *grads), (*want, *want_grads)):          # the separate operations round to bf16 at every step
        assert a.shape == b.shape and (a.float() - b.float()).abs().max() <= 2.0 ** -5 * b.float().abs().max()
    nq._forward_hooks.clear()
    # one tensor as q and as k gets both shares; an expanded gradient is taken
    one = norm_and_rotate_grid(x, x, nq, nk, rope, 4, 24)
    (g,) = torch.autograd.grad(sum(o.float().sum() for o in one), x)
    parts = [torch.autograd.grad(norm_and_rotate_grid(x, x.detach(), nq, nk, rope, 4, 24)[0].float().sum(), x)[0],
             torch.autograd.grad(norm_and_rotate_grid(x.detach(), x, nq, nk, rope, 4, 24)[1].float().sum(), x)[0]]
    assert (g.float() - (parts[0].float() + parts[1].float())).abs().max() <= 2.0 ** -7 * g.float().abs().max()


def test_captured_and_repeated():
    from ditango_b200 import ops
    q, k, norms, g = _inputs(2, 400, 24, 24, 128, torch.bfloat16, True, 8)
    rope, norms = _rope((4, 10, 10), 128), _cuda(norms)
    q, k = q.cuda(), k.cuda()
    ops.norm_rope_grid_backward(q, k, q, k, *norms, rope)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = (*ops.norm_rope_grid(q, k, *norms, rope), *ops.norm_rope_grid_backward(q, k, q, k, *norms, rope))
    q.normal_()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        want = (*ops.norm_rope_grid(q, k, *norms, rope), *ops.norm_rope_grid_backward(q, k, q, k, *norms, rope))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_backward_through_autograd():
    from ditango_b200.executor.cogvideox_dit import norm_and_rotate_grid
    torch.manual_seed(1)
    rope = _rope((2, 3, 4), 64)
    nq, nk = (nn.LayerNorm(64, eps=1e-6).cuda().to(torch.bfloat16) for _ in range(2))
    x = torch.randn(1, 24, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    leaves = [x, *nq.parameters()]

    def step():
        out = norm_and_rotate_grid(x, x, nq, nk, rope, 0)
        return torch.autograd.grad(out[0].float().square().sum(), leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.normal_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_empty_tensors():
    from ditango_b200 import ops
    _, _, norms, _ = _inputs(1, 1, 1, 1, 64, torch.bfloat16, True, 1)
    norms = _cuda(norms)
    for shape in ((0, 9, 4, 64), (2, 0, 4, 64)):
        e = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        assert all(x.shape == shape for x in ops.norm_rope_grid(e, e, *norms, _rope((1, 3, 3), 64)))
        grads = ops.norm_rope_grid_backward(e, e, e, e, *norms, _rope((1, 3, 3), 64))
        assert grads[0].shape == shape and all((x == 0).all() for x in grads[2:])


# ------------------------------------------------------------------------------------------------ in the transformer
def _model(mode, group, **kw):
    from ditango_b200.core import redundancy_map as rmod
    from ditango_b200.core.config import init_config
    from ditango_b200.executor.cogvideox_dit import CogVideoXDiT, DiTConfig
    cfg = init_config(None, make_output_dir=False)
    cfg.num_layers, cfg.num_inference_steps = 2, 2
    rmod.destroy_redundancy_map()
    rmod.init_redundancy_map(cfg, world_size=group.world_size)
    torch.manual_seed(3)
    return CogVideoXDiT(DiTConfig(num_layers=2, num_heads=4, head_dim=64, text_dim=32, time_dim=64, frames=3, height=10, width=14, text_len=9, **kw),
                        group, mode).cuda().to(torch.bfloat16)


def _latents():
    g = torch.Generator().manual_seed(4)
    return (torch.randn(2, 3, 16, 10, 14, generator=g).to(torch.bfloat16).cuda(), torch.randn(2, 9, 32, generator=g).to(torch.bfloat16).cuda(),
            torch.tensor([500.0, 500.0]).cuda())


@pytest.mark.parametrize("mode", ["ring", "ulysses"])
def test_the_transformer_on_grid_positions_is_that_on_tables(mode):
    """The tables round their angles to fp32 and the rest is the same kernel arithmetic: results agree to bf16 roundings."""
    from ditango_b200 import ops
    from ditango_b200.core.group_coordinate import SingleRankGroup
    from ditango_b200.utils import update_timestep
    update_timestep(0)
    group = SingleRankGroup(torch.device("cuda", 0))
    with torch.no_grad():
        a, b = (_model(mode, group, rotary=r)(*_latents()) for r in ("tables", "grid"))
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * a.float().abs().max()
    assert ops.read_status() == 0


@pytest.mark.parametrize("mode", ["ring", "ulysses"])
@pytest.mark.parametrize("world", [2, 4])
def test_grid_positions_on_logical_ranks(mode, world):
    """105 places over 2 and 4 ranks, so that the last pieces are padded: the same as with split tables."""
    from tests import loopback as LB
    got = []
    for rotary in ("tables", "grid"):
        def body(r, group, fabric):
            LB.stepped(fabric, r, 0)
            with torch.no_grad():
                return group.context(*_latents())
        got.append(LB.run_ranks(world, body, prepare=lambda r, group: _model(mode, group, rotary=rotary)))
    for a, b in zip(*got):
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * a.float().abs().max()


def test_the_transformer_with_local_attention():
    """One frame's worth of positions either way: the block's attention against masked attention in 64 bits; a window over everything is
    full attention; other modes refuse it."""
    from ditango_b200.core.group_coordinate import SingleRankGroup
    from ditango_b200.utils import update_timestep
    update_timestep(0)
    group = SingleRankGroup(torch.device("cuda", 0))
    model = _model("ulysses", group, rotary="grid", window_frames=1)
    g = torch.Generator().manual_seed(5)
    S = 9 + 3 * 35
    q, k, v = (torch.randn(2, S, 4, 64, generator=g).to(torch.bfloat16) for _ in range(3))
    out = model.blocks[0]._attend_whole(q.cuda(), k.cuda(), v.cuda(), 9).cpu().double()
    x = torch.arange(S)
    seen = (x[:, None] < 9) | (x[None] < 9) | ((x[:, None] - x[None]).abs() <= 35)
    s = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) / 8
    p = s.masked_fill(~seen, -math.inf).softmax(-1)
    want = torch.einsum("bhij,bjhd->bihd", p, v.double())
    spread = torch.einsum("bhij,bjhd->bihd", p, v.double().abs())
    assert ((out - want).abs() <= (2.0 ** -8 + 2e-4) * spread + 2.0 ** -8 * want.abs()).all()
    with torch.no_grad():
        wide, full = (_model("ulysses", group, rotary="grid", window_frames=w)(*_latents()) for w in (3, None))
    assert (wide.float() - full.float()).abs().max() <= 2.0 ** -5 * full.float().abs().max()
    with pytest.raises(ValueError):
        _model("ring", group, window_frames=1)
    with pytest.raises(ValueError):
        _model("ulysses", group, rotary="learned")


def test_ulysses_attention_with_a_window():
    from ditango_b200.baseline.ulysses import ulysses_attention
    from tests import loopback as LB
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(1, 200, 4, 64, generator=g).to(torch.bfloat16) for _ in range(3))

    def body(r, group, fabric):
        return ulysses_attention(*(x[:, r * 100:(r + 1) * 100].contiguous().cuda() for x in (q, k, v)), group=group, left=20, right=5, sinks=3).cpu()
    out = torch.cat(LB.run_ranks(2, body), dim=1).double()
    x = torch.arange(200)
    seen = (x[None] <= x[:, None] + 5) & ((x[None] >= x[:, None] - 20) | (x[None] < 3))
    p = (torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) / 8).masked_fill(~seen, -math.inf).softmax(-1)
    want, spread = (torch.einsum("bhij,bjhd->bihd", p, t) for t in (v.double(), v.double().abs()))
    assert ((out - want).abs() <= (2.0 ** -8 + 2e-4) * spread + 2.0 ** -8 * want.abs()).all()


@pytest.mark.parametrize("rope,kw", [(dict(grid=(1, 2, 2 ** 32 + 2)), {}), (dict(shards=2 ** 32 + 1), {}), (dict(first=-1), {}), ({}, dict(text_len=2 ** 32)),
                                     ({}, dict(text_len=-1)), ({}, dict(video_len=5)), ({}, dict(text_len=2, video_len=3))])
def test_numbers_that_an_int_does_not_hold_are_refused(rope, kw):
    from ditango_b200 import _capi, ops
    x, w = torch.zeros(1, 4, 1, 64, device="cuda"), torch.ones(64, device="cuda")
    rope = ops.GridRope(**dict(dict(grid=(1, 2, 2), axes=(16, 24, 24)), **rope))
    with pytest.raises(_capi.ExtensionError):
        ops.norm_rope_grid(x, x, (w, None, 1e-6), (w, None, 1e-6), rope, **kw)
    with pytest.raises(_capi.ExtensionError):
        ops.norm_rope_grid_backward(x, x, x, x, (w, None, 1e-6), (w, None, 1e-6), rope, **kw)


def test_no_heads_on_one_side_are_refused():
    from ditango_b200 import _capi, ops
    x, w = torch.zeros(1, 4, 1, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(_capi.ExtensionError):
        ops.norm_rope_grid(x, x[:, :, :0], (w, None, 1e-6), (w, None, 1e-6), ops.GridRope((1, 2, 2), (16, 24, 24)))


@pytest.mark.parametrize("H,D", [(1, 64), (3, 64), (24, 64), (1, 128), (8, 128)])
@pytest.mark.parametrize("tokens", [1, 3, 9, 131])
def test_what_shared_memory_held_before_does_not_matter(H, D, tokens):
    """Launches whose last CTA has room for more tokens than there are, behind launches that leave NaN in the shared memory of all SMs."""
    from ditango_b200 import ops
    q, k, norms, g = _inputs(1, tokens, H, H, D, torch.float32, True, tokens)
    dq, dk = (torch.randn(1, tokens, H, D, generator=g).cuda() for _ in range(2))
    args = (q.cuda(), k.cuda(), *_cuda(norms), _rope((1, 1, tokens), D))
    want = ops.norm_rope_grid_backward(dq, dk, *args)
    nan = torch.full((16, 2000, 24, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    for _ in range(5):
        ops.flash_window(nan[:, :1], nan, nan, left=1999, right=0)
        got = ops.norm_rope_grid_backward(dq, dk, *args)
        assert all(x.isfinite().all() and torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("front", [1, 3, 8])
def test_a_gradient_that_begins_anywhere_in_memory(front):
    """Behind `front` other values of one tensor, as the gradient of a concatenation does."""
    from ditango_b200.executor.cogvideox_dit import norm_and_rotate_grid
    torch.manual_seed(2)
    rope = _rope((2, 3, 4), 64)
    nq, nk = (nn.LayerNorm(64, eps=1e-6).cuda().to(torch.bfloat16) for _ in range(2))
    x = torch.randn(1, 24, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    leaves = [x, *nq.parameters(), *nk.parameters()]
    dz = torch.randn(front + 2 * x.numel(), device="cuda").to(torch.bfloat16)
    outs = norm_and_rotate_grid(x, x, nq, nk, rope, 0)
    got = torch.autograd.grad(torch.cat([x.new_zeros(front), *(o.flatten() for o in outs)]), leaves, dz)
    a, b = (d.clone().view_as(x) for d in dz[front:].chunk(2))
    want = torch.autograd.grad(norm_and_rotate_grid(x, x, nq, nk, rope, 0), leaves, (a, b))
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("eps", [0.0, 1e-40])
def test_norms_without_an_eps_take_the_separate_operations(eps):
    """What has an inverse root without one (no row is constant here) stays as it was; the kernel refuses such an eps."""
    from ditango_b200 import _capi, ops
    from ditango_b200.executor.cogvideox_dit import norm_and_rotate_grid
    torch.manual_seed(3)
    rope = _rope((2, 3, 4), 64)
    q, k = (torch.randn(1, 24, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    nq, nk = (nn.LayerNorm(64, eps=e).cuda().to(torch.bfloat16) for e in (eps, 1e-6))
    for norms in ((nq, nk), (nk, nq)):
        n = ops.LaunchLog.count
        outs = norm_and_rotate_grid(q, k, *norms, rope, 0)
        assert ops.LaunchLog.count == n
        for a, b in zip(outs, norm_and_rotate_grid(q, k, nk, nk, rope, 0)):     # (1e-6 beside a variance of 1; bf16 at every step)
            assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * b.float().abs().max()
        with pytest.raises(_capi.ExtensionError, match="eps"):
            ops.norm_rope_grid(q, k, *((m.weight, m.bias, m.eps) for m in norms), rope)
