"""States in 8 bits: written, read back, merged and re-blocked, against the same steps in 64 bits.

Half a step of the codes: int8 2^(b - 127) / 2; e4m3 2^-4 of a value's power of two (2^-10 * 2^(b - 127) below its smallest normal
number).  A merge is fp32: each weight is off by a few 2^-23, so the result by less than 2^-20 of the largest |value| merged."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

CODES = (torch.int8, torch.float8_e4m3fn)
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def _spread(shape, g):
    """Rows of very different size, some all zero."""
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-30, 30, shape[:-1], generator=g).float())[..., None]
    return x * (torch.rand(shape[:-1], generator=g) > 0.1)[..., None]


def _values(rows):
    v, e = rows.values.cpu().double() if rows.dtype == torch.int8 else rows.values.cpu().float().double(), rows.exponents.cpu()
    return v * torch.exp2(e.double() - 127)[..., None]


def _smallest_exponents(x, code):
    top = x.double().abs().amax(-1)
    m, e = torch.frexp(top / LARGEST[code])
    return torch.where(top == 0, torch.zeros_like(e), e - (m == 0.5).int() + 127).clamp(min=8)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 64), (1, 1, 1, 128), (2, 37, 3, 64), (41, 7, 128), (1, 515, 48, 64), (2, 1033, 24, 128)])
def test_rows_are_written_to_the_nearest_code_and_read_back_exactly(shape, dtype, code):
    from ditango_b200 import ops
    x = _spread(shape, torch.Generator().manual_seed(sum(shape))).to(dtype)
    rows = ops.quantize_rows(x.cuda(), code)
    assert rows.dtype == code and torch.equal(rows.exponents.cpu().int(), _smallest_exponents(x, code).int())
    scaled = x.double() * torch.exp2(127 - rows.exponents.cpu().double())[..., None]
    want = scaled.round() if code == torch.int8 else scaled.float().to(code).float().double()
    got = rows.values.cpu().double() if code == torch.int8 else rows.values.cpu().float().double()
    assert torch.equal(got, want)
    for back in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.dequantize_rows(rows, back).cpu().double(), _values(rows))


def test_ties_borders_and_rows_that_are_not_finite():
    from ditango_b200 import ops
    x = torch.zeros(1, 8, 1, 64)
    x[0, 0, 0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])              # ties go to even codes; the largest value is a code
    x[0, 1, 0, :2] = torch.tensor([127.5, -1.0])                        # above it: the next power of two
    x[0, 2, 0, :2] = torch.tensor([448.0, 17.0])
    x[0, 3, 0, 5] = math.inf
    x[0, 4, 0, 9] = math.nan
    x[0, 5, 0, 0] = 3e38
    x[0, 6, 0, 0] = 1e-37
    rows8, rowsf = (ops.quantize_rows(x.cuda(), c) for c in CODES)
    assert rows8.values[0, 0, 0, :4].tolist() == [127, 0, 2, -2] and rows8.exponents[0, 0, 0] == 127
    assert rows8.values[0, 1, 0, :2].tolist() == [64, 0] and rows8.exponents[0, 1, 0] == 128
    assert rowsf.values[0, 2, 0, :2].float().tolist() == [448.0, 16.0] and rowsf.exponents[0, 2, 0] == 127
    for rows in (rows8, rowsf):
        back = ops.dequantize_rows(rows)
        assert rows.exponents[0, 3:5, 0].tolist() == [255, 255] and back[0, 3:5].isnan().all()
        assert abs(float(back[0, 5, 0, 0]) / 3e38 - 1) <= 2.0 ** -4 and float(back[0, 6, 0, 0]) <= 1.1e-37
        assert (back[0, 7] == 0).all() and back[0, :3].isfinite().all()


def _merge_exact(states, shape):
    B, S, H, D = shape if len(shape) == 4 else (1, *shape)
    lses = torch.stack([(l if lay == 1 else l.transpose(-1, -2)).reshape(B, S, H).double() for _, l, lay in states])
    lse = torch.logsumexp(lses, 0)
    out = torch.zeros(B, S, H, D, dtype=torch.float64)
    for (v, _, _), l in zip(states, lses):
        w = torch.where(l == -math.inf, torch.zeros_like(l), (l - lse).exp())[..., None]
        out += torch.where(w > 0, w * v.reshape(B, S, H, D), torch.zeros_like(w))
    return out.reshape(shape), lse


def _states(shape, kinds, g, layouts=(1, 0)):
    """(states for the kernel, the same with their values in 64 bits); lse -inf in places, and there a NaN in the values."""
    from ditango_b200 import ops
    lead = shape[:-3]
    mine, exact = [], []
    for i, kind in enumerate(kinds):
        lay = layouts[i % len(layouts)]
        x = torch.randn(*shape, generator=g)
        lse = torch.randn(lead + (shape[-3:-1] if lay == 1 else (shape[-2], shape[-3])), generator=g) * 3
        empty = torch.rand(lse.shape, generator=g) < 0.15
        lse[empty] = -math.inf
        x[empty if lay == 1 else empty.transpose(-1, -2)] = math.nan
        v = ops.quantize_rows(x.cuda(), kind) if kind in CODES else x.to(kind).cuda()
        mine.append((v, lse.cuda(), lay))
        exact.append((_values(v) if kind in CODES else v.cpu().double(), lse, lay))
    return mine, exact


F, H16, I, E = torch.float32, torch.bfloat16, *CODES


@pytest.mark.parametrize("shape,kinds", [
    ((1, 1, 1, 64), (I,)), ((1, 1, 1, 128), (F, E)), ((2, 37, 3, 64), (E, F, I, H16)), ((41, 7, 128), (H16, I)),
    ((1, 333, 48, 64), (F,) + (E,) * 7), ((2, 129, 24, 128), (I,) * 7 + (F,)), ((1, 65, 5, 64), (I, E) * 8), ((1, 65, 5, 128), (E, H16, F, I) * 4)])
@pytest.mark.parametrize("layout", [0, 1])
def test_merge_reads_states_of_every_type(shape, kinds, layout):
    from ditango_b200 import ops
    mine, exact = _states(shape, kinds, torch.Generator().manual_seed(len(kinds)))
    want, want_lse = _merge_exact(exact, shape)
    b16 = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    out, lse = ops.merge_states(mine, lse_out_layout=layout, out_bf16=b16)
    top = max(v[v.isfinite()].abs().max() for v, _, _ in exact)
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -20 * top).all()
    assert ((b16.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -20 * top).all()
    got = (lse if layout == 1 else lse.transpose(-1, -2)).cpu().double().reshape(want_lse.shape)
    live = want_lse > -math.inf
    assert torch.equal(got == -math.inf, ~live) and ((got - want_lse)[live].abs() <= 2.0 ** -19 * (1 + want_lse[live].abs())).all()
    assert (out.cpu()[~live.reshape(out.shape[:-1])] == 0).all()
    only, none = ops.merge_states(mine, out_bf16=b16, fp32_out=False, want_lse=False)
    assert only is b16 and none is None


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("shape", [(1, 1, 3, 64), (2, 97, 7, 128), (1, 700, 48, 64)])
def test_a_merged_block_is_written_in_8_bits(shape, code):
    """Its values are within half a step of the merge in 64 bits (and an fp32 rounding of the merge, which may tip a tie)."""
    from ditango_b200 import ops
    mine, exact = _states(shape, (code, F, code, H16), torch.Generator().manual_seed(9))
    want, _ = _merge_exact(exact, shape)
    rows, lse = ops.merge_states(mine, out_rows=code, fp32_out=False)
    assert isinstance(rows, ops.QuantizedRows) and rows.dtype == code and lse.shape == shape[:-1]
    step = torch.exp2(rows.exponents.cpu().double() - 127)[..., None]
    half = step / 2 if code == torch.int8 else torch.maximum(want.abs() * 2.0 ** -4, step * 2.0 ** -10)
    top = max(v[v.isfinite()].abs().max() for v, _, _ in exact)
    assert ((_values(rows) - want).abs() <= half + 2.0 ** -19 * top).all()
    again, _ = ops.merge_states(mine, out_rows=ops.QuantizedRows(torch.empty_like(rows.values), torch.empty_like(rows.exponents)), fp32_out=False)
    assert torch.equal(again.values.view(torch.uint8), rows.values.view(torch.uint8)) and torch.equal(again.exponents, rows.exponents)


def test_in_place_and_captured():
    """Merged into the fp32 state that is one of the inputs; the same in a graph, replayed on other values."""
    from ditango_b200 import ops
    shape = (2, 50, 4, 64)
    g = torch.Generator().manual_seed(2)
    mine, _ = _states(shape, (F, I, E), g, layouts=(1,))
    want, want_lse = ops.merge_states(mine)
    own, own_lse = mine[0][0].clone(), mine[0][1].clone()
    out, lse = ops.merge_states([(own, own_lse, 1)] + mine[1:], out=own, lse_out=own_lse)
    assert out is own and torch.equal(own.nan_to_num(), want.nan_to_num()) and torch.equal(own_lse, want_lse)

    x = torch.randn(shape, device="cuda")
    rows = ops.quantize_rows(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.quantize_rows(x, rows=rows)
            back = ops.dequantize_rows(rows)
    torch.cuda.current_stream().wait_stream(side)
    x.copy_(torch.randn(shape, device="cuda") * 5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(back, ops.dequantize_rows(ops.quantize_rows(x)))


def test_rows_past_32_bit_offsets():
    """2^31 values and more in one tensor: the last rows come out like those of a tensor of their own."""
    from ditango_b200 import ops
    S = 2 ** 31 // (48 * 64) + 5
    x = torch.zeros(1, S, 48, 64, dtype=torch.bfloat16, device="cuda")
    x[:, -4:] = torch.randn(1, 4, 48, 64, device="cuda").to(torch.bfloat16)
    rows = ops.quantize_rows(x)
    tail = ops.quantize_rows(x[:, -4:].contiguous())
    assert torch.equal(rows.values[:, -4:], tail.values) and torch.equal(rows.exponents[:, -4:], tail.exponents)
    back = ops.dequantize_rows(rows, torch.bfloat16)
    assert torch.equal(back[:, -4:], ops.dequantize_rows(tail, torch.bfloat16)) and not back[:, :-4].any()


def test_empty_tensors_launch_nothing():
    from ditango_b200 import ops
    rows = ops.quantize_rows(torch.empty(2, 0, 3, 64, device="cuda"))
    assert rows.shape == (2, 0, 3, 64) and ops.dequantize_rows(rows).shape == (2, 0, 3, 64)


def test_a_nan_among_the_lse_shows():
    from ditango_b200 import ops
    outs, lses = torch.randn(2, 1, 5, 3, 64, device="cuda"), torch.randn(2, 1, 5, 3, device="cuda")
    lses[0, 0, 2, 1] = math.nan
    out, lse = ops.merge_states([(ops.quantize_rows(outs[0]), lses[0], ops.LSE_BSH), (outs[1], lses[1], ops.LSE_BSH)])
    assert out[0, 2, 1].isnan().all() and int(out.isnan().sum()) == 64 and lse.isnan().nonzero().tolist() == [[0, 2, 1]]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kinds", [(F, F), (H16, F), (H16, H16, H16), (F,) * 5, (F, H16) * 8, (F,), (F, I), (E, H16, F)], ids=str)
def test_a_nan_among_the_lse_shows_whatever_the_states_are_held_in(kinds, D):
    """In its own row alone, whichever state has it, beside empty states too; a row of empty states stays one."""
    from ditango_b200 import ops
    n, shape = len(kinds), (2, 37, 3, D)
    g = torch.Generator().manual_seed(n)
    outs, lses = torch.randn(n, *shape, generator=g), torch.randn(n, *shape[:-1], generator=g)
    lses[:, 0, 4, 1] = -math.inf                 # nothing in any state
    lses[:, 0, 5, 1], lses[n - 1, 0, 5, 1] = -math.inf, math.nan       # a NaN beside empty states
    lses[n // 2, 1, 36, 2] = math.nan
    lses[0, 1, 0, 0] = math.nan
    bad = [[0, 5, 1], [1, 0, 0], [1, 36, 2]]
    for layout in (ops.LSE_BSH, ops.LSE_BHS):
        mine = [(ops.quantize_rows(o.cuda(), k) if k in CODES else o.to(k).cuda(), (l if layout == 1 else l.transpose(1, 2)).contiguous().cuda(), layout)
                for k, o, l in zip(kinds, outs, lses)]
        b16 = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        out, lse = ops.merge_states(mine, lse_out_layout=layout, out_bf16=b16)
        lse = lse if layout == 1 else lse.transpose(1, 2)
        for x in (out, b16):
            assert x.isnan().all(-1).nonzero().tolist() == bad and int(x.isnan().sum()) == len(bad) * D
        assert lse.isnan().nonzero().tolist() == bad and (lse == -math.inf).nonzero().tolist() == [[0, 4, 1]] and (out[0, 4, 1] == 0).all()


@pytest.mark.parametrize("code", CODES)
def test_results_of_several_types_at_once_are_those_of_separate_calls(code):
    from ditango_b200 import ops
    shape = (2, 97, 7, 128)
    mine, _ = _states(shape, (code, F, code, H16), torch.Generator().manual_seed(3))
    rows, lse = ops.merge_states(mine, out_rows=code, fp32_out=False)
    mine_rows, b16 = ops._new_rows("cuda", shape, code), torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    out, lse2 = ops.merge_states(mine, out_bf16=b16, out_rows=mine_rows)
    assert torch.equal(mine_rows.values.view(torch.uint8), rows.values.view(torch.uint8)) and torch.equal(mine_rows.exponents, rows.exponents)
    assert torch.equal(out, ops.merge_states(mine)[0]) and torch.equal(b16, out.to(torch.bfloat16)) and torch.equal(lse, lse2)
    again = ops._new_rows("cuda", shape, code)
    got, _ = ops.merge_states(mine, out_bf16=b16, out_rows=again, fp32_out=False)
    assert got is b16 and torch.equal(again.exponents, rows.exponents)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("gap", [math.inf, 1e4, 200.0])
def test_a_weight_that_is_0_in_fp32_keeps_what_is_not_finite_out(gap, D, code):
    """A state that far below the others may hold anything, in 8 bits as in the wide types; a little nearer a NaN shows."""
    from ditango_b200 import ops
    shape = (1, 33, 3, D)
    g = torch.Generator().manual_seed(D)
    x, bad = torch.randn(shape, generator=g).cuda(), torch.randn(shape, generator=g)
    bad[0, 5:20, 1, 7], bad[0, 9, 2, 0] = math.nan, math.inf
    lse = torch.randn(shape[:-1], generator=g).cuda()
    for kind in (code, F, H16):
        rows = ops.quantize_rows(bad.cuda(), code) if kind in CODES else bad.to(kind).cuda()
        mine = [(rows, lse - gap, ops.LSE_BSH), (x, lse, ops.LSE_BSH)]
        out, out_lse = ops.merge_states(mine)
        assert torch.equal(out, x) and torch.equal(out_lse, lse)
        back = ops.merge_states(mine, out_rows=code, fp32_out=False)[0]
        assert torch.equal(back.exponents, ops.quantize_rows(x, code).exponents) and int(back.exponents.max()) < 255
        near, _ = ops.merge_states([(rows, lse - 20, ops.LSE_BSH), (x, lse, ops.LSE_BSH)])
        assert near[0, 5:20, 1].isnan().any() and not near[0, 5:20, 0].isnan().any()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [F, H16])
@pytest.mark.parametrize("D", [64, 128])
def test_values_below_the_smallest_normal_number(D, dtype, code):
    """Rows whose values are smaller than 2^-126, all of them or some: codes and what they stand for, through a merge too."""
    from ditango_b200 import ops
    g = torch.Generator().manual_seed(D)
    x = (torch.randn(1, 60, 3, D, generator=g).double() * torch.exp2(-100 - torch.arange(60, dtype=torch.float64) / 2)[None, :, None, None]).to(dtype)
    assert (x.double().abs().amax(-1) < 2.0 ** -126).any()
    rows = ops.quantize_rows(x.cuda(), code)
    scale = torch.exp2(127 - rows.exponents.cpu().double())[..., None]
    assert torch.equal(rows.exponents.cpu().int(), _smallest_exponents(x, code).int())
    want = (x.double() * scale).round() if code == torch.int8 else (x.double() * scale).float().to(code).float().double()
    got = rows.values.cpu().double() if code == torch.int8 else rows.values.cpu().float().double()
    assert torch.equal(got, want) and (got[:, 52:] != 0).any() == (code != torch.int8)
    for back in (F, H16):
        assert torch.equal(ops.dequantize_rows(rows, back).cpu().double(), _values(rows))
    lse = torch.zeros(1, 60, 3, device="cuda")
    out, _ = ops.merge_states([(rows, lse, ops.LSE_BSH)])
    assert torch.equal(out.cpu().double(), _values(rows))
    again, _ = ops.merge_states([(rows, lse, ops.LSE_BSH)], out_rows=code, fp32_out=False)
    assert torch.equal(_values(again), _values(rows))
