"""The reuse path with its cache in 8 bits, on logical ranks of one GPU.

A state's rounding to codes is off by at most half a step: less than A / 127 in int8 (the step is below 2 A / 127) and 2^-4 A in e4m3,
A the largest value of a state.  A merge is a convex combination, so it neither grows A nor the error, and a state is
rounded once when it is stored and once more each time its block merges into a coarser one.  This comes on top of what the
unquantised path is allowed, 2e-2."""
import pytest
import torch

from oracle import ring_oracle as O
from tests.test_loopback_ring import RING_CASES, _init_schedule, _ring_on_loopback
from tests import loopback as LB

pytestmark = pytest.mark.gpu

CODES = (torch.int8, torch.float8_e4m3fn)
HALF_STEP = {torch.int8: 1 / 127, torch.float8_e4m3fn: 2.0 ** -4}


def _largest_state(data, world):
    top = 0.0
    for q, k, v in data:
        n = k.shape[1] // world
        for c in range(world):
            o, _ = O.partial_attention(q, k[:, c * n:(c + 1) * n], v[:, c * n:(c + 1) * n], out_dtype=torch.float32)
            top = max(top, float(o.abs().max()))
    return top


def _in_8_bits(code, seen=None):
    def setup(layer):
        layer.cache_dtype = layer.cache.store_dtype = code
        layer.output_dtype = torch.bfloat16
        if seen is not None:
            seen.append(layer)
    return setup


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("name", ["trace_n4", "n8", "cfg1_n2"])
def test_reuse_with_a_cache_in_8_bits(name, code):
    from ditango_b200 import ops
    c = RING_CASES[name]
    world, div = c["world"], c["dividers"]
    data = O.drifting_qkv(c["B"], c["S"], c["H"], c["D"], len(div), seed=c["seed"], drift=c["drift"], dtype=torch.bfloat16)
    _init_schedule(world, div)
    res = _ring_on_loopback(world, data, torch.device("cuda"), layer_setup=_in_8_bits(code))
    ref, _ = O.run_ring_group(world, div, data)
    rounds = 1 + len({d for d in div if d > 1}) - 1
    most = 2e-2 + rounds * HALF_STEP[code] * _largest_state(data, world)
    for r in range(world):
        for t in range(len(div)):
            assert (res[r][0][t] - ref[t][r]).abs().max() <= most
    assert ops.read_status() == 0


@pytest.mark.parametrize("code", CODES)
def test_slots_hold_rows_and_their_bytes_are_counted(code):
    from ditango_b200 import ops
    from ditango_b200.core.attention import proAttention
    world, div = 4, [1, 4, 2, 2]
    data = O.drifting_qkv(1, 512, 2, 64, len(div), seed=0, dtype=torch.bfloat16)
    _init_schedule(world, div)

    def body(r, group, fabric):
        layer = proAttention(0, group)
        _in_8_bits(code)(layer)
        counts = []
        for t, (q, k, v) in enumerate(data):
            LB.stepped(fabric, r, t)
            o = layer.attn(*(x[:, r * 128:(r + 1) * 128].contiguous().cuda() for x in (q, k, v)))
            slots = [b for b in layer.cache.out_block_cache if b is not None]
            assert o.dtype == torch.bfloat16 and all(isinstance(b, ops.QuantizedRows) and b.dtype == code for b in slots)
            counts.append((len(slots), layer.cache.cached_bytes()))
        return counts, layer.cache.block_size_mb
    for counts, size in LB.run_ranks(world, body):
        assert any(n for n, _ in counts)
        assert size == 128 * 2 * (64 + 5) / 2 ** 20 and all(b == n * 128 * 2 * (64 + 5) for n, b in counts)


@pytest.mark.parametrize("code", CODES)
def test_packed_segments_and_the_pair_map(code):
    """Packed calls, and chunks cached one by one under a per-pair map."""
    from ditango_b200 import ops
    world, T, S, H, D = 4, 4, 560, 2, 64
    g = torch.Generator().manual_seed(3)
    reusable = torch.rand(T, world, world, generator=g) < 0.6
    reusable[0] = False
    data = O.drifting_qkv(1, S, H, D, T, seed=6, drift=0.05, dtype=torch.bfloat16)
    _init_schedule(world, steps=T, pair_map=reusable.numpy())
    want = O.run_pair_map_group(world, reusable.numpy(), data)
    cu = [[0, S // world, S // world]] * world
    for kw in (dict(), dict(cu=cu)):
        res = _ring_on_loopback(world, data, torch.device("cuda"), layer_setup=_in_8_bits(code), **kw)
        most = 2e-2 + HALF_STEP[code] * _largest_state(data, world)
        for r in range(world):
            for t in range(T):
                assert (res[r][0][t] - want[t][r]).abs().max() <= most
    assert ops.read_status() == 0


def test_overlapping_launches_give_the_same_bits():
    world, div = 4, [1, 4, 4, 2, 1]
    data = O.drifting_qkv(1, 1204, 2, 128, len(div), seed=1, drift=0.05, dtype=torch.bfloat16)
    got = []
    for chain in (False, True):
        _init_schedule(world, div)

        def setup(layer):
            _in_8_bits(torch.int8)(layer)
            layer.chain_launches = chain
        got.append(_ring_on_loopback(world, data, torch.device("cuda"), layer_setup=setup))
    for a, b in zip(*got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
