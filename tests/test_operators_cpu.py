"""What the entry points of the operators refuse, on tensors and pointers that never reach a GPU."""
import ctypes
import os
import re

import pytest
import torch


def _ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


def _ints(*values):
    return (ctypes.c_int * len(values))(*values)


def _merge_rows(lib, *, n=1, outs=(16,), dts=(2,), exps=(16,), lses=(16,), lays=(1,), out=None, lse=None, lse_lay=1, b16=None,
                codes=None, code_t=2, code_e=None, B=1, S=2, H=3, D=64):
    return lib.dtb_merge_rows(n, _ptrs(*outs), _ints(*dts), _ptrs(*exps), _ptrs(*lses), _ints(*lays), out, lse, lse_lay, b16,
                              codes, code_t, code_e, B, S, H, D, None)


@pytest.mark.parametrize("args,word", [
    (dict(n=17, out=32), "nstates"), (dict(n=0, out=32), "nstates"), (dict(D=96, out=32), "head_dim"), (dict(), "no result"),
    (dict(out=32, dts=(7,)), "dtype"), (dict(out=32, exps=(None,)), "null"), (dict(out=32, outs=(None,)), "null"),
    (dict(out=32, outs=(24,)), "aligned"), (dict(out=40), "aligned"), (dict(codes=32, code_e=None), "exponents"),
    (dict(codes=32, code_e=64, code_t=1), "8-bit result"), (dict(out=32, lses=(None,), lse=64), "lse"),
    (dict(n=2, outs=(16, 32), dts=(2, 0), exps=(16, None), lses=(16, None), lays=(1, 1), out=64), "lse"),
    (dict(out=32, lays=(2,)), "layout"), (dict(out=32, lse=64, lse_lay=5), "lse_out_layout"), (dict(codes=16, code_e=64), "own type"),
    (dict(out=16), "own type"), (dict(out=32, lse=16, lse_lay=0), "matching layouts"), (dict(out=32, S=-1), "shape"),
    (dict(out=32, B=65536, S=65536), "2^31"), (dict(out=32, S=2 ** 30, H=4), "2^31")])
def test_merge_rows_refuses(args, word):
    from ditango_b200 import _capi
    lib = _capi.load()
    assert _merge_rows(lib, **args) == -1 and word in lib.dtb_last_error().decode()


def test_rows_on_the_cpu_and_of_other_types_are_refused():
    from ditango_b200 import ops
    from ditango_b200._capi import ExtensionError
    x = torch.zeros(1, 2, 3, 64)
    rows = ops.QuantizedRows(x.to(torch.int8), torch.zeros(1, 2, 3, dtype=torch.uint8))
    for call in (lambda: ops.quantize_rows(x), lambda: ops.dequantize_rows(rows), lambda: ops.dequantize_rows(rows, torch.float16),
                 lambda: ops.merge_states([(rows, torch.zeros(1, 2, 3), ops.LSE_BSH)]),
                 lambda: ops.merge_states([(x, torch.zeros(1, 2, 3), ops.LSE_BSH)], out_rows=torch.float16, fp32_out=False)):
        with pytest.raises(ExtensionError):
            call()
    with pytest.raises(ExtensionError):
        ops._new_rows(x.device, x.shape, torch.uint8)


def test_single_states_refuse():
    from ditango_b200 import _capi
    lib = _capi.load()
    for rc in (lib.dtb_quantize_rows(16, 2, 16, 2, 16, 5, 64, None), lib.dtb_quantize_rows(16, 0, None, 2, 16, 5, 64, None),
               lib.dtb_quantize_rows(16, 0, 32, 1, 16, 5, 64, None), lib.dtb_quantize_rows(16, 0, 32, 2, None, 5, 64, None),
               lib.dtb_quantize_rows(16, 0, 32, 2, 16, -1, 64, None), lib.dtb_quantize_rows(16, 0, 32, 2, 16, 2 ** 31, 64, None),
               lib.dtb_dequantize_rows(16, 0, 16, 32, 0, 5, 64, None), lib.dtb_dequantize_rows(16, 2, 16, 32, 2, 5, 64, None),
               lib.dtb_dequantize_rows(16, 2, None, 32, 0, 5, 64, None), lib.dtb_dequantize_rows(16, 2, 16, None, 0, 5, 64, None),
               lib.dtb_dequantize_rows(16, 2, 16, 32, 0, 5, 80, None)):
        assert rc == -1


@pytest.mark.parametrize("key,dtype", [("int8", torch.int8), ("e4m3", torch.float8_e4m3fn), ("bf16", torch.bfloat16), ("fp32", torch.float32)])
def test_the_cache_type_is_a_config_key(key, dtype, tmp_path):
    from ditango_b200.core.attention import proAttention
    from ditango_b200.core import config
    from ditango_b200.core.group_coordinate import SingleRankGroup
    (tmp_path / "c.yaml").write_text(f"cache-dtype: {key}\n")
    before = config.DITANGO_CONFIG
    try:
        config.init_config(str(tmp_path / "c.yaml"), make_output_dir=False)
        layer = proAttention(0, SingleRankGroup(torch.device("cpu")))
        assert layer.cache_dtype == layer.cache.store_dtype == dtype
    finally:
        config.DITANGO_CONFIG = before


def _window(lib, *, q=16, k=16, v=16, qt=192, qb=1920, kt=192, kb=1920, vt=192, vb=1920, out=16, odt=0, lse=16, lay=0, acc=0, cq=None, ck=None,
            sl=None, n=2, sq=10, sk=10, tq=20, tk=20, H=3, Hk=3, D=64, scale=0.1, left=3, right=3, sinks=0, qs=0, ks=0, scratch=None):
    return lib.dtb_flash_window(q, k, v, qt, qb, kt, kb, vt, vb, out, odt, lse, lay, acc, cq, ck, sl, n, sq, sk, tq, tk, H, Hk, D, scale,
                                left, right, sinks, qs, ks, scratch, 0, None)


@pytest.mark.parametrize("args,word", [
    (dict(q=None), "null"), (dict(lse=None), "null"), (dict(D=80), "head_dim"), (dict(H=3, Hk=2), "query heads"), (dict(Hk=0), "query heads"),
    (dict(n=0), "nseg"), (dict(sq=-1), "negative"), (dict(n=1, sq=2 ** 30, tq=2 ** 30), "too many"), (dict(cq=16), "cu_seqlens"),
    (dict(cq=16, ck=16, sl=16), "seqlens_k"), (dict(tq=21), "total"), (dict(tk=19), "total"), (dict(left=-2), "window"), (dict(right=2 ** 30 + 1), "window"),
    (dict(sinks=-1), "sinks"), (dict(qs=2 ** 30 + 1), "position"), (dict(ks=-2 ** 30 - 1), "position"), (dict(qt=128), "token stride"),
    (dict(kb=128), "batch stride"), (dict(vt=196), "multiples of 8"), (dict(q=24), "aligned"), (dict(odt=2), "out_dtype"), (dict(lay=2), "lse_layout"),
    (dict(acc=1, odt=1), "accumulate"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scratch=24), "scratch")])
def test_flash_window_refuses(args, word):
    from ditango_b200 import _capi
    lib = _capi.load()
    assert _window(lib, **args) == -1 and word in lib.dtb_last_error().decode()


@pytest.mark.parametrize("args,word", [((0, 9, 9, 2, 2, 64, 1, 1, 0), "shape"), ((1, -1, 9, 2, 2, 64, 1, 1, 0), "shape"), ((1, 9, 9, 3, 2, 64, 1, 1, 0), "shape"),
                                       ((1, 9, 9, 2, 0, 64, 1, 1, 0), "shape"), ((1, 9, 9, 2, 2, 32, 1, 1, 0), "shape"), ((1, 9, 9, 2, 2, 64, -2, 1, 0), "window"),
                                       ((1, 9, 9, 2, 2, 64, 1, 1, -1), "sinks")])
def test_flash_window_scratch_refuses(args, word):
    from ditango_b200 import _capi
    lib = _capi.load()
    assert lib.dtb_flash_window_scratch_bytes(*args) == -1 and word in lib.dtb_last_error().decode()


def test_flash_window_takes_gpu_tensors_only():
    from ditango_b200 import ops
    from ditango_b200._capi import ExtensionError
    q = torch.zeros(1, 8, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ExtensionError):
        ops.flash_window(q, q, q, left=3)


def _grid_rope(lib, *, q=16, qt=192, qb=1920, qo=16, qw=16, qbias=None, q_eps=1e-6, k=16, dtype=1, grid=(2, 3, 4), axes=(16, 24, 24), place=(1e4, 0, 0, 0, 1, 1, 1),
               first=0, shards=1, B=1, S=10, text=2, video=8, H=3, Hk=3, D=64, back=False, scratch=16, scratch_bytes=1 << 30):
    arrays = (ctypes.c_int * 3)(*grid), (ctypes.c_int * 3)(*axes), (ctypes.c_double * 7)(*place)
    rest = (dtype, 0, *arrays, first, shards, B, S, text, video, H, Hk, D)
    if back:
        return lib.dtb_norm_rope_grid_backward(16, 192, 1920, 16, qt, qb, q, qt, qb, qw, q_eps, k, 192, 1920, 16, 1e-6, qo, 16, 16, None, 16, None,
                                               *rest, scratch, scratch_bytes, None)
    return lib.dtb_norm_rope_grid(q, qt, qb, qo, qw, qbias, q_eps, k, 192, 1920, 16, 16, None, 1e-6, *rest, None)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("args,word", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(qw=None), "null"), (dict(D=32), "head_dim"), (dict(dtype=2), "dtype"), (dict(H=0), "shape"),
    (dict(text=3), "text and"), (dict(video=-1), "text and"), (dict(text=-1), "text and"), (dict(grid=(2, -1, 4)), "negative grid"),
    (dict(grid=(2 ** 16, 2 ** 10, 2 ** 10)), "2^31"), (dict(axes=(16, 25, 23)), "channels"), (dict(axes=(16, 24, 26)), "channels"),
    (dict(axes=(-2, 34, 32)), "channels"), (dict(first=-1), "first"), (dict(shards=0), "shards"), (dict(place=(0, 0, 0, 0, 1, 1, 1)), "base"),
    (dict(place=(1e4, float("nan"), 0, 0, 1, 1, 1)), "finite"), (dict(q_eps=0.0), "eps"), (dict(q_eps=float("nan")), "eps"), (dict(qt=196), "multiples"), (dict(qo=24), "aligned")])
def test_norm_rope_grid_refuses(args, word, back):
    from ditango_b200 import _capi
    lib = _capi.load()
    assert _grid_rope(lib, back=back, **args) == -1 and word in lib.dtb_last_error().decode()


def test_norm_rope_grid_takes_gpu_tensors_only():
    from ditango_b200 import _capi, ops
    x, w = torch.zeros(1, 8, 1, 64), torch.ones(64)
    with pytest.raises(_capi.ExtensionError):
        ops.norm_rope_grid(x, x, (w, None, 1e-6), (w, None, 1e-6), ops.GridRope((1, 2, 4), (16, 24, 24)))
    with pytest.raises(_capi.ExtensionError):
        ops.norm_rope_grid_backward(x, x, x, x, (w, None, 1e-6), (w, None, 1e-6), ops.GridRope((1, 2, 4), (16, 24, 24)))


def test_grid_positions_on_the_cpu_take_the_tables():
    """The general path, on tensors that no kernel takes, gives what norm_and_rotate gives on the model's tables."""
    from ditango_b200.executor.cogvideox_dit import DiTConfig, norm_and_rotate, norm_and_rotate_grid, rotary_tables
    cfg = DiTConfig(frames=2, height=6, width=8)
    torch.manual_seed(0)
    q, k = (torch.randn(1, 3 + cfg.video_tokens, 2, 64) for _ in range(2))
    norms = [torch.nn.LayerNorm(64) for _ in range(2)]
    a = norm_and_rotate(q, k, *norms, *rotary_tables(cfg, "cpu"), 3)
    b = norm_and_rotate_grid(q, k, *norms, cfg.grid_rope, 3)
    assert all((x - y).abs().max() < 1e-5 for x, y in zip(a, b))


@pytest.mark.parametrize("kw", [dict(), dict(fp32_out=False, out_bf16=True), dict(out_bf16=True), dict(out=True)])
def test_new_rows_that_the_caller_would_not_get_are_refused(kw):
    """A merge returns one result: rows beside another one are the caller's."""
    from ditango_b200 import ops
    from ditango_b200._capi import ExtensionError
    x, lse = torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 3)
    kw = {k: v if k == "fp32_out" else torch.empty_like(x, dtype=torch.bfloat16 if k == "out_bf16" else torch.float32) for k, v in kw.items()}
    with pytest.raises(ExtensionError, match="out_rows is a type only"):
        ops.merge_states([(x, lse, ops.LSE_BSH)], out_rows=torch.int8, **kw)
    rows = ops._new_rows(x.device, x.shape, torch.int8)
    for given in (dict(out_rows=torch.int8, fp32_out=False), dict(out_rows=rows, **kw)):     # (taken, and then refused for their device)
        with pytest.raises(ExtensionError, match="CUDA tensors only"):
            ops.merge_states([(x, lse, ops.LSE_BSH)], **given)


def test_what_a_result_may_take_the_place_of_is_read_by_ordinary_loads():
    """Loads for memory that stays as it is during a kernel are for codes and exponents alone: dtb_merge_rows may write the result over a
    state's wide values, and lse_out over its lse."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ditango_b200", "csrc")
    source = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, "merge_rows.cu")).read())
    lines = [line for line in source.splitlines() if re.search(r"__ldg|ld\.global\.nc|__restrict__", line)]
    assert len(lines) == 2 and "load_codes16(const void* p)" in lines[0] and "p.exponents[" in lines[1]
    uses = [line for line in source.splitlines() if "load_codes16(" in line][1:]
    assert len(uses) == 1 and "c0 + k < n8" in uses[0]               # the first n8 states are those in 8 bits


def test_merge_rows_refuses_a_state_s_exponents_for_the_result():
    from ditango_b200 import _capi
    lib = _capi.load()
    assert _merge_rows(lib, n=2, outs=(16, 32), dts=(0, 3), exps=(None, 48), lses=(16, 16), lays=(1, 1), codes=64, code_e=48) == -1
    assert "exponents of an 8-bit result" in lib.dtb_last_error().decode()


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("eps", [1e-40, 1.1e-38, -1e-6])
def test_norm_rope_grid_refuses_an_eps_that_the_kernels_count_as_0(eps, back):
    from ditango_b200 import _capi
    lib = _capi.load()
    assert _grid_rope(lib, back=back, q_eps=eps) == -1 and "eps" in lib.dtb_last_error().decode()
    assert _grid_rope(lib, back=back, q_eps=1.2e-38, S=0, text=0, video=0) != -1 or "eps" not in lib.dtb_last_error().decode()


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("first", [2 ** 63 - 1, 2 ** 62 + 1])
def test_norm_rope_grid_refuses_a_first_token_that_cannot_be_counted_on_from(first, back):
    from ditango_b200 import _capi
    lib = _capi.load()
    assert _grid_rope(lib, back=back, first=first) == -1 and "first token" in lib.dtb_last_error().decode()


def test_a_grid_s_numbers_are_taken_by_their_values():
    """A tensor among them that changes in place changes what the next call is given."""
    from ditango_b200 import ops
    q, w = torch.zeros(1, 8, 2, 64), torch.ones(64)
    base, at, step = torch.tensor(1e4), torch.tensor(0.5, dtype=torch.float64), torch.tensor(1.0)
    rope = ops.GridRope((1, 2, 4), (16, 24, 24), base=base, origin=(0.0, at, 0.0), step=(1.0, 1.0, step))
    place = lambda: list(ops._grid_rope_args(q, q, ((w, None, 1e-6),) * 2, rope, 0, None)[3][2])
    assert place() == [1e4, 0.0, 0.5, 0.0, 1.0, 1.0, 1.0]
    base.fill_(500.0), at.fill_(-3.25), step.fill_(2.0)
    assert place() == [500.0, 0.0, -3.25, 0.0, 1.0, 1.0, 2.0]
