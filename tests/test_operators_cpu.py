"""What the entry points of the operators refuse, on tensors and pointers that never reach a GPU."""
import ctypes

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
        ops._new_rows((1, 2, 3, 64), torch.uint8, "cpu")


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
