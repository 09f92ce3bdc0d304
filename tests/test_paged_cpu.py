"""What the entry points of paged keys and values refuse, on pointers and tensors that never reach a GPU."""
import pytest
import torch


def _lib():
    from ditango_b200 import _capi
    return _capi.load()


def _extend(lib, *, table=16, lens=16, new=16, free=16, count=16, B=2, M=4, pages=8, P=16, slots=16, tokens=5, cu=16, out=16, cnt=16, missing=16):
    return lib.dtb_extend_pages(table, lens, new, free, count, B, M, pages, P, slots, tokens, cu, out, cnt, missing, None)


def _release(lib, *, table=16, to=16, lens=16, begin=16, end=16, free=16, count=16, B=2, M=4, pages=8, P=16, out=16, cnt=16):
    return lib.dtb_release_pages(table, to, lens, begin, end, free, count, B, M, pages, P, out, cnt, None)


def _write(lib, *, k=16, v=16, kt=192, vt=192, tokens=5, slots=16, kp=16, ks=(4096, 192, 64), vp=16, vs=(4096, 192, 64), pages=8, P=16, Hk=3, D=64):
    return lib.dtb_write_pages(k, v, kt, vt, tokens, slots, kp, *ks, vp, *vs, pages, P, Hk, D, None)


def _flash(lib, *, q=16, qt=384, qb=3840, kp=16, ks=(4096, 192, 64), vp=16, vs=(4096, 192, 64), pages=8, P=16, table=16, M=4, lens=16, cu=None, out=16, odt=0, lse=16,
           lay=0, acc=0, n=2, sq=10, sk=10, tq=20, H=6, Hk=3, D=64, scale=0.1, left=3, right=3, sinks=0, scratch=16, size=1 << 40):
    return lib.dtb_flash_paged(q, qt, qb, kp, *ks, vp, *vs, pages, P, table, M, lens, cu, out, odt, lse, lay, acc, n, sq, sk, tq, H, Hk, D, scale, left, right, sinks,
                               scratch, size, None)


TABLES = [(dict(P=8), "page size"), (dict(P=48), "page size"), (dict(P=0), "page size"), (dict(P=2 ** 21), "page size"), (dict(pages=0), "pages"), (dict(M=0), "table"),
          (dict(M=2 ** 26), "too many tokens"), (dict(pages=2 ** 27), "too many tokens")]


@pytest.mark.parametrize("args,word", TABLES + [
    (dict(B=0), "table"), (dict(B=16385), "streams"), (dict(table=None), "null"), (dict(missing=None), "null"), (dict(slots=None), "null"), (dict(cu=None), "null"),
    (dict(tokens=-1), "tokens"), (dict(tokens=2 ** 31), "tokens"), (dict(slots=20), "aligned")])
def test_extend_refuses(args, word):
    lib = _lib()
    assert _extend(lib, **args) == -1 and word in lib.dtb_last_error().decode()


@pytest.mark.parametrize("args,word", TABLES + [
    (dict(B=-1), "table"), (dict(to=None), "null"), (dict(begin=None), "null"), (dict(free=None), "null"), (dict(cnt=None), "null"), (dict(B=2 ** 19), "too large")])
def test_release_refuses(args, word):
    lib = _lib()
    assert _release(lib, **args) == -1 and word in lib.dtb_last_error().decode()


@pytest.mark.parametrize("args,word", [
    (dict(P=24), "page size"), (dict(pages=2 ** 27), "too many tokens"), (dict(D=96), "head_dim"), (dict(Hk=0), "heads"), (dict(tokens=-1), "tokens"), (dict(k=None), "null"),
    (dict(slots=None), "null"), (dict(kp=None), "null"), (dict(kt=128), "strides"), (dict(vt=196), "strides"), (dict(k=24), "aligned"), (dict(vp=24), "aligned"),
    (dict(ks=(4096, 192, 60)), "multiples of 8"), (dict(ks=(4096, 32, 64)), "stride below"), (dict(vs=(4096, 192, 0)), "stride below"), (dict(vs=(2 ** 38, 192, 64)), "2^38"),
    (dict(ks=(4096, 128, 64)), "lie over"), (dict(ks=(2048, 192, 64)), "lie over"), (dict(vs=(64, 192, 64)), "lie over")])
def test_write_refuses(args, word):
    lib = _lib()
    assert _write(lib, **args) == -1 and word in lib.dtb_last_error().decode()


@pytest.mark.parametrize("args,word", [
    (dict(P=24), "page size"), (dict(M=0), "table"), (dict(n=16, M=2 ** 24, P=16), "2^31"), (dict(D=80), "head_dim"), (dict(H=4), "query heads"), (dict(Hk=0), "query heads"),
    (dict(n=0), "nseg"), (dict(sq=-1), "length"), (dict(n=1, sq=2 ** 30, tq=2 ** 30), "length"), (dict(n=1, sq=2 ** 29, tq=2 ** 29), "rows"), (dict(q=None), "null"),
    (dict(table=None), "null"), (dict(lens=None), "null"), (dict(lse=None), "null"), (dict(kp=None), "null"), (dict(tq=21), "total"), (dict(left=-2), "window"), (dict(right=2 ** 30 + 1), "window"),
    (dict(sinks=-1), "sinks"), (dict(qt=128), "stride"), (dict(qb=128), "stride"), (dict(qt=388), "multiples of 8"), (dict(q=24), "aligned"), (dict(vp=24), "aligned"),
    (dict(ks=(4096, 192, 60)), "multiples of 8"), (dict(vs=(4096, 128, 64)), "lie over"), (dict(odt=2), "out_dtype"), (dict(lay=2), "lse_layout"), (dict(acc=1, odt=1), "accumulate"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scratch=24), "scratch")])
def test_flash_refuses(args, word):
    lib = _lib()
    assert _flash(lib, **args) == -1 and word in lib.dtb_last_error().decode()


@pytest.mark.parametrize("args,word", [((0, 9, 9, 9, 2, 2, 64), "nseg"), ((1, -1, 9, 9, 2, 2, 64), "length"), ((1, 9, 9, 9, 3, 2, 64), "heads"), ((1, 9, 9, 9, 2, 2, 32), "head_dim")])
def test_flash_scratch_refuses(args, word):
    lib = _lib()
    assert lib.dtb_flash_paged_scratch_bytes(*args) == -1 and word in lib.dtb_last_error().decode()


def test_tensors_on_the_cpu_and_of_other_types_are_refused():
    from ditango_b200 import ops
    from ditango_b200._capi import ExtensionError
    i = torch.zeros(2, dtype=torch.int32)
    one, table, pages = i[:1], torch.zeros(2, 4, dtype=torch.int32), torch.zeros(8, 16, 3, 64, dtype=torch.bfloat16)
    k, q = torch.zeros(5, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.extend_pages(table, i, i, i, one, 16, 5), lambda: ops.extend_pages(table.long(), i, i, i, one, 16, 5),
                 lambda: ops.extend_pages(table, one, i, i, one, 16, 5), lambda: ops.extend_pages(table, i, i, i, i, 16, 5),
                 lambda: ops.extend_pages(table, i, i, i, one, 2 ** 40, 5), lambda: ops.extend_pages(table, i, i, i, one, 16, -1),
                 lambda: ops.extend_pages(table.t(), i, i, i, one, 16, 5),
                 lambda: ops.release_pages(table, i, i, one, i, i, 16), lambda: ops.release_pages(table, i, i, one, i, i, 16, out_table=table[:1]),
                 lambda: ops.release_pages(table, i, i, one, i, one, 16),
                 lambda: ops.write_pages(k, k, pages, pages, torch.zeros(5, dtype=torch.int32)), lambda: ops.flash_paged(q, pages, pages, table, i)):
        with pytest.raises(ExtensionError):
            call()


@pytest.mark.parametrize("args", [dict(page_size=24), dict(page_size=8), dict(layers=0), dict(head_dim=96), dict(left=-2), dict(sinks=-1), dict(max_tokens=0),
                                  dict(page_size=1 << 21), dict(max_tokens=(1 << 30) - 3), dict(streams=16385), dict(streams=9, max_tokens=1 << 28),
                                  dict(num_pages=1 << 27), dict(left=(1 << 30) + 1)])
def test_stream_cache_refuses(args):
    from ditango_b200.core.stream_cache import StreamCache
    with pytest.raises(ValueError):
        StreamCache(**{**dict(layers=1, streams=1, num_pages=1, kv_heads=1, head_dim=64, max_tokens=10, device="cpu"), **args})


def test_stream_cache_has_no_fallback():
    from ditango_b200._capi import ExtensionError
    from ditango_b200.core.stream_cache import StreamCache
    with pytest.raises(ExtensionError):
        StreamCache(1, 1, 1, 1, 64, 10, device="cpu")
