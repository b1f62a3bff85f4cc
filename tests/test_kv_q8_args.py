"""Refusals of the 8-bit KV cache operators: every check runs on the host before anything is launched, so that no GPU
(and no device memory: the addresses here are never read) is needed."""
import ctypes

import pytest

from llm_simple_b200 import ops

A = 1 << 20                     # some 16-byte aligned address
E_INVALID, E_UNSUPPORTED, E_WORKSPACE = -1, -2, -3


def _desc(batch=2, H=8, kvH=2, cap=256, layout="head", dt=5):
    return ops.make_desc(dt, batch, H, kvH, 1, cap, layout=layout)


def _kv(max_pos=256, outer=512, head=256, **kw):
    kv = ops.KvQ8()
    kv.k = kv.v = kv.k_exp = kv.v_exp = A
    kv.exp_outer_stride, kv.exp_head_stride, kv.max_pos = outer, head, max_pos
    for k, v in kw.items():
        setattr(kv, k, v)
    return kv


def _pages(size=64, table_stride=4, page_stride=2 * 64 * 128, n_pages=9, table=A):
    pg = ops.KvPages()
    pg.page_table, pg.table_stride, pg.page_size, pg.page_stride, pg.n_pages = table, table_stride, size, page_stride, n_pages
    return pg


def _r(x):
    return None if x is None else ctypes.byref(x)


def _append(d, pg, kv, q_out=A, q=A, k=A, v=A, f=A, tok=A, pos=A, total=5):
    return ops.lib().gpu_rope_kv_append_q8_layer(_r(d), _r(pg), _r(kv), q_out, q, k, v, f, tok, pos, total, None)


def _read(d, pg, kv, k=A, v=A, tok=A, pos=None, total=5):
    return ops.lib().gpu_kv_read_q8_layer(_r(d), _r(pg), _r(kv), k, v, tok, pos, total, None)


def _decode(d, pg, kv, out=A, q=A, lens=A, mx=256, window=0, sink=0, ws=A, n=1 << 30):
    return ops.lib().gpu_attn_decode_q8_layer(_r(d), _r(pg), _r(kv), out, q, lens, mx, window, sink, ws, n, None)


def _chunk(d, pg, kv, out=A, q=A, tok=A, pos=A, total=5, new=3, mx=256, window=0, sink=0, ws=A, n=1 << 30):
    return ops.lib().gpu_attn_chunk_q8_layer(_r(d), _r(pg), _r(kv), out, q, tok, pos, total, new, mx, window, sink, ws, n, None)


EVERY = [_append, _read, _decode, _chunk]


def _refused(rc, code, text):
    assert rc == code, (rc, ops.last_error_string())
    assert text in ops.last_error_string()


@pytest.mark.parametrize("call", EVERY)
def test_geometry(call):
    _refused(call(None, None, _kv()), E_INVALID, "desc")
    _refused(call(_desc(), None, None), E_INVALID, "kv is NULL")
    _refused(call(_desc(dt=6), None, _kv()), E_UNSUPPORTED, "dtype")
    d = _desc()
    d.head_dim = 64
    _refused(call(d, None, _kv()), E_UNSUPPORTED, "head_dim")
    for field, value in (("batch", 0), ("n_heads", 7), ("n_kv_heads", 0)):
        d = _desc()
        setattr(d, field, value)
        _refused(call(d, None, _kv()), E_INVALID, "n_heads")


@pytest.mark.parametrize("call", EVERY)
def test_cache(call):
    for name in ("k", "v", "k_exp", "v_exp"):
        _refused(call(_desc(), None, _kv(**{name: None})), E_INVALID, "null cache")
        _refused(call(_desc(), None, _kv(**{name: A + 8})), E_INVALID, "16-byte")
    _refused(call(_desc(), None, _kv(max_pos=0)), E_INVALID, "max_pos")
    _refused(call(_desc(), None, _kv(max_pos=257, head=272, outer=544)), E_INVALID, "do not fit the cache")
    _refused(call(_desc(), None, _kv(head=240)), E_INVALID, "exponent strides")
    _refused(call(_desc(), None, _kv(head=264)), E_INVALID, "multiples of 16")
    _refused(call(_desc(), None, _kv(outer=496)), E_INVALID, "exponent rows")
    one = _desc(batch=1)                                          # one sequence: its positions must not run into the next head
    _refused(call(one, None, _kv(max_pos=257, head=272)), E_INVALID, "do not fit the cache")
    _refused(call(_desc(batch=1, layout="token", H=8, kvH=2, cap=256), None, _kv(max_pos=0)), E_INVALID, "max_pos")
    d = _desc(layout="token")
    d.cache_head_stride = 256                                     # two heads of 128 bytes in a position of 256
    _refused(call(d, None, _kv()), E_INVALID, "do not fit the cache")
    d = _desc(layout="token")
    d.cache_pos_stride = 512                                      # positions twice as far apart, sequences not
    _refused(call(d, None, _kv()), E_INVALID, "do not fit the cache")
    for field, value in (("cache_pos_stride", 136), ("cache_head_stride", 256 * 128 + 8), ("cache_seq_stride", 2 * 256 * 128 + 8)):
        d = _desc()
        setattr(d, field, value)
        _refused(call(d, None, _kv()), E_INVALID, "multiples of 16")
    for field, value in (("cache_pos_stride", 112), ("cache_head_stride", -256 * 128), ("cache_seq_stride", 0)):
        d = _desc()
        setattr(d, field, value)
        _refused(call(d, None, _kv()), E_INVALID, "cache strides")


@pytest.mark.parametrize("call", EVERY)
def test_pages(call):
    d = _desc(cap=64)
    kv = _kv(head=64, outer=128)
    _refused(call(d, _pages(table=None), kv), E_INVALID, "page table")
    for size in (32, 48, 96):
        _refused(call(d, _pages(size=size), kv), E_UNSUPPORTED, "page size")
    _refused(call(d, _pages(table_stride=3), kv), E_INVALID, "page table rows")
    _refused(call(d, _pages(n_pages=0), kv), E_INVALID, "pages 0")
    _refused(call(d, _pages(page_stride=2 * 64 * 128 - 16), kv), E_INVALID, "do not fit the cache")
    _refused(call(d, _pages(), _kv(head=48, outer=128)), E_INVALID, "exponent strides")


def test_append_and_read():
    for name in ("k", "v", "f", "tok", "pos", "q"):
        _refused(_append(_desc(), None, _kv(), **{name: None}), E_INVALID, "null")
    for name in ("k", "v", "f", "q", "q_out"):
        _refused(_append(_desc(), None, _kv(), **{name: A + 8}), E_INVALID, "16-byte")
    _refused(_append(_desc(), None, _kv(), total=-1), E_INVALID, "total_tokens")
    _refused(_read(_desc(), None, _kv(), total=-1), E_INVALID, "total_tokens")
    _refused(_read(_desc(), None, _kv(), tok=None), E_INVALID, "tok_start")
    _refused(_read(_desc(), None, _kv(), k=None, v=None), E_INVALID, "no output")
    d = _desc()
    d.kv_in_tok_stride = 2 * 128 - 8
    _refused(_append(d, None, _kv()), E_INVALID, "kv_in_tok_stride")
    _refused(_read(d, None, _kv()), E_INVALID, "kv_in_tok_stride")
    d = _desc()
    d.q_tok_stride = 8 * 128 + 4
    _refused(_append(d, None, _kv()), E_INVALID, "q_tok_stride")
    assert _append(_desc(), None, _kv(), total=0) == 0 and _read(_desc(), None, _kv(), total=0) == 0    # nothing to do


@pytest.mark.parametrize("call", [_decode, _chunk])
def test_attention(call):
    _refused(call(_desc(), None, _kv(), out=None), E_INVALID, "null")
    _refused(call(_desc(), None, _kv(), q=None), E_INVALID, "null")
    _refused(call(_desc(), None, _kv(), q=A + 4), E_INVALID, "16-byte")
    _refused(call(_desc(), None, _kv(), window=-1), E_INVALID, "window")
    _refused(call(_desc(), None, _kv(), sink=-1), E_INVALID, "n_sink")
    _refused(call(_desc(), None, _kv(), mx=0), E_INVALID, "max_kv_len")
    _refused(call(_desc(H=34, kvH=2), None, _kv()), E_UNSUPPORTED, "group size")
    for field in ("q_seq_stride", "out_seq_stride") if call is _decode else ("q_tok_stride", "out_tok_stride"):
        d = _desc()
        setattr(d, field, 8 * 128 - 8)
        _refused(call(d, None, _kv()), E_INVALID, field)
    if call is _chunk:
        _refused(_chunk(_desc(), None, _kv(), pos=None), E_INVALID, "start_pos")
        _refused(_chunk(_desc(), None, _kv(), new=0), E_INVALID, "max_new")
        assert _chunk(_desc(), None, _kv(), total=0) == 0
        _refused(_chunk(_desc(batch=16001), None, _kv(), new=5), E_UNSUPPORTED, "at most 16000")
    else:
        _refused(_decode(_desc(), None, _kv(), lens=None), E_INVALID, "kv_len")


def test_workspace():
    need = ops.gpu_attn_decode_q8_workspace_bytes(_desc(), 256)
    assert need > 0
    _refused(_decode(_desc(), None, _kv(), ws=None), E_WORKSPACE, "workspace")
    _refused(_decode(_desc(), None, _kv(), n=need - 1), E_WORKSPACE, "%d needed" % need)
    _refused(_decode(_desc(), None, _kv(), ws=A + 8), E_INVALID, "workspace must be")
    need = ops.gpu_attn_chunk_q8_workspace_bytes(_desc(), 5, 3, 256)
    _refused(_chunk(_desc(), None, _kv(), n=need - 1), E_WORKSPACE, "%d needed" % need)
    for bad in ((None, 256), (_desc(), 0)):
        assert ops.lib().gpu_attn_decode_q8_workspace_bytes(_r(bad[0]), bad[1]) == 0


def test_struct_matches_the_header_layout():
    assert ctypes.sizeof(ops.KvQ8) == 4 * 8 + 2 * 8 + 2 * 4
    assert ops.KvQ8.exp_outer_stride.offset == 32 and ops.KvQ8.max_pos.offset == 48
