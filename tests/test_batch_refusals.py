"""CPU: the int8 cache and batched decode calls refuse bad arguments with a
code and a message, before anything is launched."""
import numpy as np
import pytest

from sf37_b200 import _lib

EINVAL, EUNSUPPORTED = 1, 4
P = 1 << 20  # addresses that no refused call touches


def _append(n=1):
    d = np.zeros(n, _lib.APPEND_I8_LAYER)
    for i in range(n):
        d[i] = (P * (2 * i + 1), P * (2 * i + 2), 16, 0, 0, 0, 0, 4, P, P)
    return d


def _read(n=1):
    d = np.zeros(n, _lib.READ_I8_LAYER)
    for i in range(n):
        d[i] = (P, 2 * P, 16, 0, 0, 0, 3 * P, 4 * P, 16, 0, 0, 0, 0, 4)
    return d


def _seqs(n=1):
    d = np.zeros(n, _lib.DECODE_SEQ)
    for i in range(n):
        d[i] = (P * (2 * i + 1), P * (2 * i + 2), 64, 0, 0, 0, 20, 0, P, 0, P, 0, 0)
    return d


def _groups(seqs, prefix_len=8):
    d = np.zeros(1, _lib.SHARED_GROUP)
    d[0] = (100 * P, 101 * P, 32, 0, 0, 0, prefix_len, len(seqs), seqs.ctypes.data)
    return d


def _refused(rc, code, word):
    assert rc == code and word in _lib.last_error(), (rc, _lib.last_error())


def test_record_sizes_match_the_c_structs():
    assert _lib.APPEND_I8_LAYER.itemsize == 56 and _lib.READ_I8_LAYER.itemsize == 72
    assert _lib.DECODE_SEQ.itemsize == 80 and _lib.SHARED_GROUP.itemsize == 48


def test_sizes():
    L = _lib.lib()
    assert L.sf37kv_i8_cache_bytes(2049, 8, 128) == 2049 * 8 * 132 + (-2049 * 8 * 132) % 256
    assert L.sf37kv_i8_cache_bytes(1 << 30, 8, 128) == (1 << 30) * 8 * 132
    assert L.sf37kv_i8_cache_bytes(16, 8, 64) == 0
    small = L.sf37kv_decode_i8_workspace(1, 64, 8)
    assert 0 < small <= L.sf37kv_decode_i8_workspace(200, 64, 8) < 64 << 20
    assert L.sf37kv_decode_i8_workspace(1 << 20, 64, 8) == L.sf37kv_decode_i8_workspace(1 << 30, 64, 8)
    assert L.sf37kv_decode_shared_workspace(1, 64, 64, 8) > L.sf37kv_decode_i8_workspace(64, 64, 8)
    assert L.sf37kv_decode_i8_workspace(1, 65, 8) == 0 and L.sf37kv_decode_shared_workspace(1, 1, 64, 0) == 0


@pytest.mark.parametrize("field,value,word", [("k_cache", 0, "cache 0"), ("v_cache", P + 8, "aligned"),
                                              ("cap", 0, "cap"), ("cap", 1 << 31, "cap"), ("k", 0, "rows"),
                                              ("v", P + 4, "aligned"), ("pos0", (1 << 31) - 2, "positions"),
                                              ("v_cache", P, "one buffer")])
def test_append_refuses(field, value, word):
    d = _append()
    d[field] = value
    _refused(_lib.lib().sf37kv_append_i8(d.ctypes.data, 1, 8, 128, 0, None), EINVAL, word)


def test_append_refuses_calls():
    L, d = _lib.lib(), _append(3)
    _refused(L.sf37kv_append_i8(None, 1, 8, 128, 0, None), EINVAL, "NULL")
    _refused(L.sf37kv_append_i8(d.ctypes.data, 1, 8, 64, 0, None), EUNSUPPORTED, "head_dim")
    _refused(L.sf37kv_append_i8(d.ctypes.data, 1, 0, 128, 0, None), EINVAL, "KV heads")
    _refused(L.sf37kv_append_i8(d.ctypes.data, 1, 8, 128, 2, None), EINVAL, "row type")
    d[2]["k_cache"] = d[0]["k_cache"]
    _refused(L.sf37kv_append_i8(d.ctypes.data, 3, 8, 128, 0, None), EINVAL, "twice")
    big = _append()
    big["cap"] = big["n_tok"] = (1 << 31) - 2
    _refused(L.sf37kv_append_i8(big.ctypes.data, 1, 8, 128, 0, None), EINVAL, "too many rows")
    assert L.sf37kv_append_i8(None, 0, 8, 128, 0, None) == 0  # nothing to do


@pytest.mark.parametrize("field,value,word", [("src_k_cache", 0, "cache 0"), ("dst_v_cache", 4, "aligned"),
                                              ("rows", 17, "17 rows"), ("dst_cap", 3, "4 rows"),
                                              ("first_pos", (1 << 31) - 2, "positions"), ("dst_k_cache", P, "same cache"),
                                              ("dst_v_cache", P, "same cache")])
def test_read_refuses(field, value, word):
    d = _read()
    d[field] = value
    _refused(_lib.lib().sf37kv_read_i8(d.ctypes.data, 1, 8, 128, 2, None), EINVAL, word)


def test_read_refuses_calls():
    L, d = _lib.lib(), _read()
    _refused(L.sf37kv_read_i8(None, 1, 8, 128, 2, None), EINVAL, "NULL")
    _refused(L.sf37kv_read_i8(d.ctypes.data, 1, 8, 128, 1, None), EINVAL, "dtype")
    _refused(L.sf37kv_read_i8(d.ctypes.data, 1, 8, 256, 2, None), EUNSUPPORTED, "head_dim")


@pytest.mark.parametrize("field,value,word", [("q", 0, "q and out"), ("out", P + 8, "aligned"), ("cap", 0, "cap"),
                                              ("k_new", P, "only one"), ("gate", 2, "gate"),
                                              ("pos", (1 << 31) - 1, "position")])
def test_decode_refuses(field, value, word):
    L, d = _lib.lib(), _seqs()
    d[field] = value
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 1, 64, 8, 128, 0, P, 1 << 40, None), EINVAL, word)
    g = _groups(d)
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, P, 1 << 40, None), EINVAL, word)


def test_decode_refuses_calls():
    L, d = _lib.lib(), _seqs(3)
    a = (P, 1 << 40, None)
    _refused(L.sf37kv_decode_i8(None, 1, 64, 8, 128, 0, *a), EINVAL, "NULL")
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 1, 60, 8, 128, 0, *a), EINVAL, "divide")
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 1, 64, 8, 64, 0, *a), EUNSUPPORTED, "head_dim")
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 1, 136, 8, 128, 0, *a), EUNSUPPORTED, "16 query heads")
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 1, 64, 8, 128, 2, *a), EINVAL, "io type")
    need = L.sf37kv_decode_i8_workspace(3, 64, 8)
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 3, 64, 8, 128, 0, None, need, None), EINVAL, "workspace")
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 3, 64, 8, 128, 0, P + 16, need, None), EINVAL, "workspace")
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 3, 64, 8, 128, 0, P, need - 1, None), EINVAL, "workspace")
    d["k_new"][1] = d["v_new"][1] = P
    d["sliding"][1] = 1
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 3, 64, 8, 128, 0, P, need, None), EINVAL, "window of no rows")
    d["sliding"][1] = 0
    d["k_cache"][2] = d["k_cache"][1]
    _refused(L.sf37kv_decode_i8(d.ctypes.data, 3, 64, 8, 128, 0, P, need, None), EINVAL, "twice")
    assert L.sf37kv_decode_i8(None, 0, 64, 8, 128, 0, None, 0, None) == 0


def test_shared_refuses_calls():
    L, d = _lib.lib(), _seqs(2)
    a = (P, 1 << 40, None)
    g = _groups(d)
    _refused(L.sf37kv_decode_shared(None, 1, 64, 8, 128, 2, 0, *a), EINVAL, "NULL")
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 4, 0, *a), EUNSUPPORTED, "dtype")
    g["prefix_len"] = 33
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "exceeds its cache")
    g["prefix_len"] = 8
    g["prefix_k_cache"] = 0
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "cache 0")
    g = _groups(d)
    g["seqs"] = 0
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "sequences")
    g = _groups(d)
    d["pos"][1] = 6
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "inside the prefix")
    d["pos"][1] = 7
    d["k_new"][1] = d["v_new"][1] = P
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "the prefix's")
    d["pos"][1] = 8 + 64  # 65 own rows in a cache of 64
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "own rows")
    d["pos"][1] = 20
    d["k_cache"][1] = 100 * P
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "prefix's cache")
    d["k_cache"][1] = d["k_cache"][0]
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, *a), EINVAL, "twice")
    d["k_cache"][1] = 50 * P
    need = L.sf37kv_decode_shared_workspace(1, 2, 64, 8)
    _refused(L.sf37kv_decode_shared(g.ctypes.data, 1, 64, 8, 128, 2, 0, P, need - 1, None), EINVAL, "workspace")
    empty = _groups(d)
    empty["n_seqs"] = 0
    assert L.sf37kv_decode_shared(empty.ctypes.data, 1, 64, 8, 128, 2, 0, None, 0, None) == 0


def test_other_calls_still_refuse_the_i8_dtype():
    L = _lib.lib()
    lay = (_lib.DecodeLayer * 1)()
    lay[0].cache.cap = 16
    lay[0].cache.k_cache = lay[0].cache.v_cache = lay[0].q = lay[0].out = P
    assert L.sf37kv_decode(lay, 1, 8, 2, 128, 1, None) == EINVAL
    ap = (_lib.AppendLayer * 1)()
    ap[0].cache.cap = ap[0].n_tok = 1
    ap[0].cache.k_cache = ap[0].cache.v_cache = ap[0].k = ap[0].v = P
    assert L.sf37kv_append(ap, 1, 1024, 1, None) == EINVAL
