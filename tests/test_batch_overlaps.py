"""CPU: the int8 and batched decode calls refuse memory that one part of a call writes and another one uses,
wherever in the call the two are."""
import numpy as np
import pytest

from sf37_b200 import _lib

EINVAL = 1
P = 1 << 24  # addresses that no refused call touches, farther apart than the caches are long


def _refused(rc, word):
    assert rc == EINVAL and word in _lib.last_error(), (rc, _lib.last_error())


# ------------------------------------------------------------ read back
ROW = 8 * 128 * 2  # bytes of a destination row: 8 heads in f16


def _read(n):
    d = np.zeros(n, _lib.READ_I8_LAYER)
    i = np.arange(n, dtype=np.uint64)
    d["src_k_cache"], d["src_v_cache"] = P * (4 * i + 1), P * (4 * i + 2)
    d["dst_k_cache"], d["dst_v_cache"] = P * (4 * i + 3), P * (4 * i + 4)
    d["src_cap"], d["dst_cap"], d["rows"] = 16, 16, 4
    return d


def _read_call(d):
    return _lib.lib().sf37kv_read_i8(d.ctypes.data, len(d), 8, 128, 2, None)


@pytest.mark.parametrize("n,a,b", [(2, 0, 1), (3, 2, 0), (100, 1, 99)])
def test_read_refuses_one_destination_twice(n, a, b):
    for x, y in (("dst_k_cache", "dst_k_cache"), ("dst_v_cache", "dst_v_cache"), ("dst_k_cache", "dst_v_cache")):
        d = _read(n)
        d[x][b] = d[y][a]
        _refused(_read_call(d), "another")
        d[x][b] += 3 * ROW  # the last of the four rows
        _refused(_read_call(d), "another")


@pytest.mark.parametrize("n,a,b", [(2, 0, 1), (2, 1, 0), (100, 99, 1)])
def test_read_refuses_a_destination_that_is_another_layers_source(n, a, b):
    for x, y in (("src_k_cache", "dst_k_cache"), ("src_v_cache", "dst_k_cache")):
        d = _read(n)
        d[x][b] = d[y][a]
        _refused(_read_call(d), "another")


def test_read_refuses_rows_that_meet_past_a_rings_end():
    d = _read(2)
    d["dst_k_cache"][1], d["dst_v_cache"][1] = d["dst_k_cache"][0], d["dst_v_cache"][0]
    d["first_pos"] = [14, 17]  # slots 14, 15, 0, 1 and 1 to 4
    _refused(_read_call(d), "another")


def test_read_refuses_k_and_v_that_overlap():
    d = _read(1)
    d["dst_v_cache"] = d["dst_k_cache"] + 2 * ROW
    _refused(_read_call(d), "another")


# ------------------------------------------------------------ append
def _append(n):
    d = np.zeros(n, _lib.APPEND_I8_LAYER)
    i = np.arange(n, dtype=np.uint64)
    d["k_cache"], d["v_cache"] = P * (2 * i + 1), P * (2 * i + 2)
    d["cap"], d["n_tok"], d["k"], d["v"] = 16, 4, P, P
    return d


@pytest.mark.parametrize("n,a,b", [(2, 0, 1), (65, 0, 64), (200, 3, 199)])
def test_append_refuses_one_cache_twice(n, a, b):
    for x, y in (("k_cache", "k_cache"), ("v_cache", "v_cache"), ("k_cache", "v_cache")):
        d = _append(n)
        d[x][b] = d[y][a]
        _refused(_lib.lib().sf37kv_append_i8(d.ctypes.data, n, 8, 128, 0, None), "twice")
        d[x][b] += 16 * 8 * 132 - 32  # the last scales
        _refused(_lib.lib().sf37kv_append_i8(d.ctypes.data, n, 8, 128, 0, None), "twice")


# ------------------------------------------------------------ decode
def _seqs(n):
    d = np.zeros(n, _lib.DECODE_SEQ)
    i = np.arange(n, dtype=np.uint64)
    d["k_cache"], d["v_cache"] = P * (2 * i + 1), P * (2 * i + 2)
    d["cap"], d["pos"], d["q"], d["out"] = 64, 20, P, P
    return d


def _decode(d):
    return _lib.lib().sf37kv_decode_i8(d.ctypes.data, len(d), 64, 8, 128, 0, P, 1 << 40, None)


def _shared(arrays, prefix_len=0, dtype=2):
    g = np.zeros(len(arrays), _lib.SHARED_GROUP)
    for i, d in enumerate(arrays):
        g[i] = (P * (10001 + 2 * i), P * (10002 + 2 * i), 32, 0, 0, 0, prefix_len, len(d), d.ctypes.data)
    return _lib.lib().sf37kv_decode_shared(g.ctypes.data, len(g), 64, 8, 128, dtype, 0, P, 1 << 40, None)


@pytest.mark.parametrize("n,a,b", [(2, 0, 1), (2, 1, 0), (257, 0, 256), (600, 599, 1)])
def test_decode_refuses_an_appended_cache_that_is_anothers(n, a, b):
    for x, y in (("k_cache", "k_cache"), ("v_cache", "v_cache"), ("k_cache", "v_cache")):
        for off in (0, 63 * 8 * 128 - 32):  # the same cache, or one that begins in its last codes
            d = _seqs(n)
            d["k_new"][a] = d["v_new"][a] = P
            d[x][b] = d[y][a] + off
            _refused(_decode(d), "twice")
            _refused(_shared([d]), "twice")
            _refused(_shared([d], dtype=1), "twice")


def test_shared_refuses_an_appended_cache_of_another_groups_sequence():
    one, two = _seqs(300), _seqs(300)
    for c in ("k_cache", "v_cache"):
        two[c] += 5000 * P
    one["k_new"][0] = one["v_new"][0] = P
    two["v_cache"][299] = one["v_cache"][0]
    _refused(_shared([one, two]), "twice")


@pytest.mark.parametrize("dtype,row", [(1, 132), (2, 256)])
def test_shared_refuses_an_append_to_another_groups_prefix(dtype, row):
    one, two = _seqs(3), _seqs(3)
    for c in ("k_cache", "v_cache"):
        two[c] += 5000 * P
    one["k_new"][2] = one["v_new"][2] = P
    for c in ("k_cache", "v_cache"):
        for prefix in (P * 10003, P * 10004):  # K and V of the second group's prefix of 8 rows
            keep = one[c][2]
            for at in (prefix, prefix + 7 * 8 * 256, prefix - 64 * 8 * row + 32):
                one[c][2] = at
                _refused(_shared([one, two], 8, dtype), "prefix")
            one[c][2] = keep
