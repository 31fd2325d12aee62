"""Torch-facing mirror of the KV-cache C ABI.

torch supplies device memory and streams only; every computation runs in
libsf37kv.so.  Function names and argument meaning follow the reference's
``sf37_cuda.h`` entry points (drop-in layer, fp32 caches, return True/False
like the reference's int 1/0) and ``include/sf37kv.h`` (native layer, raises
on error).
"""
import ctypes

import numpy as np
import torch

from ._lib import (APPEND_I8_LAYER, DECODE_SEQ, READ_I8_LAYER, SHARED_GROUP, AppendLayer, Cache, DecodeLayer, PackLayer,
                   Tensor, check, lib)

I8, F16, F32 = 1, 2, 4
Q_F32, Q_BF16 = 0, 1
FMT_RAW, FMT_I8G = 0, 1
_DT = {torch.float16: F16, torch.float32: F32}


def view(t):
    """sf37_cuda_tensor view {ptr, bytes} of a torch CUDA tensor (None -> NULL)."""
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous()
    return ctypes.byref(Tensor(t.data_ptr(), t.numel() * t.element_size()))


def _sp(stream):
    if stream is None:
        return None
    return ctypes.c_void_p(stream.cuda_stream)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------- drop-in layer
def store_kv_cache_batch(k_cache, v_cache, k, v, pos0, n_tok, cache_cap, kv_dim) -> bool:
    return bool(lib().sf37_cuda_store_kv_cache_batch(view(k_cache), view(v_cache), view(k), view(v),
                                                     pos0, n_tok, cache_cap, kv_dim))


def attention_decode_heads(out, q, k_cache, v_cache, gate, n_cache, cache_cap, q_heads, kv_heads,
                           head_dim, sliding, window) -> bool:
    return bool(lib().sf37_cuda_attention_decode_heads(view(out), view(q), view(k_cache),
                                                       view(v_cache), view(gate), n_cache,
                                                       cache_cap, q_heads, kv_heads, head_dim,
                                                       int(sliding), window))


def attention_decode_heads_at(out, q, k_cache, v_cache, gate, pos, cache_cap, q_heads, kv_heads,
                              head_dim, sliding, window) -> bool:
    return bool(lib().sf37_cuda_attention_decode_heads_at(view(out), view(q), view(k_cache),
                                                          view(v_cache), view(gate), pos, cache_cap,
                                                          q_heads, kv_heads, head_dim, int(sliding),
                                                          window))


def attention_prefill_heads(out, q, k_cache, v_cache, gate, pos0, n_tok, cache_cap, q_heads,
                            kv_heads, head_dim, sliding, window) -> bool:
    return bool(lib().sf37_cuda_attention_prefill_heads(view(out), view(q), view(k_cache),
                                                        view(v_cache), view(gate), pos0, n_tok,
                                                        cache_cap, q_heads, kv_heads, head_dim,
                                                        int(sliding), window))


def gqa_single_token_heads(out, v, gate, q_heads, kv_heads, head_dim) -> bool:
    return bool(lib().sf37_cuda_gqa_single_token_heads(view(out), view(v), view(gate), q_heads,
                                                       kv_heads, head_dim))


def kv_pack_rows(host_dst, k_cache, v_cache, first_pos, rows, cache_cap, kv_dim, fmt=FMT_RAW,
                 group=64, variant=1) -> bool:
    """sf37_cuda_kv_pack_rows_{f32,i8g}; host_dst: a writable numpy array."""
    p = host_dst.ctypes.data
    if fmt == FMT_RAW:
        return bool(lib().sf37_cuda_kv_pack_rows_f32(p, view(k_cache), view(v_cache), first_pos,
                                                     rows, cache_cap, kv_dim))
    return bool(lib().sf37_cuda_kv_pack_rows_i8g(p, view(k_cache), view(v_cache), first_pos, rows,
                                                 cache_cap, kv_dim, group, variant))


def kv_unpack_rows(host_src, k_cache, v_cache, first_pos, rows, cache_cap, kv_dim, fmt=FMT_RAW,
                   group=64) -> bool:
    p = host_src.ctypes.data
    if fmt == FMT_RAW:
        return bool(lib().sf37_cuda_kv_unpack_rows_f32(p, view(k_cache), view(v_cache), first_pos,
                                                       rows, cache_cap, kv_dim))
    return bool(lib().sf37_cuda_kv_unpack_rows_i8g(p, view(k_cache), view(v_cache), first_pos, rows,
                                                   cache_cap, kv_dim, group))


# ------------------------------------------------------------- native layer
def cache_desc(k_cache, v_cache, cap, sliding=False, window=512):
    return Cache(k_cache.data_ptr(), v_cache.data_ptr(), cap, int(bool(sliding)), window, 0)


def decode_layers_desc(layers):
    """layers: list of dicts with k_cache, v_cache, cap, sliding, window, pos, q, gate, out,
    k_new, v_new (tensors or None).  Returns a ctypes array (reusable)."""
    arr = (DecodeLayer * len(layers))()
    for i, L in enumerate(layers):
        arr[i] = DecodeLayer(cache_desc(L["k_cache"], L["v_cache"], L["cap"], L.get("sliding", 0),
                                        L.get("window", 512)), L["pos"], 0, _ptr(L["q"]),
                             _ptr(L.get("gate")), _ptr(L.get("out")), _ptr(L.get("k_new")),
                             _ptr(L.get("v_new")))
    return arr


def decode(layers, q_heads, kv_heads, head_dim, dtype, stream=None):
    arr = layers if not isinstance(layers, list) else decode_layers_desc(layers)
    check(lib().sf37kv_decode(arr, len(arr), q_heads, kv_heads, head_dim, dtype, _sp(stream)),
          "sf37kv_decode")


def qk_prep_desc(preps):
    """preps: list of dicts q_norm, k_norm (bf16 tensors as int16/uint16/bfloat16),
    rotary_dim, theta, llama3, eps.  Returns a ctypes array (reusable)."""
    from ._lib import QkPrep
    arr = (QkPrep * len(preps))()
    for i, p in enumerate(preps):
        arr[i] = QkPrep(_ptr(p["q_norm"]), _ptr(p.get("k_norm")), float(p["theta"]), int(p["rotary_dim"]),
                        int(p.get("llama3", 0)), float(p.get("eps", 1e-5)), 0)
    return arr


def decode_prep(layers, preps, q_heads, kv_heads, head_dim, dtype, stream=None):
    """sf37kv_decode with the q / k_new heads normalized and rotated in the kernel."""
    arr = layers if not isinstance(layers, list) else decode_layers_desc(layers)
    pa = preps if not isinstance(preps, list) else qk_prep_desc(preps)
    check(lib().sf37kv_decode_prep(arr, pa, len(arr), q_heads, kv_heads, head_dim, dtype, _sp(stream)),
          "sf37kv_decode_prep")


def append(layers, kv_dim, dtype, stream=None):
    arr = (AppendLayer * len(layers))()
    for i, L in enumerate(layers):
        arr[i] = AppendLayer(cache_desc(L["k_cache"], L["v_cache"], L["cap"]), L["pos0"], L["n_tok"],
                             _ptr(L["k"]), _ptr(L["v"]))
    check(lib().sf37kv_append(arr, len(arr), kv_dim, dtype, _sp(stream)), "sf37kv_append")


def prefill(k_cache, v_cache, cap, q, gate, out, pos0, n_tok, q_heads, kv_heads, head_dim, dtype,
            sliding=False, window=512, stream=None):
    c = cache_desc(k_cache, v_cache, cap, sliding, window)
    qt = Q_BF16 if q.dtype == torch.bfloat16 else Q_F32
    check(lib().sf37kv_prefill(ctypes.byref(c), _ptr(q), qt, _ptr(gate), _ptr(out), pos0, n_tok,
                               q_heads, kv_heads, head_dim, dtype, _sp(stream)), "sf37kv_prefill")


def row_bytes(kv_dim, fmt, group=64) -> int:
    return int(lib().sf37kv_row_bytes(kv_dim, fmt, group))


def pack_layers_desc(layers, kv_dim, fmt, group=64):
    """layers: list of dicts with k_cache, v_cache, cap, first_pos, rows.  Sections are laid
    out back to back; returns (ctypes array, total bytes)."""
    arr = (PackLayer * len(layers))()
    rb = row_bytes(kv_dim, fmt, group)
    off = 0
    for i, L in enumerate(layers):
        arr[i] = PackLayer(cache_desc(L["k_cache"], L["v_cache"], L["cap"]), L["first_pos"],
                           L["rows"], off)
        off += 2 * L["rows"] * rb
    return arr, off


def pack(dst, arr, kv_dim, dtype, fmt, group=64, variant=1, stream=None):
    """dst: torch CUDA uint8 tensor (or an int device/mapped-host address)."""
    p = dst if isinstance(dst, int) else dst.data_ptr()
    check(lib().sf37kv_pack(p, arr, len(arr), kv_dim, dtype, fmt, group, variant, _sp(stream)),
          "sf37kv_pack")


def unpack(src, arr, kv_dim, dtype, fmt, group=64, stream=None):
    p = src if isinstance(src, int) else src.data_ptr()
    check(lib().sf37kv_unpack(p, arr, len(arr), kv_dim, dtype, fmt, group, _sp(stream)),
          "sf37kv_unpack")


def pack_to_host(host_ptr, arr, kv_dim, dtype, fmt, group=64, variant=1):
    check(lib().sf37kv_pack_to_host(host_ptr, arr, len(arr), kv_dim, dtype, fmt, group, variant),
          "sf37kv_pack_to_host")


def unpack_from_host(host_ptr, arr, kv_dim, dtype, fmt, group=64):
    check(lib().sf37kv_unpack_from_host(host_ptr, arr, len(arr), kv_dim, dtype, fmt, group),
          "sf37kv_unpack_from_host")


def set_stream(stream):
    lib().sf37kv_set_stream(_sp(stream))


def launch_count() -> int:
    return int(lib().sf37kv_launch_count())


def device_error(clear=False) -> int:
    """The device error flag (0 = none, 2 = a bounded wait timed out); syncs."""
    return lib().sf37kv_device_error(int(bool(clear)))


def oproj(layers, in_dim, out_dim, stream=None):
    """Q8_0 o_proj matvec of every layer in one launch (sf37kv_oproj_q8_0)."""
    check(lib().sf37kv_oproj_q8_0(layers, len(layers), in_dim, out_dim, _sp(stream)), "sf37kv_oproj_q8_0")


# ------------------------------------------- int8 caches and batched decode
# The *_desc functions fill a descriptor array once; a decode loop keeps it and
# writes what changes (``seqs["pos"] = positions``).  They take tensors with a
# leading dimension of n layers or sequences, or lists of n tensors; the tensors
# have to outlive the descriptors.
_IO = {torch.float32: Q_F32, torch.bfloat16: Q_BF16}


class Descriptors(np.ndarray):
    """Descriptor array.  `held` says what its tensors hold (so do slices' and copies'); the calls refuse, before
    anything is launched, head counts and types that do not fit them."""

    def __array_finalize__(self, source):
        self.held = getattr(source, "held", None)
        self.at = None  # this array's address, once asked for


class _Held:
    """device; kv_heads, q_heads: of the rows and queries, or None; cache_heads: the most that every cache has room
    for; dtype: of the rows, queries or destinations; cache: of the caches."""

    __slots__ = ("device", "kv_heads", "q_heads", "cache_heads", "dtype", "cache")

    def __init__(self, device, cache_heads, dtype, cache, kv_heads=None, q_heads=None):
        self.device, self.cache_heads, self.dtype, self.cache = device, cache_heads, dtype, cache
        self.kv_heads, self.q_heads = kv_heads, q_heads

    def check(self, what, device, kv_heads, dtype, cache, q_heads):
        if self.kv_heads not in (None, kv_heads) or kv_heads > self.cache_heads:
            has = f"rows of {self.kv_heads}" if self.kv_heads not in (None, kv_heads) else f"room for {self.cache_heads}"
            raise ValueError(f"{what}: kv_heads is {kv_heads}, the tensors have {has}")
        if q_heads != self.q_heads:
            raise ValueError(f"{what}: q_heads is {q_heads}, the queries have {self.q_heads}")
        if dtype is not self.dtype:
            raise ValueError(f"{what}: dtype is {dtype}, the tensors are {self.dtype}")
        if cache is not self.cache:
            raise ValueError(f"{what}: caches of {cache} are needed, the descriptors' are {self.cache}")
        if device != self.device:
            raise ValueError(f"{what}: the tensors are on CUDA device {self.device}, the current one is {device}")


def _addresses(name, x, n, dtypes=None, inner=None):
    """Addresses of the n items of a stacked tensor or a list of tensors."""
    items = [x] if isinstance(x, torch.Tensor) else list(x)
    for t in items:
        if not t.is_cuda or t.device != items[0].device or t.device.index != torch.cuda.current_device():
            raise ValueError(f"{name}: tensors on the current CUDA device are needed, got {t.device}")
        if dtypes is not None and t.dtype not in dtypes:
            raise ValueError(f"{name}: dtype {t.dtype} is not one of {dtypes}")
        if t.dtype != items[0].dtype:
            raise ValueError(f"{name}: tensors of one dtype are needed, got {items[0].dtype} and {t.dtype}")
    if isinstance(x, torch.Tensor):
        if x.dim() < 1 or x.shape[0] != n:
            raise ValueError(f"{name}: a leading dimension of {n} is needed, got shape {tuple(x.shape)}")
        items, first = [x[0]] if n else [], x.data_ptr()
        at = first + np.arange(n, dtype=np.uint64) * np.uint64(x.stride(0) * x.element_size() if n > 1 else 0)
    else:
        if len(items) != n:
            raise ValueError(f"{name}: {n} tensors are needed, got {len(items)}")
        at = np.array([t.data_ptr() for t in items], dtype=np.uint64)
    for t in items:
        if not t.is_contiguous():
            raise ValueError(f"{name}: each item has to be contiguous")
        if inner is not None and tuple(t.shape) != tuple(inner):
            raise ValueError(f"{name}: items of shape {tuple(inner)} are needed, got {tuple(t.shape)}")
    return at


def _count(x):
    return x.shape[0] if isinstance(x, torch.Tensor) else len(x)


def _item(x):
    return x[0]


def _room(name, x, cap):
    """KV heads that every cache of x has room for at its cap (an array), 128 elements (int8: 132 bytes) each."""
    one = isinstance(x, torch.Tensor)
    sizes = np.array([_item(x).numel()] if one else [t.numel() for t in x], dtype=np.int64)
    per = (132 if _item(x).dtype == torch.uint8 else 128) * np.maximum(cap.astype(np.int64), 1)
    heads = int((sizes // per).min())
    if heads < 1:
        raise ValueError(f"{name}: smaller than cap rows of one head")
    return heads


def _row_heads(name, items, rows):
    """KV heads of row tensors [rows][kv_heads][128], the same in all."""
    heads = None
    for t, r in zip(items, rows):
        if r == 0:
            continue
        h, rest = divmod(t.numel(), r * 128)
        if rest or heads not in (None, h):
            raise ValueError(f"{name}: rows of one number of heads of 128 are needed, got shape {tuple(t.shape)}")
        heads = h
    return heads


def _records(layers, dtype, name):
    """Address and length of a descriptor array."""
    if layers.dtype != dtype or layers.ndim != 1 or not layers.flags.c_contiguous:
        raise ValueError(f"a contiguous array of {name}() is needed")
    if type(layers) is not Descriptors:
        return layers.ctypes.data, len(layers)
    if layers.at is None:  # (ctypes: 1 us; __array_interface__ lists all fields first: 12)
        layers.at = layers.ctypes.data
    return layers.at, len(layers)


def _checked(layers, what, device, kv_heads, dtype, cache, q_heads):
    if type(layers) is Descriptors and layers.held is not None:  # a plain array of records is the caller's own
        layers.held.check(what, device, kv_heads, dtype, cache, q_heads)


def _space(workspace):
    """Device, address and bytes of a workspace."""
    device = workspace.get_device()  # -1 on the CPU
    if device != torch.cuda.current_device() or not workspace.is_contiguous():
        raise ValueError("workspace: a contiguous tensor on the current CUDA device is needed")
    return device, workspace.data_ptr(), workspace.nbytes


def i8_cache_bytes(cap, kv_heads, head_dim=128) -> int:
    """Bytes of one int8 cache of K (or V); allocate it as uint8 (zero-filled or not)."""
    return int(lib().sf37kv_i8_cache_bytes(cap, kv_heads, head_dim))


def append_i8_desc(k_cache, v_cache, cap, pos0, k, v):
    """k, v: [n][n_tok][kv_heads][128] f32 or bf16 (or lists of [n_tok][kv_heads][128])."""
    n, stacked = _count(k), isinstance(k, torch.Tensor)
    d = np.zeros(n, APPEND_I8_LAYER).view(Descriptors)
    d["k_cache"], d["v_cache"] = (_addresses("k_cache", k_cache, n, (torch.uint8,)),
                                  _addresses("v_cache", v_cache, n, (torch.uint8,)))
    shapes = [tuple(_item(k).shape)] if stacked else [tuple(t.shape) for t in k]
    d["cap"], d["pos0"], d["n_tok"] = cap, pos0, shapes[0][0] if stacked else [x[0] for x in shapes]
    d["k"], d["v"] = _addresses("k", k, n, tuple(_IO)), _addresses("v", v, n, (_item(k).dtype,))
    if any(tuple(a.shape) != tuple(b.shape) for a, b in ([(_item(k), _item(v))] if stacked and isinstance(v, torch.Tensor)
                                                         else zip(k, v))):
        raise ValueError("v: rows of the same shape as k's are needed")
    heads = _row_heads("k", [_item(k)] if stacked else k, [x[0] for x in shapes])
    d.held = _Held(_item(k).get_device(), min(_room("k_cache", k_cache, d["cap"]), _room("v_cache", v_cache, d["cap"])),
                   _item(k).dtype, torch.uint8, heads)
    return d


def append_i8(layers, kv_heads, head_dim, dtype, stream=None):
    """Quantises the rows of append_i8_desc() into their caches; dtype: the rows' torch dtype."""
    _checked(layers, "append_i8", torch.cuda.current_device(), kv_heads, dtype, torch.uint8, None)
    check(lib().sf37kv_append_i8(*_records(layers, APPEND_I8_LAYER, "append_i8_desc"), kv_heads, head_dim, _IO[dtype], _sp(stream)),
          "sf37kv_append_i8")


def read_i8_desc(k_cache, v_cache, cap, dst_k, dst_v, dst_cap, first_pos, rows):
    """dst_k, dst_v: f16 or f32 caches of dst_cap rows, [n][dst_cap][kv_heads][128]."""
    n = _count(dst_k)
    d = np.zeros(n, READ_I8_LAYER).view(Descriptors)
    d["src_k_cache"], d["src_v_cache"] = (_addresses("k_cache", k_cache, n, (torch.uint8,)),
                                          _addresses("v_cache", v_cache, n, (torch.uint8,)))
    d["dst_k_cache"] = _addresses("dst_k", dst_k, n, tuple(_DT))
    d["dst_v_cache"] = _addresses("dst_v", dst_v, n, (_item(dst_k).dtype,))
    d["src_cap"], d["dst_cap"], d["first_pos"], d["rows"] = cap, dst_cap, first_pos, rows
    room = min(_room(name, x, d[at]) for name, x, at in (("k_cache", k_cache, "src_cap"), ("v_cache", v_cache, "src_cap"),
                                                        ("dst_k", dst_k, "dst_cap"), ("dst_v", dst_v, "dst_cap")))
    d.held = _Held(_item(dst_k).get_device(), room, _item(dst_k).dtype, torch.uint8)
    return d


def read_i8(layers, kv_heads, head_dim, dtype, stream=None):
    """Reads the rows of read_i8_desc() back; dtype: the destinations' torch dtype."""
    _checked(layers, "read_i8", torch.cuda.current_device(), kv_heads, dtype, torch.uint8, None)
    check(lib().sf37kv_read_i8(*_records(layers, READ_I8_LAYER, "read_i8_desc"), kv_heads, head_dim, _DT[dtype], _sp(stream)),
          "sf37kv_read_i8")


def decode_seqs_desc(k_cache, v_cache, cap, pos, q, out, gate=None, k_new=None, v_new=None, sliding=False,
                     window=512):
    """q, out: [n][q_heads][128] f32 or bf16; gate: [n][q_heads] f32; k_new, v_new: [n][kv_heads][128] like q;
    caches: all uint8 (int8 caches) or all f16."""
    n = _count(q)
    d = np.zeros(n, DECODE_SEQ).view(Descriptors)
    d["k_cache"] = _addresses("k_cache", k_cache, n, (torch.uint8, torch.float16))
    d["v_cache"] = _addresses("v_cache", v_cache, n, (_item(k_cache).dtype,))
    d["cap"], d["sliding"], d["window"], d["pos"] = cap, np.asarray(sliding, dtype=bool), window, pos
    room = min(_room("k_cache", k_cache, d["cap"]), _room("v_cache", v_cache, d["cap"]))
    heads, dtype, kv_heads = _item(q).shape[0], (_item(q).dtype,), None
    d["q"], d["out"] = _addresses("q", q, n, tuple(_IO), (heads, 128)), _addresses("out", out, n, dtype, (heads, 128))
    if gate is not None:
        d["gate"] = _addresses("gate", gate, n, (torch.float32,), (heads,))
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None:
        inner = tuple(_item(k_new).shape)
        d["k_new"], d["v_new"] = _addresses("k_new", k_new, n, dtype, inner), _addresses("v_new", v_new, n, dtype, inner)
        kv_heads = _row_heads("k_new", [_item(k_new)], [1])
    d.held = _Held(_item(q).get_device(), room, dtype[0], _item(k_cache).dtype, kv_heads, heads)
    return d


def decode_i8_workspace(n_seqs, q_heads, kv_heads) -> int:
    """Bytes of a workspace for decode_i8(): allocate it zero-filled (torch.zeros, uint8)."""
    return int(lib().sf37kv_decode_i8_workspace(n_seqs, q_heads, kv_heads))


def decode_i8(seqs, q_heads, kv_heads, head_dim, dtype, workspace, stream=None):
    """One decode step over int8 caches; dtype: torch dtype of q and out."""
    device, at, size = _space(workspace)
    _checked(seqs, "decode_i8", device, kv_heads, dtype, torch.uint8, q_heads)
    check(lib().sf37kv_decode_i8(*_records(seqs, DECODE_SEQ, "decode_seqs_desc"), q_heads, kv_heads, head_dim, _IO[dtype],
                                 at, size, _sp(stream)),
          "sf37kv_decode_i8")


def shared_groups_desc(groups):
    """groups: list of dicts k_cache, v_cache (f16 [cap][kv_heads][128], or None), prefix_len, seqs (an array of
    decode_seqs_desc(), which the result refers to: later changes of it count)."""
    d = np.zeros(len(groups), SHARED_GROUP)
    prefixes = []
    for i, g in enumerate(groups):
        if g["prefix_len"]:
            k, v = g["k_cache"], g["v_cache"]
            d[i]["prefix_k_cache"] = _addresses("prefix k_cache", [k], 1, (torch.float16,))[0]
            d[i]["prefix_v_cache"] = _addresses("prefix v_cache", [v], 1, (torch.float16,), tuple(k.shape))[0]
            d[i]["prefix_cap"] = k.shape[0]
            prefixes.append(_row_heads("prefix k_cache", [k], [k.shape[0]]))
        d[i]["prefix_len"] = g["prefix_len"]
        d[i]["seqs"], d[i]["n_seqs"] = _records(g["seqs"], DECODE_SEQ, "decode_seqs_desc")
    return _Groups(d, [g["seqs"] for g in groups], prefixes)


class _Groups:
    """Group descriptors, the sequence arrays that they point to, and the KV heads of the prefixes."""

    def __init__(self, desc, seqs, prefixes):
        self.desc, self.seqs, self.prefixes, self.at = desc, seqs, prefixes, desc.ctypes.data


def decode_shared_workspace(n_groups, n_seqs, q_heads, kv_heads) -> int:
    """Bytes of a workspace for decode_shared(), n_seqs over all groups: allocate it zero-filled."""
    return int(lib().sf37kv_decode_shared_workspace(n_groups, n_seqs, q_heads, kv_heads))


def decode_shared(groups, q_heads, kv_heads, head_dim, cache_dtype, dtype, workspace, stream=None):
    """One decode step of groups that share a prefix; cache_dtype: F16 or I8, of the sequences' own caches."""
    device, at, size = _space(workspace)
    for seqs in groups.seqs:
        _checked(seqs, "decode_shared", device, kv_heads, dtype, torch.uint8 if cache_dtype == I8 else torch.float16, q_heads)
    for heads in groups.prefixes:
        if heads != kv_heads:
            raise ValueError(f"decode_shared: kv_heads is {kv_heads}, the prefixes have {groups.prefixes}")
    check(lib().sf37kv_decode_shared(groups.at, len(groups.seqs), q_heads, kv_heads, head_dim, cache_dtype, _IO[dtype],
                                     at, size, _sp(stream)),
          "sf37kv_decode_shared")
