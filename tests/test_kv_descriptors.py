"""CPU: the Python layer of the int8 and shared-prefix calls refuses tensors that do not fit the call, before it
reaches the library.  Tensors that say they are on the GPU stand in for ones that are."""
import numpy as np
import pytest
import torch

from sf37_b200 import _lib, kv

D = 128


class OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.get_device()))

    def get_device(self):
        return 0


class OnOther(OnGpu):
    def get_device(self):
        return 1


def gpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


def i8(n, cap, heads):
    return gpu(n, (cap * heads * 132 + 255) // 256 * 256, dtype=torch.uint8)


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """A GPU 0 that is current, and a library that records what reaches it."""
    seen = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: seen.append((name, a)) or 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(kv, "lib", Library)
    return seen


def append(n=2, cap=16, heads=4, n_tok=3, dtype=torch.float32):
    return kv.append_i8_desc(i8(n, cap, heads), i8(n, cap, heads), cap, 0, gpu(n, n_tok, heads, D, dtype=dtype),
                             gpu(n, n_tok, heads, D, dtype=dtype))


def read(n=2, cap=16, heads=4, dst_cap=8, dtype=torch.float16):
    return kv.read_i8_desc(i8(n, cap, heads), i8(n, cap, heads), cap, gpu(n, dst_cap, heads, D, dtype=dtype),
                           gpu(n, dst_cap, heads, D, dtype=dtype), dst_cap, 0, dst_cap)


def seqs(n=2, cap=16, heads=4, group=2, cache="i8", dtype=torch.float32, new=True):
    make = (lambda: i8(n, cap, heads)) if cache == "i8" else (lambda: gpu(n, cap, heads, D, dtype=torch.float16))
    rows = [gpu(n, heads, D, dtype=dtype) if new else None for _ in range(2)]
    return kv.decode_seqs_desc(make(), make(), cap, 9, gpu(n, heads * group, D, dtype=dtype),
                               gpu(n, heads * group, D, dtype=dtype), k_new=rows[0], v_new=rows[1])


def groups(s, heads=4, cap=10):
    return kv.shared_groups_desc([dict(k_cache=gpu(cap, heads, D, dtype=torch.float16),
                                       v_cache=gpu(cap, heads, D, dtype=torch.float16), prefix_len=8, seqs=s)])


def space():
    return gpu(1 << 10, dtype=torch.uint8)


def test_calls_that_fit_reach_the_library(calls):
    kv.append_i8(append(), 4, D, torch.float32)
    kv.append_i8(append(dtype=torch.bfloat16)[:1], 4, D, torch.bfloat16)
    kv.read_i8(read(), 4, D, torch.float16)
    kv.decode_i8(seqs(), 8, 4, D, torch.float32, space())
    kv.decode_i8(seqs(new=False).copy(), 8, 4, D, torch.float32, space())
    kv.decode_shared(groups(seqs(cache="f16")), 8, 4, D, kv.F16, torch.float32, space())
    kv.decode_shared(groups(seqs()), 8, 4, D, kv.I8, torch.float32, space())
    lists = [gpu(3, 4, D), gpu(1, 4, D)]
    kv.append_i8(kv.append_i8_desc([i8(1, 16, 4)[0], i8(1, 5, 4)[0]], list(i8(2, 16, 4)), [16, 5], 0, lists, lists), 4, D,
                 torch.float32)
    # larger buffers than the caches, and a plain array of records, are the caller's business
    kv.append_i8(kv.append_i8_desc(i8(1, 99, 4), i8(1, 16, 4), 16, 0, gpu(1, 3, 4, D), gpu(1, 3, 4, D)), 4, D, torch.float32)
    kv.append_i8(np.zeros(1, _lib.APPEND_I8_LAYER), 4, D, torch.float32)
    assert len(calls) == 10
    d = seqs(n=3)
    d[1] = seqs(n=1)[0]  # one sequence's record replaced
    kv.decode_i8(d, 8, 4, D, torch.float32, space())
    with pytest.raises(ValueError, match="kv_heads"):
        kv.decode_i8(d, 16, 8, D, torch.float32, space())


def test_kv_heads_that_the_rows_or_caches_do_not_have(calls):
    for call in (lambda h: kv.append_i8(append(), h, D, torch.float32),
                 lambda h: kv.decode_i8(seqs(), 2 * h, h, D, torch.float32, space()),
                 lambda h: kv.decode_shared(groups(seqs(cache="f16", new=False)), 8, h, D, kv.F16, torch.float32, space())):
        for h in (2, 8):
            with pytest.raises(ValueError, match="kv_heads"):
                call(h)
    for call in (lambda: kv.read_i8(read(), 8, D, torch.float16),
                 lambda: kv.decode_i8(seqs(new=False), 8, 8, D, torch.float32, space())):
        with pytest.raises(ValueError, match="room for 4"):
            call()
    with pytest.raises(ValueError, match="q_heads"):
        kv.decode_i8(seqs(), 16, 4, D, torch.float32, space())
    assert not calls


def test_caches_smaller_than_their_rows(calls):
    k = gpu(2, 3, 4, D)
    for small, full in ((i8(2, 15, 4), i8(2, 16, 4)), (i8(2, 16, 4), i8(2, 15, 4))):
        with pytest.raises(ValueError, match="room for 3"):
            kv.append_i8(kv.append_i8_desc(small, full, 16, 0, k, k), 4, D, k.dtype)
        with pytest.raises(ValueError, match="room for 3"):
            kv.decode_i8(kv.decode_seqs_desc(small, full, 16, 9, gpu(2, 8, D), gpu(2, 8, D)), 8, 4, D, k.dtype, space())
        with pytest.raises(ValueError, match="room for 3"):
            kv.read_i8(kv.read_i8_desc(small, full, 16, gpu(2, 8, 4, D), gpu(2, 8, 4, D), 8, 0, 8), 4, D, k.dtype)
    for a, b in ((7, 8), (8, 7)):
        with pytest.raises(ValueError, match="room for 3"):
            kv.read_i8(kv.read_i8_desc(i8(2, 16, 4), i8(2, 16, 4), 16, gpu(2, a, 4, D), gpu(2, b, 4, D), 8, 0, 8), 4, D, k.dtype)
    with pytest.raises(ValueError, match="smaller than cap"):
        kv.append_i8_desc(i8(2, 16, 4), i8(2, 16, 4), 80, 0, k, k)
    with pytest.raises(ValueError, match="room for 1"):  # one of a list
        kv.append_i8(kv.append_i8_desc([i8(1, 16, 4)[0], i8(1, 4, 4)[0]], list(i8(2, 16, 4)), 16, 0, list(k), list(k)), 4, D,
                     k.dtype)
    assert not calls


def test_types_that_the_call_does_not_name(calls):
    with pytest.raises(ValueError, match="dtype"):
        kv.append_i8(append(), 4, D, torch.bfloat16)
    with pytest.raises(ValueError, match="dtype"):
        kv.read_i8(read(), 4, D, torch.float32)
    with pytest.raises(ValueError, match="dtype"):
        kv.decode_i8(seqs(), 8, 4, D, torch.bfloat16, space())
    with pytest.raises(ValueError, match="caches of"):
        kv.decode_i8(seqs(cache="f16"), 8, 4, D, torch.float32, space())
    with pytest.raises(ValueError, match="caches of"):
        kv.decode_shared(groups(seqs()), 8, 4, D, kv.F16, torch.float32, space())
    with pytest.raises(ValueError, match="caches of"):
        kv.decode_shared(groups(seqs(cache="f16")), 8, 4, D, kv.I8, torch.float32, space())
    q = gpu(2, 8, D)
    with pytest.raises(ValueError, match="dtype"):
        kv.decode_seqs_desc(i8(2, 16, 4), gpu(2, 16, 4, D, dtype=torch.float16), 16, 9, q, q.clone())
    with pytest.raises(ValueError, match="one dtype"):
        kv.decode_seqs_desc([i8(1, 16, 4)[0], gpu(16, 4, D, dtype=torch.float16)], i8(2, 16, 4), 16, 9, q, q.clone())
    k = [gpu(3, 4, D), gpu(3, 4, D, dtype=torch.bfloat16)]
    with pytest.raises(ValueError, match="one dtype"):
        kv.append_i8_desc(i8(2, 16, 4), i8(2, 16, 4), 16, 0, k, k)
    assert not calls


def test_rows_and_prefixes_of_different_shapes(calls):
    with pytest.raises(ValueError, match="v: "):
        kv.append_i8_desc(i8(2, 16, 4), i8(2, 16, 4), 16, 0, gpu(2, 3, 4, D), gpu(2, 2, 4, D))
    with pytest.raises(ValueError, match="v: "):
        kv.append_i8_desc(i8(2, 16, 4), i8(2, 16, 4), 16, 0, [gpu(3, 4, D), gpu(2, 4, D)], [gpu(3, 4, D), gpu(1, 4, D)])
    with pytest.raises(ValueError, match="one number of heads"):
        kv.append_i8_desc(i8(2, 16, 4), i8(2, 16, 4), 16, 0, [gpu(3, 4, D), gpu(3, 2, D)], [gpu(3, 4, D), gpu(3, 2, D)])
    half = lambda *s: gpu(*s, dtype=torch.float16)  # noqa: E731
    with pytest.raises(ValueError, match="prefix v_cache"):
        kv.shared_groups_desc([dict(k_cache=half(10, 4, D), v_cache=half(9, 4, D), prefix_len=8, seqs=seqs(cache="f16"))])
    with pytest.raises(ValueError, match="prefixes"):
        kv.decode_shared(groups(seqs(cache="f16"), heads=2), 8, 4, D, kv.F16, torch.float32, space())
    assert not calls


def test_workspaces_and_devices(calls, monkeypatch):
    s, append_0 = seqs(), append()
    for ws in (torch.zeros(1 << 10, dtype=torch.uint8), space()[::2], torch.zeros(8, dtype=torch.uint8).as_subclass(OnOther)):
        with pytest.raises(ValueError, match="workspace"):
            kv.decode_i8(s, 8, 4, D, torch.float32, ws)
        with pytest.raises(ValueError, match="workspace"):
            kv.decode_shared(groups(seqs(cache="f16")), 8, 4, D, kv.F16, torch.float32, ws)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)  # another device than when the array was made
    with pytest.raises(ValueError, match="workspace"):
        kv.decode_i8(s, 8, 4, D, torch.float32, space())
    for call in (lambda ws: kv.decode_i8(s, 8, 4, D, torch.float32, ws), lambda ws: kv.append_i8(append_0, 4, D, torch.float32)):
        with pytest.raises(ValueError, match="device 0"):
            call(torch.zeros(8, dtype=torch.uint8).as_subclass(OnOther))
    assert not calls
