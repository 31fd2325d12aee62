"""GPU: steps of int8 caches and shared prefixes at fixed addresses that follow one another without a wait.  Each
kernel starts while the one before drains and reads what it wrote: queries, appended rows and scales."""
import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, i8_cache, rows, workspace

pytestmark = pytest.mark.gpu


class Chain:
    """n sequences over a prefix and a second model part over int8 caches; each call's outputs are the next one's
    queries, and its appended rows are parts of them."""

    def __init__(self, n, heads, group, cache, dtype, plen=700, cap=48):
        self.n, self.heads, self.qh, self.dtype, self.plen = n, heads, heads * group, dtype, plen
        self.cache = kv.I8 if cache == "i8" else kv.F16
        make = (lambda: i8_cache(n, cap, heads, 0)) if cache == "i8" else (
            lambda: torch.zeros(n, cap, heads, D, dtype=torch.float16, device="cuda"))
        self.own, self.raw = [make(), make()], [i8_cache(n, cap, heads, 0), i8_cache(n, cap, heads, 0)]
        self.pk, self.pv = rows(1, plen, heads).half(), rows(2, plen, heads).half()
        self.x, self.y = (torch.zeros(n, self.qh, D, device="cuda", dtype=dtype) for _ in range(2))
        self.back = [torch.zeros(n, cap, heads, D, device="cuda") for _ in range(2)]
        self.start = 3 * rows(3, n, self.qh, dtype=dtype)
        self.a = kv.decode_seqs_desc(self.own[0], self.own[1], cap, plen, self.x, self.y,
                                     k_new=self.x[:, :heads], v_new=self.x[:, -heads:])
        self.b = kv.decode_seqs_desc(self.raw[0], self.raw[1], cap, 0, self.y, self.x,
                                     k_new=self.y[:, :heads], v_new=self.y[:, -heads:])
        self.g = kv.shared_groups_desc([dict(k_cache=self.pk, v_cache=self.pv, prefix_len=plen, seqs=self.a)])
        self.r = kv.read_i8_desc(self.raw[0], self.raw[1], cap, self.back[0], self.back[1], cap, 0, cap)
        self.ws = workspace(kv.decode_shared_workspace(1, n, self.qh, heads))

    def reset(self):
        for t in self.own + self.raw + self.back:
            t.zero_()
        self.x.copy_(self.start)
        torch.cuda.synchronize()

    def run(self, steps, wait, stream=None, back=True):
        for t in range(steps):
            self.a["pos"], self.b["pos"] = self.plen + t, t
            for call in (lambda: kv.decode_shared(self.g, self.qh, self.heads, D, self.cache, self.dtype, self.ws, stream=stream),
                         lambda: kv.decode_i8(self.b, self.qh, self.heads, D, self.dtype, self.ws, stream=stream)):
                call()
                if wait:
                    torch.cuda.synchronize()
        kv.read_i8(self.r, self.heads, D, torch.float32, stream=stream)

    def result(self):
        torch.cuda.synchronize()
        return [t.clone() for t in self.own + self.raw + self.back + [self.x, self.y]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cache", ["i8", "f16"])
# (sequences, KV heads): above 37 pairs the own rows are joined by a third launch, below by the second itself
@pytest.mark.parametrize("n,heads", [(9, 8), (40, 8), (2, 4)])
def test_steps_without_a_wait(n, heads, cache, dtype):
    c, steps = Chain(n, heads, 8, cache, dtype), 30
    c.reset()
    c.run(steps, True)
    want = c.result()
    assert torch.isfinite(want[-1]).all() and want[-1].abs().sum() > 0
    for _ in range(3):
        c.reset()
        c.run(steps, False)
        for got, w in zip(c.result(), want):
            assert torch.equal(got, w)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    c.reset()
    with torch.cuda.graph(g, stream=s):
        c.run(steps, False, stream=s)
    for _ in range(3):
        c.reset()
        g.replay()
        for got, w in zip(c.result(), want):
            assert torch.equal(got, w)
    assert kv.device_error() == 0


def test_the_workspace_is_left_zeroed_where_calls_meet():
    """Counters and the flag between the prefix launch and the one beside it are zero after each call."""
    for n, heads in ((9, 8), (2, 4), (300, 1)):
        c = Chain(n, heads, 4, "f16", torch.float32)
        c.reset()
        c.run(2, False)
        torch.cuda.synchronize()
        assert not c.ws[:16384 * 4 + 256].any()
