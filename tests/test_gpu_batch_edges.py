"""GPU: calls of the int8 cache and batched decode entry points at the edges: long
caches, large batches, captures in a fresh process, streams, and launches that
follow one another without a wait."""
import os
import subprocess
import sys

import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, attend, attended, bound, check, fill_i8, i8_cache, rows, values, workspace

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_many_splits_of_one_head():
    # more splits than the direct map from CTA to sequence holds; all sequences read one cache
    n, cap = 256, 6000
    raw_k, kx = fill_i8(1, cap, 1, 1)
    raw_v, vx = fill_i8(1, cap, 1, 2)
    q = rows(3, n, 4)
    out = torch.full_like(q, float("nan"))
    d = kv.decode_seqs_desc([raw_k[0]] * n, [raw_v[0]] * n, cap, [cap - 1] * n, q, out)
    ws = workspace(kv.decode_i8_workspace(n, 4, 1))
    for _ in range(2):
        kv.decode_i8(d, 4, 1, D, q.dtype, ws)
    for i in range(n):
        want, mag, reach = attend(q[i], kx[0], vx[0], None)
        check(out[i], want, bound(want, mag, reach, cap, q.dtype, False), f"sequence {i}")


def test_one_group_over_two_launches():
    n, plen, heads, qh = 300, 200, 1, 4
    pk, pv = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    ko, vo = rows(3, n, 6, heads).half(), rows(4, n, 6, heads).half()
    q = rows(5, n, qh)
    out = torch.full_like(q, float("nan"))
    pos = [plen + i % 6 for i in range(n)]
    d = kv.decode_seqs_desc(ko, vo, 6, pos, q, out)
    ws = workspace(kv.decode_shared_workspace(1, n, qh, heads))
    kv.decode_shared(kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)]), qh, heads, D, kv.F16,
                     q.dtype, ws)
    for i in range(n):
        k = torch.cat([pk.double(), attended(ko[i].double(), 6, pos[i], plen)])
        v = torch.cat([pv.double(), attended(vo[i].double(), 6, pos[i], plen)])
        want, mag, reach = attend(q[i], k, v, None)
        check(out[i], want, bound(want, mag, reach, k.shape[0], q.dtype, False), f"sequence {i}")


def test_cache_offsets_past_32_bits():
    # 4.2 million rows of 8 heads: codes and scales lie beyond 4 GiB
    heads, cap, window = 8, 4_200_000, 40
    raw = [torch.empty(1, kv.i8_cache_bytes(cap, heads), dtype=torch.uint8, device="cuda") for _ in range(2)]
    first = cap - 30
    k, v = rows(1, 1, 50, heads), rows(2, 1, 50, heads)
    kv.append_i8(kv.append_i8_desc(raw[0], raw[1], cap, first, k, v), heads, D, k.dtype)  # past the ring's end too
    back = [torch.zeros(1, 50, heads, D, device="cuda") for _ in range(2)]
    kv.read_i8(kv.read_i8_desc(raw[0], raw[1], cap, back[0], back[1], 50, first, 50), heads, D, torch.float32)
    at = (first + torch.arange(50, device="cuda")) % 50
    for x, y in zip(back, (k, v)):
        assert ((x[0, at] - y[0]).abs() <= y[0].abs().amax(-1, keepdim=True) / 253.9).all()
    q = rows(3, 1, 64)
    out = torch.empty_like(q)
    pos = first + 49
    kv.decode_i8(kv.decode_seqs_desc(raw[0], raw[1], cap, pos, q, out, sliding=True, window=window), 64, heads, D, q.dtype,
                 workspace(kv.decode_i8_workspace(1, 64, heads)))
    want, mag, reach = attend(q[0], back[0][0, at][50 - window:].double(), back[1][0, at][50 - window:].double(), None)
    check(out[0], want, bound(want, mag, reach, window, q.dtype, False))


def test_prefix_offsets_past_32_bits():
    heads, plen, qh = 8, 2_200_000, 64
    pk, pv = (torch.empty(plen, heads, D, dtype=torch.float16, device="cuda") for _ in range(2))
    pk[-300:], pv[-300:] = rows(1, 300, heads).half(), rows(2, 300, heads).half()
    ko, vo = rows(3, 2, 8, heads).half(), rows(4, 2, 8, heads).half()
    q = rows(5, 2, qh)
    out = torch.empty_like(q)
    d = kv.decode_seqs_desc(ko, vo, 8, [plen + 3, plen + 7], q, out, sliding=True, window=250)
    kv.decode_shared(kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)]), qh, heads, D, kv.F16,
                     q.dtype, workspace(kv.decode_shared_workspace(1, 2, qh, heads)))
    for i, p in enumerate((plen + 3, plen + 7)):
        at = torch.arange(plen, p + 1, device="cuda") % 8
        k, v = (torch.cat([a[p + 1 - 250:].double(), b[i][at].double()]) for a, b in ((pk, ko), (pv, vo)))
        want, mag, reach = attend(q[i], k, v, None)
        check(out[i], want, bound(want, mag, reach, 250, q.dtype, False))
    assert kv.device_error() == 0


def test_first_calls_inside_a_capture():
    """A process whose first library calls are captured."""
    script = """
import torch
from sf37_b200 import kv
from tests.batch_util import rows
h, n, cap, plen = 2, 3, 40, 200
raw = [torch.zeros(n, kv.i8_cache_bytes(cap, h), dtype=torch.uint8, device="cuda") for _ in range(2)]
k, v = rows(1, n, 20, h), rows(2, n, 20, h)
pk, pv = rows(3, plen, h).half(), rows(4, plen, h).half()
q = rows(5, n, 16)
outs = [torch.zeros_like(q) for _ in range(2)]
ws = [torch.zeros(kv.decode_shared_workspace(1, n, 16, h), dtype=torch.uint8, device="cuda") for _ in range(2)]
ap = kv.append_i8_desc(raw[0], raw[1], cap, 0, k, v)
d0 = kv.decode_seqs_desc(raw[0], raw[1], cap, 19, q, outs[0])
ap2 = kv.append_i8_desc(raw[0], raw[1], cap, plen, k, v)
d1 = kv.decode_seqs_desc(raw[0], raw[1], cap, plen + 19, q, outs[1])
g1 = kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d1)])
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
def step(stream):
    kv.append_i8(ap, h, 128, k.dtype, stream=stream)
    kv.decode_i8(d0, 16, h, 128, q.dtype, ws[0], stream=stream)
    kv.append_i8(ap2, h, 128, k.dtype, stream=stream)
    kv.decode_shared(g1, 16, h, 128, kv.I8, q.dtype, ws[1], stream=stream)
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    step(s)
g.replay(); torch.cuda.synchronize()
got = [o.clone() for o in outs]
step(s); torch.cuda.synchronize()
assert all(torch.equal(a, b) and a.abs().sum() > 0 for a, b in zip(got, outs))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", script], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_steps_that_follow_without_a_wait():
    """Each step reads the row that the one before appended; mixed with sf37kv_decode on caches that the calls write."""
    heads, qh, plen, steps, cap = 4, 32, 500, 12, 64
    pk, pv = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    q = rows(5, steps, 2, qh)
    new = rows(6, steps, 2, heads), rows(7, steps, 2, heads)

    def run(wait):
        raw = [i8_cache(2, cap, heads, 0) for _ in range(2)]
        own = [torch.zeros(2, cap, heads, D, dtype=torch.float16, device="cuda") for _ in range(2)]
        whole = [torch.zeros(cap, heads, D, dtype=torch.float16, device="cuda") for _ in range(2)]
        outs = [torch.zeros(steps, 2, qh, D, device="cuda") for _ in range(4)]
        ws = workspace(kv.decode_shared_workspace(1, 2, qh, heads))
        keep = []
        for t in range(steps):
            a = kv.decode_seqs_desc(raw[0], raw[1], cap, t, q[t], outs[0][t], k_new=new[0][t], v_new=new[1][t])
            b = kv.decode_seqs_desc(own[0], own[1], cap, plen + t, q[t], outs[1][t], k_new=new[0][t], v_new=new[1][t])
            g = kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=b)])
            r = kv.read_i8_desc([raw[0][0]], [raw[1][0]], cap, [whole[0]], [whole[1]], cap, 0, t + 1)
            keep += [a, b, g, r]
            kv.decode_i8(a, qh, heads, D, q.dtype, ws)
            if wait:
                torch.cuda.synchronize()
            kv.decode_shared(g, qh, heads, D, kv.F16, q.dtype, ws)
            if wait:
                torch.cuda.synchronize()
            # the f16 cache that the shared call has just written, slots from (plen % cap) on
            kv.decode([dict(k_cache=own[0][0], v_cache=own[1][0], cap=cap, pos=plen + t, sliding=1, window=t + 1, q=q[t, 0],
                            out=outs[2][t, 0])], qh, heads, D, kv.F16)
            if wait:
                torch.cuda.synchronize()
            kv.read_i8(r, heads, D, torch.float16)
            kv.decode([dict(k_cache=whole[0], v_cache=whole[1], cap=cap, pos=t, q=q[t, 1], out=outs[3][t, 0])], qh, heads, D,
                      kv.F16)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs

    want = run(True)
    for _ in range(3):
        for a, b in zip(run(False), want):
            assert torch.equal(a, b)


def test_two_streams_with_a_workspace_each():
    heads, cap, n = 8, 5000, 6
    raw_k, raw_v = fill_i8(n, cap, heads, 1)[0], fill_i8(n, cap, heads, 2)[0]
    qs = [rows(s, n, 64, dtype=torch.bfloat16) for s in (1, 2)]
    want = []
    for q in qs:
        o = torch.empty_like(q)
        kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, cap - 1, q, o), 64, heads, D, q.dtype,
                     workspace(kv.decode_i8_workspace(n, 64, heads)))
        want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[torch.empty_like(q) for _ in range(8)] for q in qs]
    wss = [workspace(kv.decode_i8_workspace(n, 64, heads)) for _ in qs]
    torch.cuda.synchronize()
    for k in range(8):
        for q, o, ws, s in zip(qs, outs, wss, streams):
            kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, cap - 1, q, o[k]), 64, heads, D, q.dtype, ws, stream=s)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)


def test_a_padded_batch_leaves_the_rest_alone():
    # descriptors of a fixed batch, of which a step uses the first few; other outputs and caches stay
    heads, cap, n, used = 2, 50, 8, 3
    raw_k, raw_v = fill_i8(n, cap, heads, 1)[0], fill_i8(n, cap, heads, 2)[0]
    q, new = rows(3, n, 16), rows(4, n, heads)
    out = torch.full((n, 16, D), 5.0, device="cuda")
    before = raw_k.clone(), raw_v.clone()
    d = kv.decode_seqs_desc(raw_k, raw_v, cap, 20, q, out, k_new=new, v_new=new)
    kv.decode_i8(d[:used], 16, heads, D, q.dtype, workspace(kv.decode_i8_workspace(n, 16, heads)))
    assert (out[used:] == 5).all() and torch.isfinite(out[:used]).all()
    assert torch.equal(raw_k[used:], before[0][used:]) and torch.equal(raw_v[used:], before[1][used:])
    assert not torch.equal(raw_k[:used], before[0][:used])


@pytest.mark.parametrize("group", [8, 12])
def test_f32_sums_over_long_splits(group):
    # 48 sequences over one cache of 20000 rows: a warp takes hundreds of blocks, O is taken out of the tensor core's
    # truncating sums every 32 of them.  Each MMA drops at most 2^-23 of O: 32 * 2^-23 = 3.8e-6 of the output, and the
    # scores' and weights' parts (bound() without its rows) of the weighted magnitude.
    n, cap, heads = 48, 20000, 8
    raw_k, kx = fill_i8(1, cap, heads, 1)
    raw_v, vx = fill_i8(1, cap, heads, 2)
    q = rows(3, n, group * heads)
    out = torch.full_like(q, float("nan"))
    d = kv.decode_seqs_desc([raw_k[0]] * n, [raw_v[0]] * n, cap, [cap - 1 - i for i in range(n)], q, out)
    kv.decode_i8(d, group * heads, heads, D, q.dtype, workspace(kv.decode_i8_workspace(n, group * heads, heads)))
    for i in range(0, n, 7):
        want, mag, reach = attend(q[i], kx[0][:cap - i], vx[0][:cap - i], None)
        assert torch.isfinite(out[i]).all()
        err = (out[i].double() - want).norm() / want.norm()
        limit = 3.8e-6 + 2 * (0.6932 * reach.max().item() * 2.0 ** -21 + 2.0 ** -21)
        assert err <= limit, f"sequence {i}: {err:.3g}"


def test_f32_sums_over_a_long_prefix():
    # few splits of many tiles: the prefix kernel takes O into memory between them
    n, plen, heads, group = 80, 9000, 8, 12
    qh = heads * group
    pk, pv = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    ko, vo = rows(3, n, 4, heads).half(), rows(4, n, 4, heads).half()
    q = rows(5, n, qh, scale=1.5)
    out = torch.full_like(q, float("nan"))
    d = kv.decode_seqs_desc(ko, vo, 4, [plen + i % 4 for i in range(n)], q, out)
    ws = workspace(kv.decode_shared_workspace(1, n, qh, heads))
    for _ in range(2):
        kv.decode_shared(kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)]), qh, heads, D, kv.F16,
                         q.dtype, ws)
    for i in range(0, n, 9):
        own = i % 4 + 1
        at = torch.arange(plen, plen + own, device="cuda") % 4
        k, v = torch.cat([pk.double(), ko[i][at].double()]), torch.cat([pv.double(), vo[i][at].double()])
        want, mag, reach = attend(q[i], k, v, None)
        check(out[i], want, bound(want, mag, reach, plen, q.dtype, False), f"sequence {i}")
        # 256 MMAs of at most 2^-23 each between two of them, and the scores' 16
        assert (out[i].double() - want).norm() <= (256 + 16 * 0.6932 * reach.max().item()) * 2.0 ** -23 * want.norm()
    assert kv.device_error() == 0
