"""GPU: queries with a dominant channel over int8 caches.  The bound is the output's own rounding and the
errors of bound(), so a query held to a coarser grid than its type's shows."""
import math

import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, attend, bound, check, i8_cache, rows, values, workspace

IO = [torch.float32, torch.bfloat16]


def fine_q(q, k):
    """Largest error (log2 units) of a score from a query held in three 8-bit digits: half a unit, 2^-22 of the power of
    two at its head's largest element, against sum |k|.  q [q_heads, 128], k [rows, kv_heads, 128]."""
    step = 2.0 ** torch.floor(torch.log2(q.double().abs().amax(-1))) * 2.0 ** -22
    reach = k.abs().sum(-1).amax(0).repeat_interleave(q.shape[0] // k.shape[1])
    return (step * reach * (math.log2(math.e) / math.sqrt(D))).view(-1, 1)


def dominant(seed, n, qh, heads, cap, channel, dtype, device):
    """Queries of which one channel is `channel` times the rest, and keys whose rows differ little in it."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    q = torch.randn(n, qh, D, device=device, generator=g)
    q[..., 17] = channel
    k, v = (torch.randn(n, cap, heads, D, device=device, generator=g) for _ in range(2))
    k[..., 17] = 1 + 0.01 * k[..., 17]
    return q.to(dtype), k, v


def quantised(x):
    """Values of an int8 cache of the rows x [..., 128]."""
    s = x.abs().amax(-1, keepdim=True).double() / 127
    return torch.round(x.double() / s) * s


def digits(q, bits):
    """q held as integers of 2^-bits of the power of two at its head's largest element."""
    unit = 2.0 ** (torch.floor(torch.log2(q.double().abs().amax(-1, keepdim=True))) - bits)
    return torch.round(q.double() / unit) * unit


@pytest.mark.parametrize("channel", [100, 300])
def test_the_bound_tells_three_digits_from_two(channel):
    """CPU: a query of two digits leaves the bound that one of three keeps."""
    cap, heads, group = 700, 2, 8
    q, k, v = dominant(1, 1, heads * group, heads, cap, channel, torch.bfloat16, "cpu")
    k, v = quantised(k[0]), quantised(v[0])
    want, mag, reach = attend(q[0], k, v, None)
    tol = bound(want, mag, reach, cap, torch.bfloat16, False, score=fine_q(q[0], k))
    for bits, inside in ((21, True), (13, False)):
        got = attend(digits(q[0], bits), k, v, None)[0].to(torch.bfloat16).double()
        assert bool(((got - want).abs() <= tol).all()) is inside


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("group", [8, 12])
@pytest.mark.parametrize("channel", [30, 100, 300])
def test_decode(channel, group, dtype):
    n, heads, cap = 3, 2, 700
    q, k, v = dominant(channel, n, heads * group, heads, cap, channel, dtype, "cuda")
    raw_k, raw_v = i8_cache(n, cap, heads), i8_cache(n, cap, heads)
    kv.append_i8(kv.append_i8_desc(raw_k, raw_v, cap, 0, k, v), heads, D, k.dtype)
    out = torch.full_like(q, float("nan"))
    kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, cap - 1, q, out), heads * group, heads, D, dtype,
                 workspace(kv.decode_i8_workspace(n, heads * group, heads)))
    kx, vx = values(raw_k, cap, heads), values(raw_v, cap, heads)
    for i in range(n):
        want, mag, reach = attend(q[i], kx[i], vx[i], None)
        check(out[i], want, bound(want, mag, reach, cap, dtype, p_f16=group > 8 and dtype == torch.bfloat16,
                                  score=fine_q(q[i], kx[i])), f"sequence {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("group", [8, 12])
@pytest.mark.parametrize("channel", [30, 300])
def test_decode_shared(channel, group, dtype):
    n, heads, cap, plen = 5, 2, 300, 260
    q, k, v = dominant(channel, n, heads * group, heads, cap, channel, dtype, "cuda")
    raw_k, raw_v = i8_cache(n, cap, heads), i8_cache(n, cap, heads)
    kv.append_i8(kv.append_i8_desc(raw_k, raw_v, cap, plen, k, v), heads, D, k.dtype)
    pk, pv = rows(7, plen, heads), rows(8, plen, heads).half()
    pk[..., 17] = 1 + 0.01 * pk[..., 17]
    pk = pk.half()
    out = torch.full_like(q, float("nan"))
    d = kv.decode_seqs_desc(raw_k, raw_v, cap, plen + cap - 1, q, out)
    g = kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)])
    kv.decode_shared(g, heads * group, heads, D, kv.I8, dtype, workspace(kv.decode_shared_workspace(1, n, heads * group, heads)))
    at = (plen + torch.arange(cap, device="cuda")) % cap
    kx, vx = values(raw_k, cap, heads)[:, at], values(raw_v, cap, heads)[:, at]
    for i in range(n):
        ki, vi = torch.cat([pk.double(), kx[i]]), torch.cat([pv.double(), vx[i]])
        want, mag, reach = attend(q[i], ki, vi, None)
        check(out[i], want, bound(want, mag, reach, plen + cap, dtype, p_f16=dtype == torch.bfloat16, score=fine_q(q[i], ki)),
              f"sequence {i}")
    assert kv.device_error() == 0
