"""Plain 64-bit forms of the int8 caches and of batched decode, and the error
bounds their tests use."""
import math

import numpy as np
import torch

from sf37_b200 import kv

D = 128


def rows(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (scale * torch.randn(*shape, D, device="cuda", generator=g)).to(dtype)


def i8_cache(n, cap, heads, fill=0xA5):
    """n int8 caches of K or V as bytes, filled with a pattern."""
    return torch.full((n, kv.i8_cache_bytes(cap, heads)), fill, dtype=torch.uint8, device="cuda")


def i8_views(raw, cap, heads):
    """Codes [n, cap, heads, 128] (u8) and scales [n, heads, cap] of caches held as bytes."""
    c = cap * heads * D
    return raw[:, :c].view(-1, cap, heads, D), raw[:, c:c + 4 * heads * cap].view(torch.float32).view(-1, heads, cap)


def quantise(x):
    """(codes c + 128, scales) of the heads of x [..., 128], numpy, decided in 64 bits."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        a = np.max(np.abs(x), -1)
        s = (a.astype(np.float64) / 127).astype(np.float32)
        s = np.where(s < np.float32(2.0 ** -126), np.float32(0), s)
        s = np.where(np.isfinite(x).all(-1), s, np.float32(np.nan))
        q = x.astype(np.float64) / s.astype(np.float64)[..., None]
        c = np.where((s > 0)[..., None], np.rint(q), 0.0)
    return (c + 128).astype(np.uint8), s


def fill_i8(n, cap, heads, seed, scale=1.0):
    """Stacked int8 caches of random rows, and their values [n, cap, heads, 128] in 64 bits."""
    raw = i8_cache(n, cap, heads, 0)
    codes, scales = i8_views(raw, cap, heads)
    c, s = quantise(rows(seed, n, cap, heads, scale=scale).cpu().numpy())
    codes.copy_(torch.from_numpy(c))
    scales.copy_(torch.from_numpy(np.ascontiguousarray(np.swapaxes(s, 1, 2))))
    return raw, values(raw, cap, heads)


def values(raw, cap, heads):
    codes, scales = i8_views(raw, cap, heads)
    return (codes.double() - 128) * scales.double().transpose(1, 2).unsqueeze(-1)


def attend(q, k, v, gate):
    """softmax(q k^T / sqrt(128)) v * sigmoid(gate) in 64 bits: q [q_heads, 128], k, v [rows, kv_heads, 128].
    Also sum p|v| * gate and the largest sum |q_d k_d| * log2(e) / sqrt(128) of each head."""
    heads = k.shape[1]
    q = q.double().view(heads, -1, D)
    g = torch.ones(q.shape[0] * q.shape[1], dtype=torch.float64, device=q.device) if gate is None else torch.sigmoid(gate.double())
    g = g.view(heads, -1, 1)
    if k.shape[0] == 0:
        z = torch.zeros_like(q).view(-1, D)
        return z, z, torch.zeros(z.shape[0], 1, dtype=torch.float64, device=q.device)
    s = torch.einsum("hgd,rhd->hgr", q, k) / math.sqrt(D)
    p = torch.softmax(s, -1)
    o = torch.einsum("hgr,rhd->hgd", p, v) * g
    mag = torch.einsum("hgr,rhd->hgd", p, v.abs()) * g
    reach = torch.einsum("hgd,rhd->hgr", q.abs(), k.abs()).amax(-1, keepdim=True) * (math.log2(math.e) / math.sqrt(D))
    return o.reshape(-1, D), mag.reshape(-1, D), reach.reshape(-1, 1)


def coarse_q(q, k):
    """Largest error (log2 units) of a score over int8 caches from a bf16 query: held to half a unit of 2^-13 of the
    power of two below its largest element, against sum |k|.  q [q_heads, 128], k [rows, kv_heads, 128]."""
    if k.shape[0] == 0:
        return 0.0
    step = 2.0 ** torch.floor(torch.log2(q.double().abs().amax(-1))) * 2.0 ** -14
    reach = k.abs().sum(-1).amax(0).repeat_interleave(q.shape[0] // k.shape[1])
    return (step * reach * (math.log2(math.e) / math.sqrt(D))).view(-1, 1)


def bound(want, mag, reach, n_rows, dtype, p_f16, score=0.0):
    """Largest error of an output, `score` being an error of the scores beyond the following.  A score (log2 units) sums 8 tile products in f32 (each step may drop 2^-23 of at
    most `reach`) of operands held to 22 bits: 2^-19 * reach, a relative error ln 2 of that in its weight; the
    exponential 2^-21; the weight 2^-22 in two f16 parts, or 2^-11 in one; the output sums n_rows / 16 tile products at
    2^-23 each, and the merge and the division a few 2^-23.  Numerator and denominator each carry it."""
    w = 0.6932 * (reach * 2.0 ** -19 + score) + 2.0 ** -21 + (2.0 ** -11 if p_f16 else 2.0 ** -22) + (n_rows / 16 + 16) * 2.0 ** -23
    return 2 * w * mag + 1e-30 + (2.0 ** -8 * want.abs() * (1 + 2 * 2.0 ** -8) if dtype == torch.bfloat16 else 0)


def check(got, want, tol, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() / tol).max().item()
    assert over <= 1, f"{what}: {over:.3g} times the bound"


def attended(cache_values, cap, pos, first):
    """Rows first..pos of one cache [cap, heads, 128]."""
    at = torch.arange(first, pos + 1, device=cache_values.device)
    return cache_values[at % cap]


def workspace(size):
    return torch.zeros(size, dtype=torch.uint8, device="cuda")
