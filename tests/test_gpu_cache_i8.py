"""GPU: int8 caches, written and read back, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, i8_cache, i8_views, quantise, rows

pytestmark = pytest.mark.gpu


def _append(raw_k, raw_v, cap, pos0, k, v, heads):
    kv.append_i8(kv.append_i8_desc(raw_k, raw_v, cap, pos0, k, v), heads, D, k.dtype)


def _expect(raw, cap, heads, pos0, x):
    """The cache bytes after a sequential append of x [n, n_tok, heads, 128] to a copy of raw."""
    codes, scales = (t.clone() for t in i8_views(raw, cap, heads))
    c, s = quantise(x.float().cpu().numpy())
    for t in range(x.shape[1]):
        slot = (pos0 + t) % cap
        codes[:, slot] = torch.from_numpy(c[:, t]).cuda()
        scales[:, :, slot] = torch.from_numpy(s[:, t]).cuda()
    return codes, scales


@pytest.mark.parametrize("n,heads,cap,pos0,n_tok", [(1, 1, 1, 0, 1), (3, 8, 5, 3, 1), (2, 8, 64, 60, 9), (1, 3, 17, 40, 17),
                                                    (2, 5, 7, 2, 31), (70, 2, 4, 9, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_codes_and_scales(n, heads, cap, pos0, n_tok, dtype):
    k, v = rows(1, n, n_tok, heads, dtype=dtype), rows(2, n, n_tok, heads, dtype=dtype, scale=30.0)
    raw_k, raw_v = i8_cache(n, cap, heads), i8_cache(n, cap, heads, 0x3C)
    want = [_expect(r, cap, heads, pos0, x) for r, x in ((raw_k, k), (raw_v, v))]
    tails = [r[:, cap * heads * 132:].clone() for r in (raw_k, raw_v)]
    _append(raw_k, raw_v, cap, pos0, k, v, heads)
    for raw, (codes, scales), tail in zip((raw_k, raw_v), want, tails):
        got_c, got_s = i8_views(raw, cap, heads)
        assert torch.equal(got_c, codes)
        assert torch.equal(got_s.view(torch.int32), scales.view(torch.int32))
        assert torch.equal(raw[:, cap * heads * 132:], tail)  # the padding stays


def test_append_special_values():
    # ties, exact multiples, tiny, subnormal, huge, zero and non-finite heads
    x = torch.zeros(1, 9, 1, D)
    x[0, 0, 0, :5] = torch.tensor([127.0, 0.5, 1.5, -2.5, 126.5])  # scale 1: ties to even
    x[0, 1] = 0
    x[0, 2] = 1e-39 * torch.arange(D)        # scale below 2^-126: zeros
    x[0, 3] = 2.0 ** -119 * torch.linspace(-1, 1, D)
    x[0, 4] = 3.4e38 * torch.linspace(-1, 1, D)
    x[0, 5] = torch.linspace(-1, 1, D)
    x[0, 5, 0, 7] = float("nan")
    x[0, 6, 0, 3] = float("inf")
    x[0, 7, 0, 100] = -float("inf")
    x[0, 8] = 2.0 ** -20 * torch.randint(-10 ** 6, 10 ** 6, (D,), generator=torch.Generator().manual_seed(3))
    x = x.cuda()
    raw_k, raw_v = i8_cache(1, 9, 1), i8_cache(1, 9, 1)
    _append(raw_k, raw_v, 9, 0, x, x, 1)
    c, s = quantise(x.cpu().numpy())
    codes, scales = i8_views(raw_k, 9, 1)
    assert np.array_equal(codes.cpu().numpy(), c)
    got = scales.cpu().numpy()[0, 0]
    assert np.array_equal(got, s[0, :, 0], equal_nan=True)
    assert list(codes[0, 0, 0, :5].tolist()) == [255, 128, 130, 126, 254]
    dst_k, dst_v = torch.zeros(1, 9, 1, D, device="cuda"), torch.zeros(1, 9, 1, D, device="cuda")
    kv.read_i8(kv.read_i8_desc(raw_k, raw_v, 9, dst_k, dst_v, 9, 0, 9), 1, D, torch.float32)
    assert torch.isnan(dst_k[0, 5:8]).all() and torch.isfinite(dst_k[0, :5]).all()
    # values are within half a scale; the product c * s is one f32 rounding (2^-24 of at most 127 s)
    live = [0, 1, 3, 4, 8]
    err = (dst_k[0, live].double() - x[0, live].double()).abs()
    half = scales[0, 0, live].double().view(-1, 1, 1) * (0.5 + 127 * 2.0 ** -24)
    assert (err <= half).all()


@pytest.mark.parametrize("n,heads,cap,first,n_rows,dst_cap", [(1, 1, 1, 0, 1, 1), (2, 8, 40, 100, 40, 64), (3, 3, 33, 20, 17, 17),
                                                              (66, 1, 5, 3, 4, 9), (1, 8, 1000, 1500, 777, 800)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_read_back(n, heads, cap, first, n_rows, dst_cap, dtype):
    raw = []
    for seed in (5, 6):
        r = torch.randint(0, 256, i8_cache(n, cap, heads).shape, dtype=torch.uint8, device="cuda",
                          generator=torch.Generator(device="cuda").manual_seed(seed))
        codes, scales = i8_views(r, cap, heads)
        codes.clamp_(min=1)
        scales.copy_(rows(seed, n, heads * cap)[..., 0].view(n, heads, cap).abs())
        raw.append(r)
    dst = [torch.full((n, dst_cap, heads, D), 7.0, device="cuda", dtype=dtype) for _ in range(2)]
    kv.read_i8(kv.read_i8_desc(raw[0], raw[1], cap, dst[0], dst[1], dst_cap, first, n_rows), heads, D, dtype)
    at = torch.arange(first, first + n_rows, device="cuda")
    for r, got in zip(raw, dst):
        codes, scales = i8_views(r, cap, heads)
        x = ((codes.float() - 128) * scales.transpose(1, 2).unsqueeze(-1))[:, at % cap]
        want = torch.full_like(got, 7.0)  # other rows stay
        want[:, at % dst_cap] = x.to(dtype)
        assert torch.equal(got, want)


def test_side_stream_and_graph():
    heads, cap = 8, 64
    k, v = rows(1, 2, 10, heads), rows(2, 2, 10, heads)
    raw_k, raw_v = i8_cache(2, cap, heads), i8_cache(2, cap, heads)
    dst_k, dst_v = (torch.zeros(2, 10, heads, D, device="cuda", dtype=torch.float16) for _ in range(2))
    ap = kv.append_i8_desc(raw_k, raw_v, cap, 60, k, v)
    rd = kv.read_i8_desc(raw_k, raw_v, cap, dst_k, dst_v, 10, 60, 10)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        kv.append_i8(ap, heads, D, k.dtype, stream=s)
        kv.read_i8(rd, heads, D, dst_k.dtype, stream=s)
    k.copy_(rows(11, 2, 10, heads))  # the replay takes what is there now
    g.replay()
    torch.cuda.synchronize()
    c, sc = quantise(k.cpu().numpy())
    want = ((c.astype(np.float32) - 128) * sc[..., None]).astype(np.float16)
    at = (60 + np.arange(10)) % 10
    assert np.array_equal(dst_k.cpu().numpy()[:, at], want)


def test_descriptor_checks():
    raw = i8_cache(2, 4, 1)
    k = rows(1, 2, 3, 1)
    with pytest.raises(ValueError, match="leading dimension"):
        kv.append_i8_desc(raw[:1], raw, 4, 0, k, k)
    with pytest.raises(ValueError, match="contiguous"):
        kv.append_i8_desc(raw, raw.clone(), 4, 0, k, rows(1, 2, 2, 3).transpose(1, 2))
    with pytest.raises(ValueError, match="dtype"):
        kv.append_i8_desc(raw, raw.clone(), 4, 0, k.half(), k.half())
    with pytest.raises(ValueError, match="CUDA"):
        kv.append_i8_desc(raw, raw.clone(), 4, 0, k.cpu(), k.cpu())
    other = raw.clone()
    d = kv.append_i8_desc(raw, other, 4, 0, k, k)
    with pytest.raises(ValueError, match="contiguous array"):
        kv.append_i8(d[::-1], 1, D, k.dtype)
    with pytest.raises(ValueError, match="contiguous array"):
        kv.read_i8(d, 1, D, torch.float32)
    q = rows(1, 2, 4)
    with pytest.raises(ValueError, match="smaller than cap"):
        kv.decode_seqs_desc(raw, other, 4000, 0, q, q.clone())
