"""GPU: queries, scores and values at the ends of their ranges, and not finite ones, in batched decode."""
import math

import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, attend, bound, check, fill_i8, i8_cache, i8_views, rows, values, workspace

pytestmark = pytest.mark.gpu

IO = [torch.float32, torch.bfloat16]


def _shared(prefix, own, pos, q, heads, cache=kv.F16, gate=None):
    """One shared call of a group: prefix (k, v) f16 [rows, heads, 128] or None, own caches stacked."""
    n, qh, cap = q.shape[0], q.shape[1], own[0].shape[1] if cache == kv.F16 else own[2]
    out = torch.full_like(q, 5.0)
    d = kv.decode_seqs_desc(own[0], own[1], cap, pos, q, out, gate=gate)
    g = kv.shared_groups_desc([dict(k_cache=prefix[0], v_cache=prefix[1], prefix_len=prefix[0].shape[0], seqs=d) if prefix
                               else dict(k_cache=None, v_cache=None, prefix_len=0, seqs=d)])
    kv.decode_shared(g, qh, heads, D, cache, q.dtype, workspace(kv.decode_shared_workspace(1, n, qh, heads)))
    torch.cuda.synchronize()
    assert kv.device_error() == 0
    return out


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("group", [8, 12])
def test_rows_that_all_score_minus_infinity(group, dtype):
    # the formula divides by a sum of zeros: NaN, not the zeros of a sequence without rows
    heads, cap = 2, 4
    k = rows(1, 2, cap, heads).half()
    k[..., 9] = -1
    v = rows(2, 2, cap, heads).half()
    q = rows(3, 2, heads * group, dtype=dtype)
    q[0, 3, 9] = math.inf
    out = _shared(None, (k, v), [3, 3], q, heads)
    assert torch.isnan(out[0, 3]).all()
    out[0, 3] = 0
    assert torch.isfinite(out).all()
    out = _shared((k[0], v[0]), (k, v), [4, 6], q, heads)
    assert torch.isnan(out[0, 3]).all()
    out[0, 3] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("group", [8, 12])
@pytest.mark.parametrize("cache", ["f16", "i8"])
@pytest.mark.parametrize("power", [22, 60, 102])
def test_scores_of_any_size(power, cache, group, dtype):
    # scores of -1e7 to -1e9, and up to -1e31 to -1e33: the largest one takes all the weight.  Rows are multiples of one row (powers of two, exact
    # in f16 and in int8 scales), so the attended row with the smallest multiple wins by far more than any rounding.
    heads, cap, n = 2, 5, 2
    size = torch.tensor([8.0, 4.0, 1.0, 2.0, 16.0], device="cuda").view(1, cap, 1, 1)
    base = torch.full((n, 1, heads, D), -0.25, device="cuda")
    k, v = base * size, rows(2, n, cap, heads)
    q = (rows(3, n, heads * group).abs() + 1) * 2.0 ** power
    q = q.to(dtype)
    prefix = (base[0] * 64).half().expand(3, heads, D).contiguous(), rows(4, 3, heads).half()
    if cache == "i8":
        raw = i8_cache(n, cap, heads), i8_cache(n, cap, heads)
        kv.append_i8(kv.append_i8_desc(raw[0], raw[1], cap, 0, k, v), heads, D, k.dtype)
        own, v = (raw[0], raw[1], cap), values(raw[1], cap, heads)
    else:
        own, v = (k.half(), v.half()), v.half().double()
    for got, best in ((_shared(prefix, own, [7, 7], q, heads, kv.I8 if cache == "i8" else kv.F16), v[:, 2]),
                      (_shared(None, own, [1, 4], q, heads, kv.I8 if cache == "i8" else kv.F16), torch.stack([v[0, 1], v[1, 2]]))):
        want = best.repeat_interleave(group, 1)
        assert torch.isfinite(got).all()
        # one weight of 1: the value, a product and a division (2^-21 each at most), and the output's rounding
        assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -20 + (2.0 ** -8 if dtype == torch.bfloat16 else 0))).all()
    # over the prefix alone, equal scores: the mean of its rows
    got = _shared(prefix, own, [2, 2], q, heads, kv.I8 if cache == "i8" else kv.F16)
    want = prefix[1].double().mean(0).repeat_interleave(group, 0).expand(n, -1, -1)
    mag = prefix[1].double().abs().mean(0).repeat_interleave(group, 0)
    assert ((got.double() - want).abs() <= mag * 2.0 ** -18 + (want.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else 0)).all()


def _scaled_rows(heads, score, scale):
    """An int8 cache whose row r scores score[r] (log2 units) against queries of ones, with values of size scale[r]."""
    cap = len(score)
    raw_k, raw_v = i8_cache(1, cap, heads, 0), fill_i8(1, cap, heads, 5)[0]
    codes, scales = i8_views(raw_k, cap, heads)
    codes[:] = 128
    codes[..., 0] = 255  # c = 127 in one channel: q . K = 127 * scale
    scales.copy_((torch.tensor(score, dtype=torch.float64) * math.sqrt(D) / math.log2(math.e) / 127).float().cuda().expand_as(scales))
    i8_views(raw_v, cap, heads)[1].copy_(torch.tensor(scale, dtype=torch.float64).float().cuda().expand(1, heads, cap))
    return raw_k, raw_v, cap


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("group", [8, 12])
# rows whose scores rise as their values shrink, each worth as much as the others, and the reverse; a row that scores
# little and is very large among very small ones; rows that score a little more and are very small after very large ones
@pytest.mark.parametrize("case", ["falling", "rising", "rising by 115", "large one", "small last"])
def test_values_of_any_size(case, group, dtype):
    heads, n, cap = 8, 64, 768  # more pairs than run at once, so that a warp goes through many blocks
    if case == "falling":
        score, scale = [0.25 * x for x in range(cap)], [2.0 ** (119 - 0.25 * x) for x in range(cap)]
    elif case == "rising":
        score, scale = [0.25 * (cap - x) for x in range(cap)], [2.0 ** (-72 + 0.25 * x) for x in range(cap)]
    elif case == "rising by 115":
        score, scale = [0.15 * (cap - x) for x in range(cap)], [2.0 ** (4 + 0.15 * x) for x in range(cap)]
    elif case == "small last":
        score, scale = [0.0] * 500 + [9.0] * (cap - 500), [2.0 ** 100] * 500 + [2.0 ** -60] * (cap - 500)
    else:
        score, scale = [300.0] * cap, [2.0 ** -60] * cap
        score[600], scale[600] = 0.0, 2.0 ** 119
    raw_k, raw_v, cap = _scaled_rows(heads, score, scale)
    kx, vx = values(raw_k, cap, heads)[0], values(raw_v, cap, heads)[0]
    q = torch.ones(n, heads * group, D, device="cuda", dtype=dtype)
    out = torch.full_like(q, float("nan"))
    d = kv.decode_seqs_desc([raw_k[0]] * n, [raw_v[0]] * n, cap, cap - 1, q, out)
    kv.decode_i8(d, heads * group, heads, D, dtype, workspace(kv.decode_i8_workspace(n, heads * group, heads)))
    want, mag, reach = attend(q[0], kx, vx, None)
    assert mag.min() > 1e-20  # far above bound()'s absolute part
    tol = bound(want, mag, reach, cap, dtype, p_f16=group > 8 and dtype == torch.bfloat16)
    if case == "rising":
        # Rows that score more than 126 below the largest: their weight 2^(score - m) is below the smallest normal f32,
        # 2^-126, for a reference m that reaches the largest score, and an f32 weight may be 0.  All that they add may be lost.
        low = torch.tensor([x < score[0] - 126 for x in score], device="cuda")
        tol = tol + attend(q[0], kx, vx.abs() * low.view(-1, 1, 1), None)[0]
    check(out[0], want, tol)
    assert all(torch.equal(x, out[0]) for x in out)


def _finite_elsewhere(got, clean, where):
    """Not finite at `where`, a mask of outputs, and bit-equal to the call on finite inputs elsewhere."""
    assert not torch.isfinite(got[where]).any()
    assert torch.equal(got[~where], clean[~where])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("group", [8, 12])
@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_queries_that_are_not_finite(cache, group, dtype, bad):
    # one head of one sequence, beside others in its tiles
    heads, n, cap, plen = 2, 5, 40, 300
    prefix = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    if cache == "i8":
        own = fill_i8(n, cap, heads, 3)[0], fill_i8(n, cap, heads, 4)[0], cap
    else:
        own = rows(3, n, cap, heads).half(), rows(4, n, cap, heads).half()
    kind = kv.I8 if cache == "i8" else kv.F16
    q = rows(5, n, heads * group, dtype=dtype)
    pos = [plen + 7 * i for i in range(n)]
    where = torch.zeros(n, heads * group, D, dtype=torch.bool, device="cuda")
    where[2, 5] = True
    broken = q.clone()
    broken[2, 5, 77] = bad
    _finite_elsewhere(_shared(prefix, own, pos, broken, heads, kind), _shared(prefix, own, pos, q, heads, kind), where)
    pos = [7 * i for i in range(n)]
    _finite_elsewhere(_shared(None, own, pos, broken, heads, kind), _shared(None, own, pos, q, heads, kind), where)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("group", [8, 12])
def test_own_rows_that_are_not_finite(group, dtype, bad):
    heads, n, cap, plen = 2, 5, 40, 300
    prefix = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    k, v = rows(3, n, cap, heads).half(), rows(4, n, cap, heads).half()
    q = rows(5, n, heads * group, dtype=dtype)
    pos = [plen + 7 * i for i in range(n)]
    clean = _shared(prefix, (k, v), pos, q, heads)
    # rows that are not attended to: slots that the sequences have not reached
    held = [[(plen + x) % cap for x in range(7 * i + 1)] for i in range(n)]
    for i in range(n):
        for slot in set(range(cap)) - set(held[i]):
            k[i, slot], v[i, slot] = bad, bad
    assert torch.equal(_shared(prefix, (k, v), pos, q, heads), clean)
    # a key: every output of its KV head's queries (with a positive element, so that the score is not -inf)
    where = torch.zeros(n, heads * group, D, dtype=torch.bool, device="cuda")
    where[3, group:] = True
    q[3, :, 50] = q[3, :, 50].abs() + 0.5
    clean = _shared(prefix, (k, v), pos, q, heads)
    keep = k[3, held[3][4], 1].clone()
    k[3, held[3][4], 1, 50] = bad
    _finite_elsewhere(_shared(prefix, (k, v), pos, q, heads), clean, where)
    k[3, held[3][4], 1] = keep
    # a value: its dimension only
    where[:] = False
    where[1, :group, 9] = True
    v[1, held[1][2], 0, 9] = bad
    _finite_elsewhere(_shared(prefix, (k, v), pos, q, heads), clean, where)


@pytest.mark.parametrize("dtype", IO)
def test_int8_rows_that_are_not_finite_beside_a_prefix(dtype):
    heads, group, n, cap, plen = 2, 8, 5, 40, 300
    prefix = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    raw_k, raw_v = fill_i8(n, cap, heads, 3)[0], fill_i8(n, cap, heads, 4)[0]
    q = rows(5, n, heads * group, dtype=dtype)
    pos = [plen + 7 * i for i in range(n)]
    clean = _shared(prefix, (raw_k, raw_v, cap), pos, q, heads, kv.I8)
    i8_views(raw_k, cap, heads)[1][4, 0, (plen + 30) % cap] = math.nan  # not reached
    assert torch.equal(_shared(prefix, (raw_k, raw_v, cap), pos, q, heads, kv.I8), clean)
    where = torch.zeros(n, heads * group, D, dtype=torch.bool, device="cuda")
    where[3, group:] = True
    i8_views(raw_v, cap, heads)[1][3, 1, (plen + 11) % cap] = math.nan
    _finite_elsewhere(_shared(prefix, (raw_k, raw_v, cap), pos, q, heads, kv.I8), clean, where)


@pytest.mark.parametrize("dtype", IO)
# heads a KV head, sequences, prefix rows: one Q tile and two, one split and several
@pytest.mark.parametrize("group,n,plen", [(8, 6, 400), (12, 25, 300), (8, 40, 5000), (16, 9, 2000)])
def test_prefix_rows_that_are_not_finite(group, n, plen, dtype):
    # rows that some sequences' windows leave out: their outputs are those of the rows that they attend to
    heads, cap = 2, 20
    prefix = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    k, v = rows(3, n, cap, heads).half(), rows(4, n, cap, heads).half()
    q = rows(5, n, heads * group, dtype=dtype)
    window = [0 if i % 4 == 0 else 1 + (plen + 10) * (i % 4) // 4 for i in range(n)]
    pos = [plen + 2 + i % 9 for i in range(n)]
    first = [p + 1 - w if w else 0 for p, w in zip(pos, window)]
    bad = [0, plen // 3, plen // 3 + 1, plen // 2 - 40]
    for j, row in enumerate(bad):
        prefix[0][row, j % 2, 5] = (math.nan, math.inf)[j // 2]
        prefix[1][row, :, 7] = (math.inf, math.nan, -math.inf, math.nan)[j]
    out = torch.full_like(q, 5.0)
    d = kv.decode_seqs_desc(k, v, cap, pos, q, out, sliding=[w > 0 for w in window], window=window)
    g = kv.shared_groups_desc([dict(k_cache=prefix[0], v_cache=prefix[1], prefix_len=plen, seqs=d)])
    kv.decode_shared(g, heads * group, heads, D, kv.F16, dtype, workspace(kv.decode_shared_workspace(1, n, heads * group, heads)))
    finite = 0
    for i in range(n):
        own = torch.arange(max(plen, first[i]), pos[i] + 1, device="cuda") % cap
        ki, vi = (torch.cat([x[min(first[i], plen):], y[i][own]]).double() for x, y in zip(prefix, (k, v)))
        want, mag, reach = attend(q[i], ki, vi, None)
        tol = bound(want, mag, reach, ki.shape[0], dtype, p_f16=dtype == torch.bfloat16)
        ok = torch.isfinite(want)
        assert torch.equal(torch.isfinite(out[i]), ok), f"sequence {i}"
        if ok.any():
            check(out[i][ok], want[ok], tol[ok], f"sequence {i}")
            finite += 1
    assert 0 < finite < n and kv.device_error() == 0
