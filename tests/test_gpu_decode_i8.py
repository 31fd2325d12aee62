"""GPU: decode attention over int8 caches against 64 bits on the cached values."""
import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import (D, attend, attended, bound, check, coarse_q, fill_i8, i8_views, quantise, rows, values, workspace)

pytestmark = pytest.mark.gpu


def _start(pos, cap, window):
    have = pos + 1
    return max(0, have - cap, have - window if window else 0)


def _case(caps, poss, heads, group, dtype, window=0, append=False, gate=True, scale=1.0, seed=1):
    """Runs one call over sequences of their own caps; checks every output and appended row."""
    n, qh = len(caps), heads * group
    caches = [(fill_i8(1, c, heads, seed + 10 * i)[0], fill_i8(1, c, heads, seed + 10 * i + 1, scale=3.0)[0])
              for i, c in enumerate(caps)]
    q = rows(seed + 2, n, qh, dtype=dtype, scale=scale)
    out = torch.full((n, qh, D), float("nan"), device="cuda", dtype=dtype)
    gt = rows(seed + 3, n, qh)[..., 0].contiguous() if gate else None
    new = (rows(seed + 4, n, heads, dtype=dtype), rows(seed + 5, n, heads, dtype=dtype)) if append else (None, None)
    seqs = kv.decode_seqs_desc([k[0] for k, _ in caches], [v[0] for _, v in caches], caps, poss, q, out, gate=gt,
                               k_new=new[0], v_new=new[1], sliding=window > 0, window=window)
    ws = workspace(kv.decode_i8_workspace(n, qh, heads))
    before = [(k.clone(), v.clone()) for k, v in caches]
    for _ in range(2):  # the second call finds the workspace as the first left it
        out.fill_(float("nan"))
        kv.decode_i8(seqs, qh, heads, D, dtype, ws)
        for i in range(n):
            kvals = []
            for j in range(2):
                raw = caches[i][j]
                if append:
                    c, s = quantise(new[j][i].float().cpu().numpy())
                    codes, scales = i8_views(before[i][j], caps[i], heads)
                    codes[0, poss[i] % caps[i]] = torch.from_numpy(c).cuda()
                    scales[0, :, poss[i] % caps[i]] = torch.from_numpy(s).cuda()
                assert torch.equal(raw, before[i][j]), f"cache of sequence {i}"
                kvals.append(attended(values(raw, caps[i], heads)[0], caps[i], poss[i], _start(poss[i], caps[i], window)))
            want, mag, reach = attend(q[i], kvals[0], kvals[1], None if gt is None else gt[i])
            tol = bound(want, mag, reach, kvals[0].shape[0], dtype, p_f16=group > 8 and dtype == torch.bfloat16,
                        score=coarse_q(q[i], kvals[0]) if dtype == torch.bfloat16 else 0.0)
            check(out[i], want, tol, f"sequence {i}")


IO = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("rows_", [1, 2, 15, 16, 17, 63, 64, 65, 129, 1000, 5000])
def test_lengths(rows_, dtype):
    _case([rows_], [rows_ - 1], 8, 8, dtype)


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 3), (8, 5), (3, 8), (2, 9), (8, 12), (1, 16)])
def test_head_layouts(heads, group, dtype):
    _case([70, 301], [69, 300], heads, group, dtype, append=True)


@pytest.mark.parametrize("dtype", IO)
def test_rings_windows_and_appends(dtype):
    # full rings that have wrapped, caps below a block, windows inside and over the cap
    _case([100, 7, 1, 64], [250, 20, 5, 63], 4, 8, dtype, append=True)
    _case([100, 512, 40, 33], [250, 700, 500, 5], 4, 8, dtype, window=32, append=True)
    _case([3000], [9000], 8, 12, dtype, window=2900, append=True, gate=False)


def test_ragged_batch_of_many():
    n = 40
    _case([1 + 37 * i for i in range(n)], [37 * i for i in range(n)], 2, 4, torch.bfloat16, append=True)


def test_more_sequences_than_a_launch_holds():
    n = 300
    _case([5 + i % 3 for i in range(n)], [i % 11 for i in range(n)], 1, 2, torch.float32, append=True)


def test_many_splits_and_waves():
    _case([40000], [39999], 8, 8, torch.float32)
    _case([9000, 20000, 3], [8999, 19000, 2], 16, 8, torch.bfloat16)


@pytest.mark.parametrize("scale", [1e-6, 6.0, 300.0])
def test_peaked_and_flat_scores(scale):
    _case([700], [699], 4, 8, torch.float32, scale=scale)


def test_value_scales_far_apart():
    # value rows from 1e-12 to 1e12: the kernel's weights keep the largest contribution in f16's range
    heads, cap = 2, 200
    raw_k, kvals = fill_i8(1, cap, heads, 3)
    raw_v, _ = fill_i8(1, cap, heads, 4)
    _, scales = i8_views(raw_v, cap, heads)
    for order in (torch.linspace(-12, 12, cap), torch.linspace(12, -12, cap)):
        scales.copy_((10 ** order.double()).float().cuda().expand_as(scales))
        v = values(raw_v, cap, heads)
        q = rows(5, 1, 16)
        out = torch.empty_like(q)
        ws = workspace(kv.decode_i8_workspace(1, 16, heads))
        kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, cap - 1, q, out), 16, heads, D, q.dtype, ws)
        want, mag, reach = attend(q[0], kvals[0], v[0], None)
        check(out[0], want, bound(want, mag, reach, cap, q.dtype, False))


def test_empty_rows_and_zero_window():
    heads, cap = 2, 20
    raw_k, raw_v = fill_i8(1, cap, heads, 1)[0], fill_i8(1, cap, heads, 2)[0]
    q = rows(1, 1, 16)
    out = torch.full_like(q, float("nan"))
    ws = workspace(kv.decode_i8_workspace(1, 16, heads))
    kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, 9, q, out, sliding=True, window=0), 16, heads, D, q.dtype, ws)
    assert (out == 0).all()


def test_nan_rows_show_only_where_they_are_attended_to():
    heads, cap = 2, 64
    raw_k, raw_v = fill_i8(1, cap, heads, 1)[0], fill_i8(1, cap, heads, 2)[0]
    q = rows(1, 1, 16)
    ws = workspace(kv.decode_i8_workspace(1, 16, heads))

    def run(pos):
        out = torch.empty_like(q)
        kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, pos, q, out), 16, heads, D, q.dtype, ws)
        return out

    clean = run(40)
    bad = rows(9, 1, 1, heads)
    bad[0, 0, 1, 5] = float("nan")  # head 1 only
    for slot in (41, 50, 63):       # rows that the query does not attend to
        kv.append_i8(kv.append_i8_desc(raw_k, raw_v, cap, slot, bad, bad), heads, D, bad.dtype)
    assert torch.equal(run(40), clean)
    kv.append_i8(kv.append_i8_desc(raw_k, raw_v, cap, 3, bad, bad), heads, D, bad.dtype)
    got = run(40)
    assert torch.isfinite(got[0, :8]).all() and torch.isnan(got[0, 8:]).all()


def test_repeats_are_bit_equal():
    heads, cap = 8, 6000
    raw_k, raw_v = fill_i8(2, cap, heads, 1)[0], fill_i8(2, cap, heads, 2)[0]
    q = rows(1, 2, 64)
    ws = workspace(kv.decode_i8_workspace(2, 64, heads))
    outs = []
    for _ in range(3):
        out = torch.empty_like(q)
        kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, [5999, 4000], q, out), 64, heads, D, q.dtype, ws)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_graphs_with_a_workspace_each_run_side_by_side():
    heads, cap, n = 8, 3000, 2
    raw_k, raw_v = fill_i8(n, cap, heads, 1)[0], fill_i8(n, cap, heads, 2)[0]
    qs = [rows(s, n, 64) for s in (1, 2)]
    outs, graphs, streams, keep = [torch.empty_like(q) for q in qs], [], [], []
    want = []
    for q in qs:
        o = torch.empty_like(q)
        kv.decode_i8(kv.decode_seqs_desc(raw_k, raw_v, cap, 2999, q, o), 64, heads, D, q.dtype,
                     workspace(kv.decode_i8_workspace(n, 64, heads)))
        want.append(o)
    torch.cuda.synchronize()
    for q, o in zip(qs, outs):
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        ws = workspace(kv.decode_i8_workspace(n, 64, heads))
        d = kv.decode_seqs_desc(raw_k, raw_v, cap, 2999, q, o)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            kv.decode_i8(d, 64, heads, D, q.dtype, ws, stream=s)
        graphs.append(g)
        streams.append(s)
        keep += [ws, d]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_chunked_prefill_and_decode_over_an_i8_cache():
    """A prompt in two chunks (append, read back, prefill), then decode steps: the calls of a serving loop."""
    heads, qh, cap = 2, 16, 400
    raw_k, raw_v = (torch.zeros(kv.i8_cache_bytes(cap, heads), dtype=torch.uint8, device="cuda") for _ in range(2))
    stage = [torch.zeros(cap, heads, D, device="cuda", dtype=torch.float16) for _ in range(2)]
    pos = 0
    for chunk in (130, 77):
        k, v = rows(pos + 1, chunk, heads, dtype=torch.bfloat16), rows(pos + 2, chunk, heads, dtype=torch.bfloat16)
        q = rows(pos + 3, chunk, qh, dtype=torch.bfloat16)
        out = torch.empty(chunk, qh, D, device="cuda")
        kv.append_i8(kv.append_i8_desc([raw_k], [raw_v], cap, pos, [k], [v]), heads, D, k.dtype)
        kv.read_i8(kv.read_i8_desc([raw_k], [raw_v], cap, [stage[0]], [stage[1]], cap, 0, pos + chunk), heads, D, torch.float16)
        kv.prefill(stage[0], stage[1], cap, q, None, out, pos, chunk, qh, heads, D, kv.F16)
        kx, vx = values(raw_k[None], cap, heads)[0], values(raw_v[None], cap, heads)[0]
        for t in (0, chunk - 1):
            # the staged rows are rounded to f16: 2^-11 of a key or value, in the score and the value
            want, mag, reach = attend(q[t], kx[:pos + t + 1], vx[:pos + t + 1], None)
            check(out[t], want, bound(want, mag, reach, pos + t + 1, torch.float32, True) +
                  2 * mag * (2.0 ** -11 * (1 + 0.6932 * reach)))
        pos += chunk
    ws = workspace(kv.decode_i8_workspace(1, qh, heads))
    for step in range(3):
        k, v, q = rows(90 + step, 1, heads), rows(95 + step, 1, heads), rows(80 + step, 1, qh)
        out = torch.empty_like(q)
        kv.decode_i8(kv.decode_seqs_desc([raw_k], [raw_v], cap, pos, q, out, k_new=k, v_new=v), qh, heads, D, q.dtype, ws)
        pos += 1
        kx, vx = values(raw_k[None], cap, heads)[0], values(raw_v[None], cap, heads)[0]
        # half a scale: at most max|x| / 254 off each element of the new row, and an f32 product
        assert ((kx[pos - 1] - k[0].double()).abs() <= k[0].double().abs().amax(-1, keepdim=True) / 253.9).all()
        want, mag, reach = attend(q[0], kx[:pos], vx[:pos], None)
        check(out[0], want, bound(want, mag, reach, pos, q.dtype, False))
