"""GPU: decode attention over a shared prefix against 64 bits, and against the
same sequences decoded one by one."""
import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, attend, attended, bound, check, coarse_q, fill_i8, rows, values, workspace

pytestmark = pytest.mark.gpu

IO = [torch.float32, torch.bfloat16]


def _case(groups, heads, group, dtype, cache="f16", append=False, scale=1.0, seed=1, gate=True):
    """groups: list of (prefix_len, prefix_cap, [(own cap, own rows, window)]).  Checks every output."""
    qh, i8 = heads * group, cache == "i8"
    made, descs = [], []
    for gi, (plen, pcap, seqs) in enumerate(groups):
        s0, n = seed + 1000 * gi, len(seqs)
        pk, pv = rows(s0, max(pcap, 1), heads).half(), rows(s0 + 1, max(pcap, 1), heads).half()
        pk[plen:], pv[plen:] = float("nan"), float("nan")  # beyond the prefix: never read as values
        if i8:
            ks = [fill_i8(1, c, heads, s0 + 10 + 2 * i)[0][0] for i, (c, _, _) in enumerate(seqs)]
            vs = [fill_i8(1, c, heads, s0 + 11 + 2 * i)[0][0] for i, (c, _, _) in enumerate(seqs)]
        else:
            ks = [rows(s0 + 10 + 2 * i, c, heads).half() for i, (c, _, _) in enumerate(seqs)]
            vs = [rows(s0 + 11 + 2 * i, c, heads).half() for i, (c, _, _) in enumerate(seqs)]
        q = rows(s0 + 2, n, qh, dtype=dtype, scale=scale)
        out = torch.full((n, qh, D), float("nan"), device="cuda", dtype=dtype)
        gt = rows(s0 + 3, n, qh)[..., 0].contiguous() if gate else None
        new = (rows(s0 + 4, n, heads, dtype=dtype), rows(s0 + 5, n, heads, dtype=dtype)) if append else (None, None)
        pos = [plen + own - 1 for _, own, _ in seqs]
        d = kv.decode_seqs_desc(ks, vs, [c for c, _, _ in seqs], pos, q, out, gate=gt, k_new=new[0], v_new=new[1],
                                sliding=[w > 0 for _, _, w in seqs], window=[w for _, _, w in seqs])
        made.append((plen, seqs, pk, pv, ks, vs, q, out, gt, new, pos))
        descs.append(dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d))
    g = kv.shared_groups_desc(descs)
    ws = workspace(kv.decode_shared_workspace(len(groups), sum(len(x[2]) for x in groups), qh, heads))
    for _ in range(2):
        for m in made:
            m[7].fill_(float("nan"))
        kv.decode_shared(g, qh, heads, D, kv.I8 if i8 else kv.F16, dtype, ws)
        for plen, seqs, pk, pv, ks, vs, q, out, gt, new, pos in made:
            for i, (cap, own, window) in enumerate(seqs):
                first = max(0, pos[i] + 1 - window) if window else 0
                kx, vx = (values(x[i][None], cap, heads)[0] if i8 else x[i].double() for x in (ks, vs))
                if append and not i8:
                    slot = pos[i] % cap
                    assert torch.equal(ks[i][slot], new[0][i].half()) and torch.equal(vs[i][slot], new[1][i].half())
                kx = torch.cat([pk[first:plen].double(), attended(kx, cap, pos[i], max(first, plen))])
                vx = torch.cat([pv[first:plen].double(), attended(vx, cap, pos[i], max(first, plen))])
                want, mag, reach = attend(q[i], kx, vx, None if gt is None else gt[i])
                tol = bound(want, mag, reach, kx.shape[0], dtype, p_f16=dtype == torch.bfloat16,
                            score=coarse_q(q[i], kx) if i8 and dtype == torch.bfloat16 else 0.0)
                check(out[i], want, tol, f"prefix {plen} sequence {i}")
    assert kv.device_error() == 0


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("plen", [1, 2, 127, 128, 129, 255, 257, 1000])
def test_prefix_lengths(plen, dtype):
    _case([(plen, plen + plen % 3, [(40, 1, 0), (40, 33, 0)])], 2, 8, dtype)


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 49])
def test_batch_sizes(n, dtype):
    _case([(300, 300, [(64, 1 + (i * 7) % 64, 0) for i in range(n)])], 2, 8, dtype, append=True)


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 3), (8, 5), (2, 9), (4, 12), (1, 16), (2, 4)])
def test_head_layouts(heads, group, dtype):
    _case([(260, 300, [(50, 1 + 5 * i, 0) for i in range(9)])], heads, group, dtype, append=True)


@pytest.mark.parametrize("dtype", IO)
@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_windows(cache, dtype):
    # windows that cover all, part and none of the prefix, or a single row of it; own rings that have wrapped
    seqs = [(100, 20, 0), (100, 20, 5000), (100, 20, 150), (100, 20, 21), (100, 20, 20), (30, 90, 30), (100, 90, 100), (8, 3, 1)]
    _case([(333, 400, seqs)], 2, 8, dtype, cache, append=True)
    _case([(333, 400, [(100, 20, 21), (100, 20, 20), (100, 20, 40)])], 2, 12, dtype, cache)


@pytest.mark.parametrize("dtype", IO)
def test_groups_with_their_own_prefixes(dtype):
    _case([(700, 700, [(20, 3, 0)] * 3), (0, 1, [(20, 3, 0), (20, 20, 0)]), (5, 9, [(20, 1, 0)] * 20),
           (260, 260, [(20, 7, 5)])], 2, 8, dtype, append=True)


def test_more_groups_and_sequences_than_a_launch_holds():
    _case([(100 + i, 130, [(9, 1 + (i + j) % 9, 0) for j in range(40)]) for i in range(11)], 1, 4, torch.bfloat16, append=True)


def test_no_own_rows_yet():
    _case([(300, 300, [(16, 0, 0), (16, 0, 100), (16, 4, 0)])], 2, 8, torch.float32)


@pytest.mark.parametrize("dtype", IO)
def test_many_splits(dtype):
    _case([(20000, 20000, [(300, 1 + 60 * i, 0) for i in range(5)])], 8, 8, dtype, append=True)
    _case([(9001, 9001, [(300, 1 + 6 * i, 0) for i in range(40)])], 8, 8, dtype, "i8", append=True)


@pytest.mark.parametrize("scale", [1e-6, 6.0, 100.0])
@pytest.mark.parametrize("dtype", IO)
def test_peaked_and_flat_scores(scale, dtype):
    _case([(900, 900, [(64, 30, 0)] * 4)], 2, 8, dtype, scale=scale)


def test_a_rising_prefix_rescales():
    # scores that rise along the prefix move the running maximum in every tile
    heads, qh, plen = 2, 16, 1500
    pk = (rows(1, plen, heads) + torch.linspace(0, 40, plen, device="cuda").view(-1, 1, 1) / 11.3).half()
    pv = rows(2, plen, heads).half()
    ko, vo = rows(3, 2, 10, heads).half(), rows(4, 2, 10, heads).half()
    for dtype in IO:
        q = (rows(5, 2, qh).abs() + 0.1).to(dtype)
        out = torch.empty_like(q)
        d = kv.decode_seqs_desc(ko, vo, 10, plen + 9, q, out)
        ws = workspace(kv.decode_shared_workspace(1, 2, qh, heads))
        kv.decode_shared(kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)]), qh, heads, D, kv.F16,
                         dtype, ws)
        at = torch.arange(plen, plen + 10, device="cuda") % 10
        for i in range(2):
            want, mag, reach = attend(q[i], torch.cat([pk, ko[i][at]]).double(), torch.cat([pv, vo[i][at]]).double(), None)
            check(out[i], want, bound(want, mag, reach, plen + 10, dtype, dtype == torch.bfloat16))


def test_against_one_by_one_decode():
    """The same sequences through sf37kv_decode, each with the prefix in its own cache."""
    heads, qh, plen, n, cap = 8, 64, 777, 5, 64
    pk, pv = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    ko, vo = rows(3, n, cap, heads).half(), rows(4, n, cap, heads).half()
    q, gate = rows(5, n, qh), rows(6, n, qh)[..., 0].contiguous()
    out, single = torch.empty_like(q), torch.empty_like(q)
    own = [1, 9, 30, 63, 64]
    pos = [plen + x - 1 for x in own]
    d = kv.decode_seqs_desc(ko, vo, cap, pos, q, out, gate=gate)
    ws = workspace(kv.decode_shared_workspace(1, n, qh, heads))
    kv.decode_shared(kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)]), qh, heads, D, kv.F16,
                     q.dtype, ws)
    for i in range(n):
        at = torch.arange(plen, pos[i] + 1, device="cuda") % cap
        k, v = torch.cat([pk, ko[i][at]]).contiguous(), torch.cat([pv, vo[i][at]]).contiguous()
        kv.decode([dict(k_cache=k, v_cache=v, cap=k.shape[0], pos=pos[i], q=q[i], gate=gate[i], out=single[i])], qh, heads, D,
                  kv.F16)
        want, mag, reach = attend(q[i], k.double(), v.double(), gate[i])
        check(out[i], single[i].double(), 2 * bound(want, mag, reach, k.shape[0], q.dtype, False), f"sequence {i}")


def test_side_stream_graph_and_bit_equal_repeats():
    heads, qh, plen, n, cap = 8, 64, 2000, 20, 200
    pk, pv = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    ko, vo = rows(3, n, cap, heads).half(), rows(4, n, cap, heads).half()
    q = rows(5, n, qh, dtype=torch.bfloat16)
    outs = [torch.empty_like(q) for _ in range(2)]
    ds = [kv.decode_seqs_desc(ko, vo, cap, plen + 150, q, o) for o in outs]
    gs = [kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)]) for d in ds]
    wss = [workspace(kv.decode_shared_workspace(1, n, qh, heads)) for _ in range(2)]
    kv.decode_shared(gs[0], qh, heads, D, kv.F16, q.dtype, wss[0])
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        kv.decode_shared(gs[1], qh, heads, D, kv.F16, q.dtype, wss[1], stream=s)
    for _ in range(4):
        outs[1].fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
    assert kv.device_error() == 0
