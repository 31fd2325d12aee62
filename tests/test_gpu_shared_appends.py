"""GPU: what decode over a shared prefix writes to the sequences' own caches: the appended row, and nothing else."""
import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, i8_cache, i8_views, quantise, rows, workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cache", ["i8", "f16"])
# few pairs of sequence and KV head, more than are joined by the decode launch itself, and rows in several splits
@pytest.mark.parametrize("n,heads,group,cap", [(3, 2, 8, 70), (9, 8, 5, 33), (40, 2, 12, 50), (2, 8, 8, 3000)])
def test_whole_caches(n, heads, group, cap, cache, dtype):
    plen, qh = 300, heads * group
    pk, pv = rows(1, plen, heads).half(), rows(2, plen, heads).half()
    if cache == "i8":
        own = [i8_cache(n, cap, heads, 0x7B) for _ in range(2)]
        for x in own:
            i8_views(x, cap, heads)[1].fill_(0.01)
    else:
        own = [rows(s, n, cap, heads).half() for s in (3, 4)]
    want = [x.clone() for x in own]
    prefix = pk.clone(), pv.clone()
    out = torch.empty(n, qh, D, device="cuda", dtype=dtype)
    length = [1 + (i * (cap - 1)) // max(1, n - 1) for i in range(n)]
    ws = workspace(kv.decode_shared_workspace(1, n, qh, heads))
    for step in range(2 + cap // 30):  # the longest one wraps its ring; its window holds what is left
        new = rows(10 + step, n, heads, dtype=dtype), rows(20 + step, n, heads, dtype=dtype, scale=30.0)
        q = rows(30 + step, n, qh, dtype=dtype)
        pos = [plen + x - 1 + step for x in length]
        d = kv.decode_seqs_desc(own[0], own[1], cap, pos, q, out, k_new=new[0], v_new=new[1], sliding=True, window=cap)
        kv.decode_shared(kv.shared_groups_desc([dict(k_cache=pk, v_cache=pv, prefix_len=plen, seqs=d)]), qh, heads, D,
                         kv.I8 if cache == "i8" else kv.F16, dtype, ws)
        for x, y in zip(want, new):
            for i in range(n):
                slot = pos[i] % cap
                if cache == "i8":
                    c, s = quantise(y[i].float().cpu().numpy())
                    codes, scales = i8_views(x[i:i + 1], cap, heads)
                    codes[0, slot], scales[0, :, slot] = torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda()
                else:
                    x[i, slot] = y[i].half()
        for got, x in zip(own, want):
            assert torch.equal(got.view(torch.uint8), x.view(torch.uint8)), f"step {step}"
    assert torch.equal(pk, prefix[0]) and torch.equal(pv, prefix[1]) and torch.isfinite(out).all()
    assert kv.device_error() == 0
