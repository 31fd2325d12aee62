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
