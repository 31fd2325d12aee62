"""GPU: caches that the parts of one int8 or batched decode call may share."""
import pytest
import torch

from sf37_b200 import kv
from tests.batch_util import D, fill_i8

pytestmark = pytest.mark.gpu


def test_two_layers_read_back_into_parts_of_one_cache():
    heads, cap = 3, 20
    raw_k, kx = fill_i8(2, cap, heads, 1)
    raw_v, vx = fill_i8(2, cap, heads, 2)
    dst = [torch.full((cap, heads, D), 7.0, device="cuda", dtype=torch.float16) for _ in range(2)]
    d = kv.read_i8_desc(raw_k, raw_v, cap, [dst[0]] * 2, [dst[1]] * 2, cap, [15, 3], [8, 10])  # slots 15 to 2, and 3 to 12
    kv.read_i8(d, heads, D, torch.float16)
    for got, x in zip(dst, (kx, vx)):
        want = torch.full_like(got, 7.0)
        for layer, at in ((0, [15, 16, 17, 18, 19, 0, 1, 2]), (1, range(3, 13))):
            want[list(at)] = x[layer][list(at)].float().half()
        assert torch.equal(got, want)
