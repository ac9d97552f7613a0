"""Paged-cache operators at the edges of what their documentation allows: items that follow each other without a pause, dominant keys, offsets that overlap, memory that is shared."""
import random

import pytest
import torch

import paged_reference as R
from kyojin_mac_b200 import ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(qn):
    return _i32([sum(qn[:i]) for i in range(len(qn) + 1)])


# ------------------------------------------------------------------------------------------------ many short items
@pytest.mark.parametrize("hq,hkv,d,lo,hi", [(8, 8, 64, 17, 60), (4, 4, 128, 17, 60), (16, 4, 64, 20, 90), (8, 8, 64, 100, 150), (6, 6, 128, 100, 280)])
def test_short_items_follow_each_other(hq, hkv, d, lo, hi):
    """Several hundred short requests: each CTA goes through dozens of items of one key tile or two, with one query tile or two, one behind the other. Every call gives the
    same, all rows are written and no wait runs out."""
    r = random.Random(hq + d + hi)
    qn = [r.randint(lo, hi) for _ in range(300)]
    k, v, table = R.pool(qn, 16, hkv, d, F16, 31)
    lens, cu = _i32(qn), _offsets(qn)
    q = torch.randn((sum(qn), hq, d), device="cuda").to(F16)
    first = ops.paged_attention(q, k, v, table, lens, cu, hi)
    for _ in range(40):
        out = torch.full_like(q, 9.0)
        assert torch.equal(ops.paged_attention(q, k, v, table, lens, cu, hi, out=out), first)
    ops.check_device_status()
    want, tol = R.attention(q, k, v, table, lens, cu, d ** -0.5, 0, 0)
    assert ((first.cpu().double() - want).abs() <= tol).all()
