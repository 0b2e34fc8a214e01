"""iq_kv_append with more tokens than one launch's grid can hold (2^32 threads)."""
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say

pytestmark = pytest.mark.gpu

MANY = 2 ** 24 + 5


def test_append_of_many_tokens():
    say("append", MANY)
    cache = ops.alloc_kv(3, 16, 1, 8)
    q = torch.arange(MANY * 8, device="cuda", dtype=torch.float32).view(MANY, 1, 8)
    k, v = (torch.arange(MANY, device="cuda") % n for n in (251, 241))
    at = torch.tensor([0, 1, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, 2 ** 24 - 1, 2 ** 24, MANY - 1], device="cuda")
    slots = torch.full((MANY,), -1, dtype=torch.int64, device="cuda")
    slots[at] = torch.arange(len(at), device="cuda") * 5 + 3
    wide = lambda x: x.float()[:, None, None].expand(MANY, 1, 8).contiguous()  # noqa: E731
    out = ops.kv_append(q, wide(k), wide(v), None, slots, None, cache)
    assert torch.equal(out, q)
    for x, pool in ((k, cache.k), (v, cache.v)):
        want = torch.zeros(48, dtype=torch.bfloat16, device="cuda")
        want[slots[at]] = x[at].to(torch.bfloat16)  # (below 256: exact)
        assert torch.equal(pool.view(48, 8), want[:, None].expand(48, 8))
