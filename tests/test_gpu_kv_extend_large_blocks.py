"""iq_kv_extend where a block has so many older tokens that their 16-byte
pieces pass 2^31."""
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say

pytestmark = pytest.mark.gpu


def test_a_block_of_more_than_2_31_pieces_grows():
    """2^27 + 3 older tokens of 256 int8 codes in one block (16 pieces each),
    whose scale of keys doubles and whose scale of values stays."""
    older, d = 2 ** 27 + 3, 256
    page = older + 13
    if torch.cuda.mem_get_info()[0] < 3 * page * d:
        pytest.skip("two pools of 34 GB")
    k, v = (torch.full((1, page, 1, d), c, dtype=torch.int8, device="cuda") for c in (100, 30))
    ks, vs = (torch.ones(1, 1, 1, device="cuda") for _ in range(2))
    cache = ops.KvCache(k, v, ks, vs)
    k[0, older:] = 77
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    lens, starts = zero + older, torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 1, 1, d, device="cuda")
    x[:, 0, 0, 7] = torch.tensor([254.0, 127.0], device="cuda")
    say("extend", older)
    torch.cuda.synchronize()
    ops.kv_extend(None, x[0], x[1], None, None, cache, zero[None], lens, starts=starts)
    torch.cuda.synchronize()
    assert float(ks) == 2.0 and float(vs) == 1.0
    for a in range(0, older, 2 ** 24):
        b = min(a + 2 ** 24, older)
        assert bool((k[0, a:b] == 50).all()) and bool((v[0, a:b] == 30).all()), a
    new = torch.zeros(2, d, dtype=torch.int8)
    new[:, 7] = 127
    assert torch.equal(k[0, older, 0].cpu(), new[0]) and torch.equal(v[0, older, 0].cpu(), new[1])
    assert bool((k[0, older + 1:] == 77).all()) and bool((v[0, older + 1:] == 30).all())
    del cache, k, v
    torch.cuda.empty_cache()
