"""Outputs between the pages of a cache that is part of a larger tensor."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_outputs_between_the_pages(dtype):
    """Pages of 16 slots with as much room behind each: what is made there is
    what is made elsewhere, and the pages keep what they hold."""
    hk, d, page, pages = 2, 64, 16, 6
    gen = torch.Generator(device="cuda").manual_seed(3)
    big = [torch.zeros(pages, 8 * page, hk, d, dtype=dtype, device="cuda") for _ in range(2)]
    size = big[0].element_size()
    sc = [torch.zeros(pages, 2, hk, device="cuda") for _ in range(2)] if size == 1 else [None, None]
    cache = ops.KvCache(*[b[:, :page] for b in big], *sc)

    def room(p, *shape):  # behind page p
        n = int(np.prod(shape))
        return big[0][p, page:].reshape(-1)[:4 * n // size].view(torch.float32).view(shape)
    assert room(0, 3, 4, d).data_ptr() == big[0][0, page:].data_ptr()
    table = torch.tensor([[3, 1], [5, 0]], dtype=torch.int32, device="cuda")
    lens, starts = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.tensor([0, 20, 23], dtype=torch.int32, device="cuda")
    x = [torch.randn(23, hk, d, device="cuda", generator=gen) for _ in range(2)]
    first = torch.randn(4, hk, d, device="cuda", generator=gen)
    none, four = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    ops.kv_extend(None, first, first, None, None, cache, table[1:], none, starts=four)
    q = torch.randn(23, 1, d, device="cuda", generator=gen)
    say("extend", dtype)
    got = ops.kv_extend(q, *x, None, None, cache, table, lens, starts=starts, q_out=room(2, 23, 1, d))
    assert torch.equal(got, q)
    lens, ends = lens + torch.tensor([20, 3], dtype=torch.int32, device="cuda"), torch.tensor([0, 20, 27], dtype=torch.int32, device="cuda")
    want = ops.kv_read(cache, table, ends, T=27)
    say("read", dtype)
    got = ops.kv_read(cache, table, ends, out=(room(1, 27, hk, d), None))
    assert torch.equal(got[0], want[0])
    q = torch.randn(2, 4, d, device="cuda", generator=gen)
    want_out = ops.attn_decode(q, cache, table, lens, window=40)
    say("attention", dtype)
    assert torch.equal(ops.attn_decode(q, cache, table, lens, window=40, out=room(4, 2, 4, d)), want_out)
    assert all(torch.equal(a, b) for a, b in zip(ops.kv_read(cache, table, ends, T=27), want))
    inside = big[0][1].reshape(-1).view(torch.float32)[64:64 + 23 * d].view(23, 1, d)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.kv_extend(torch.zeros_like(inside), *x, None, None, cache, table, lens, starts=starts, q_out=inside)
