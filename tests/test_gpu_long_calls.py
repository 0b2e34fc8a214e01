"""iq_kv_append and iq_logprobs with more tokens or rows than one launch's grid
can hold (2^32 threads)."""
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv_util import EPS32

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


def test_logprobs_of_many_rows():
    """Two logits a row: log p = -log(1 + e^-d), d the difference; the sum's
    two terms, their log and two differences are roundings of about their size."""
    say("logprobs", MANY)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(MANY, 2, generator=gen, device="cuda") * 3
    tok = torch.randint(0, 2, (MANY,), generator=gen, device="cuda")
    r = ops.logprobs(x, tok, top=1)
    xd = x.double()
    lse = torch.logsumexp(xd, 1)
    best = xd.argmax(1)
    ref = xd.gather(1, tok[:, None])[:, 0] - lse
    assert torch.equal(r.top_ids[:, 0], best)
    bound = 2 * EPS32 * (ref.abs() + 2) + 16 * EPS32
    assert torch.all((r.logprob.double() - ref).abs() <= bound)
    assert torch.all((r.top_logprobs[:, 0].double() - (xd.amax(1) - lse)).abs() <= bound)
    p = torch.softmax(xd, 1)
    ent = -(p * torch.log_softmax(xd, 1)).sum(1)
    assert torch.all((r.entropy.double() - ent).abs() <= 32 * EPS32)
