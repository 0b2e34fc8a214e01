"""CachedDecodeStep with rows that take no token."""
import pytest
import torch

from tests.test_gpu_cached_decode import build

pytestmark = pytest.mark.gpu


def state(step, b):
    return [w[b].clone() for w in step.weights]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("length", [-1, -40, -2 ** 31])
def test_idle_rows(length):
    """A row of negative length stays idle: NaN logits, nothing of it changes,
    and the row beside it does not notice."""
    step, twin = (build(35, 2)[2] for _ in range(2))
    for it in range(3):
        step.step(it)
        twin.step(it)
    step.lens[1] = length
    kept = state(step, 1)
    keys = [c.k.clone() for c in step.caches]
    for it in range(3, 6):
        step.step(it)
        twin.step(it)
        assert torch.isnan(step.logits[1]).all() and torch.equal(step.logits[0], twin.logits[0])
        assert step.lens.cpu().tolist() == [it + 1, length]
    assert same(state(step, 1), kept) and same(state(step, 0), state(twin, 0))
    p = step.table[1].long()
    for c, k in zip(step.caches, keys):
        assert torch.equal(c.k[p].view(torch.int16), k[p].view(torch.int16))
    step.evict(4, 2)
    assert step.lens.cpu().tolist() == [4, length]
