"""Evictions one after the other, on the CPU and with the plain form that
iq_kv_evict is held to (kv_util.evict_moves): `recent` of up to the last
eviction's `recent` and the tokens added since keeps the newest tokens, and one
more does not."""
import numpy as np
import pytest

from tests.kv_util import evict_moves


def evictions(rng, more, n=60, rounds=8):
    """Whether every eviction kept the newest `recent`, in their order."""
    ages = np.arange(n)
    known = n  # the last `known` rows lie in the order of their age
    good = True
    for _ in range(rounds):
        added = int(rng.integers(0, 12))
        ages = np.concatenate([ages, ages.max() + 1 + np.arange(added)])
        known += added
        # half of the evictions take as many as they may
        recent = known + more if rng.random() < 0.5 else int(rng.integers(0, known + 1))
        recent = min(recent, len(ages) - 2)
        budget = int(rng.integers(recent, len(ages) - 1)) if recent else int(rng.integers(1, len(ages) - 1))
        newest = np.sort(ages)[len(ages) - recent:]
        ages = ages[evict_moves(rng.random(len(ages)), budget, recent)]
        good &= set(newest) <= set(ages) and np.array_equal(ages[budget - recent:], newest)
        known = recent
        if len(ages) < 8:
            break
    return good


def test_recent_within_what_is_in_order():
    rng = np.random.default_rng(1)
    assert all(evictions(rng, 0) for _ in range(500))


@pytest.mark.parametrize("more", [1, 5])
def test_recent_past_what_is_in_order(more):
    rng = np.random.default_rng(2)
    assert not all(evictions(rng, more) for _ in range(500))
