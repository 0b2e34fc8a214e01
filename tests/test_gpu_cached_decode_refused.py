"""CachedDecodeStep with tokens that find no place (full pages, a page that is
none), idle rows and rows that the caller sets: nothing of the row changes, the other
rows do not notice, and the row goes on once there is a place."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.test_gpu_cached_decode import build, check_layers

pytestmark = pytest.mark.gpu


def state(step, b):
    return [w[b].clone() for w in step.weights]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_full_rows_keep_their_weights_and_can_be_cut():
    """Two refused steps on full rows, an eviction and a step: the same bits as
    without the refused steps."""
    runs = []
    for extra in (2, 0):
        rng, host, step, table = build(31, 2, pages=2)
        for it in range(32):
            step.step(it)
        kept = [state(step, b) for b in range(2)]
        for it in range(extra):
            step.step(100 + it)
            assert torch.isnan(step.logits).all()
            assert all(same(state(step, b), kept[b]) for b in range(2))
        assert all(torch.isfinite(w).all() for w in step.weights)
        step.evict(20, 5)
        assert step.lens.cpu().tolist() == [20, 20]
        step.step([7, 8])
        assert torch.isfinite(step.logits).all()
        assert step.lens.cpu().tolist() == [21, 21] and step.held.cpu().tolist() == [21, 21]
        assert step.positions.cpu().tolist() == [33, 33]
        runs.append([step.logits.clone(), *step.weights, *(c.k.nan_to_num(9.0) for c in step.caches)])
    assert same(*runs)


@pytest.mark.parametrize("bad", [-1, -7, "pool", 2 ** 31 - 1])
def test_missing_page_is_made_good(bad):
    rng, host, step, table = build(32, 2, pages=2)
    twin = build(32, 2, pages=2)[2]
    if bad == "pool":
        bad = step.caches[0].pages
    step.table[1, 1] = bad
    for it in range(16):
        step.step(it)
        twin.step(it)
    kept = state(step, 1)
    for it in range(16, 19):
        step.step(it)
        twin.step(it)
        assert torch.isnan(step.logits[1]).all()
        assert torch.equal(step.logits[0], twin.logits[0])
        assert same(state(step, 1), kept) and same(state(step, 0), state(twin, 0))
    assert step.held.cpu().tolist() == [19, 16] and step.positions.cpu().tolist() == [19, 16]
    step.table[1, 1] = int(table[1, 1])
    for n in (17, 18):
        sums = [w.double().cpu().numpy() for w in step.weights]
        step.step([n, n + 50])
        torch.cuda.synchronize()
        check_layers(step, host, table, [n + 3, n], [n + 2, n - 1], sums)
        for w, s in zip(step.weights, sums):
            assert np.allclose(w.cpu().numpy(), s, rtol=1e-4, atol=0)
    assert torch.isfinite(step.logits).all()
    step.evict(10, 4)
    assert step.lens.cpu().tolist() == [10, 10] and step.held.cpu().tolist() == [10, 10]


def test_rows_that_the_caller_sets():
    """A new sequence in a full row; a length set back; the row beside them."""
    rng, host, step, table = build(33, 2, pages=2)
    for it in range(34):
        step.step(it)
    step.lens[0], step.positions[0] = 0, 0
    for w in step.weights:
        w[0] = 0
    step.lens[1], step.positions[1] = 30, 30
    sums = [w.double().cpu().numpy() for w in step.weights]
    step.step(5)
    torch.cuda.synchronize()
    assert step.lens.cpu().tolist() == [1, 31] and step.held.cpu().tolist() == [1, 31]
    check_layers(step, host, table, [1, 31], [0, 30], sums)


def test_refused_rows_in_a_graph():
    """Captured once, replayed over full pages and an eviction: as eager."""
    runs = []
    for graph in (False, True):
        rng, host, step, table = build(34, 2, pages=2)
        step.table[1, 1] = -1
        s = torch.cuda.Stream()
        ops.init(0, s)
        torch.cuda.synchronize()
        g, got = None, []
        for it in range(40):
            step.ids.fill_(it)
            torch.cuda.synchronize()
            if not graph or it == 0:
                with torch.cuda.stream(s):
                    step.step()
            else:
                if g is None:
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=s):
                        step.step()
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            if it == 20:
                step.table[1, 1] = int(table[1, 1])
            if it == 36:
                with torch.cuda.stream(s):
                    step.evict(12, 3)
            torch.cuda.synchronize()
            got.append([x.clone().nan_to_num(77.0) for x in (step.logits, step.lens, step.held, *step.weights)])
        runs.append(got)
    assert all(same(a, b) for a, b in zip(*runs))


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
