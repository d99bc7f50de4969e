"""Plan and walk of one tree on the device agree with each other."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._tree import random_parents, u32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 3, 33, 40, 256])
@pytest.mark.parametrize("seed", range(4))
def test_walk_follows_the_plan(dev, n, seed):
    """The accepted path is the last accepted node's own mask, and as long as its depth says."""
    note(f"walk follows the plan {n} {seed}")
    rng = np.random.default_rng(100 * seed + n)
    parents = random_parents(n, rng, width=(2, 4, 9, 1)[seed])
    tokens = rng.integers(0, 3, n).astype(np.uint32)
    # Answers that lead to a leaf drawn at random, by the first child of each node on the way.
    sampled = rng.integers(0, 3, n).astype(np.uint32)
    node = int(rng.integers(0, n))
    while node > 0:
        sampled[parents[node]] = tokens[node]
        node = parents[node]
    pt = eb.Tensor.from_array(dev, np.asarray(parents, np.int32))
    tt, st = (eb.Tensor.from_u32(dev, (n,), x) for x in (tokens, sampled))
    masks, depths = eb.Tensor.empty(dev, (n, -(-n // 32)), eb.DType.U32), eb.Tensor.empty(dev, (n,), eb.DType.U32)
    path, emitted = (eb.Tensor.empty(dev, (n,), eb.DType.U32) for _ in range(2))
    count = eb.Tensor.empty(dev, (1,), eb.DType.U32)
    rec = eb.Recorder(dev)
    eb.tree_plan(rec, pt, masks, depths, n)
    eb.tree_accept(rec, tt, pt, st, path, emitted, count, n)
    rec.submit()
    c = int(u32(count)[0])
    way, mask = u32(path)[:c].tolist(), u32(masks)
    last = way[-1]
    bits = [j for j in range(n) if mask[last, j // 32] >> np.uint32(j % 32) & 1]
    assert way == bits and u32(depths)[last] == c - 1 and u32(depths)[way].tolist() == list(range(c))
    assert u32(emitted)[:c].tolist() == sampled[way].tolist()
    for a, b in zip(way, way[1:]):
        assert parents[b] == a and tokens[b] == sampled[a]
    assert not any(parents[j] == last and tokens[j] == sampled[last] for j in range(n))
