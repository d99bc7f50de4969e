"""Attention of a drafted tree where values lie far apart or near the ends of their type's range."""
import numpy as np
import pytest

from tests._gpu import note
from tests._tree import Cache, Nodes, attention, random_parents, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("elem", ["f32", "i8"])
@pytest.mark.parametrize("gap,small,large", [(200, 0.0, 4e6), (200, 0.0, 1e30), (200, 1e-35, 3e38), (140, 0.0, 1e4),
                                             (100, 0.0, 1e30), (60, 0.0, 1e10), (124, 1e-30, 3e38), (110, 1e-20, 1e38)])
@pytest.mark.parametrize("n", [3, 40])
def test_light_keys_with_large_values(dev, elem, gap, small, large, n):
    """Keys whose scores lie `gap` log2 units under the others', but whose V rows are larger by far: what
    they weigh in the sum they do, and they weigh nothing where 2^-gap is below f32's range. In front of the
    others, behind them, and among them."""
    note(f"tree ranges, light keys {elem} {gap} {small} {large} n {n}")
    rng = np.random.default_rng(1)
    h, hkv, hd, pos = 8, 2, 64, 320
    nodes = Nodes(dev, random_parents(n, rng))
    q = np.zeros((n, h, hd), np.float32)
    q[:, :, 0] = 1
    for light in (np.arange(pos + n) < 160, (np.arange(pos + n) >= 160) & (np.arange(pos + n) < pos),
                  np.arange(pos + n) % 3 == 1):
        k = np.zeros((pos + n, hkv, hd), np.float32)
        k[light, :, 0] = -gap * np.log(2)
        v = np.clip(rng.standard_normal((pos + n, hkv, hd)), -1, 1)
        v = (v * np.where(light, large, small)[:, None, None]).astype(np.float32)
        c = Cache(dev, elem, pos + n, hkv, hd, k, v, 16)
        got = c.attend(dev, q, nodes, pos, 1.0)
        want, bound = attention(q, c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), 1.0)
        # A weight below 2^-126 may be taken for zero, and a result.
        lost = 2.0 ** -gap * np.abs(c.v.astype(np.float64)).max() * (gap > 125) + 2.0 ** -125
        if elem == "i8":
            # Codes carry their block's scale, whatever the row's own size: the column's largest weight times
            # scale is at least 2^6 f16 units, a half of f16's least step 2^-25, so each of the keys is off by up
            # to 2^-31 of the largest weight times scale, and times its code, at most 127 of that scale. (Here a
            # row of zeros in a block of large rows.) A weight is at most 1 / (the heavy keys seen).
            tops = [np.abs(c.v[b:b + 16].astype(np.float64)).max() * ((~light[b:b + 16]).any()) for b in range(0, pos + n, 16)]
            lost += (pos + n) * 2.0 ** -31 * 2 * max(tops) / (~light[:pos]).sum()
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= bound + lost).all(), (np.abs(got - want) / (bound + lost)).max()
