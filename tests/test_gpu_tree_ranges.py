"""Attention of a drafted tree where values lie far apart or near the ends of their type's range."""
import numpy as np
import pytest

from tests._gpu import note
from tests._tree import Cache, Nodes, attention, random_parents, rows, visible
from tests.test_gpu_tree_plans import launch

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


@pytest.mark.parametrize("power", [100, 116, 119, -100, -116, -119])
@pytest.mark.parametrize("n", [3, 40])
def test_keys_and_queries_of_unlike_size(dev, power, n):
    """f32 K rows at one end of the range and queries at the other: ordinary scores."""
    note(f"tree ranges, K 2^{power} n {n}")
    rng = np.random.default_rng(2)
    h, hkv, hd, pos = 8, 2, 64, 500
    nodes = Nodes(dev, random_parents(n, rng))
    # Multiples of 2^-6 up to 2^6: exact at either end.
    k = np.clip(np.round(rows(rng, pos + n, hkv, hd) * 64), -4096, 4096) / 64 * 2.0 ** power
    q = np.clip(np.round(rng.standard_normal((n, h, hd)) * 64), -256, 256) / 64 * 2.0 ** -power
    k, q = k.astype(np.float32), q.astype(np.float32)
    assert np.isfinite(k).all() and np.isfinite(q).all()
    c = Cache(dev, "f32", pos + n, hkv, hd, k, rows(rng, pos + n, hkv, hd))
    got = c.attend(dev, q, nodes, pos, 0.1)
    want, bound = attention(q, k, c.v, visible(nodes.seen, nodes.depth, pos, 0), 0.1)
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("size", [1e30, 1e35, 2e37])
@pytest.mark.parametrize("side", ["k", "q"])
def test_one_key_takes_all(dev, size, side):
    """K rows (or queries) near the end of f32's range against ordinary ones: scores that f32 holds, the
    largest of which takes a node's whole weight."""
    note(f"tree ranges, {side} of {size}")
    rng = np.random.default_rng(3)
    h, hkv, hd, n, pos = 8, 2, 64, 9, 300
    nodes = Nodes(dev, random_parents(n, rng))
    k, v = (np.clip(rng.standard_normal((pos + n, hkv, hd)), -3, 3).astype(np.float32) for _ in range(2))
    q = np.clip(rng.standard_normal((n, h, hd)), -3, 3).astype(np.float32)
    if side == "k":
        k = (k * np.float32(size)).astype(np.float32)
    else:
        q = (q * np.float32(size)).astype(np.float32)
    c = Cache(dev, "f32", pos + n, hkv, hd, k, v)
    got = c.attend(dev, q, nodes, pos, 0.1)
    vis = visible(nodes.seen, nodes.depth, pos, 0)
    for a in range(h):
        x = np.where(vis, q[:, a].astype(np.float64) @ k[:, a // 4].astype(np.float64).T * 0.1, -np.inf)
        order = np.sort(x, 1)
        clear = order[:, -1] - order[:, -2] > 1e-4 * np.abs(x[np.isfinite(x)]).max()  # (beyond the scores' error)
        assert clear.sum() > n // 2
        want = v[x.argmax(1), a // 4]
        assert np.isfinite(got[:, a]).all()
        assert (np.abs(got[clear, a] - want[clear]) <= 2.0 ** -21 * np.abs(want[clear]) + 2.0 ** -38).all()


def test_zero_rows_beside_large_ones_i8(dev):
    """A row of zeros in a block of large K rows against large queries: its score is zero. The large rows are
    drafted ones that the nodes here do not see."""
    note("tree ranges, zero rows i8")
    rng = np.random.default_rng(6)
    h, hkv, hd, n, pos = 4, 2, 64, 12, 40
    nodes = Nodes(dev, [-1] + [0] * (n - 1))
    k, v = np.zeros((pos + n, hkv, hd), np.float32), rows(rng, pos + n, hkv, hd)
    k[pos + 1] = 1e30 * rng.uniform(0.5, 1, (hkv, hd))
    q = (rng.standard_normal((n, h, hd)) * 1e20).astype(np.float32)
    c = Cache(dev, "i8", pos + n, hkv, hd, k, v, 16)
    got = c.attend(dev, q, nodes, pos, 1.0)
    free = ~nodes.seen[:, 1]
    want, bound = attention(np.zeros_like(q), c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), 1.0)
    assert free.sum() == n - 1 and np.isfinite(got[free]).all()
    assert (np.abs(got - want) <= bound)[free].all()


@pytest.mark.parametrize("elem,what", [("f16", np.nan), ("f16", np.inf), ("f16", -np.inf), ("e4m3", np.nan),
                                       ("f32", np.inf)])
@pytest.mark.parametrize("hd,hkv,h,n", [(64, 2, 2, 9), (64, 2, 8, 12), (128, 2, 8, 40), (128, 1, 1, 5), (256, 2, 4, 30),
                                        (256, 1, 2, 3), (24, 2, 4, 21), (120, 2, 6, 50)])
@pytest.mark.parametrize("side", ["k", "v"])
def test_bad_cached_row_that_all_see(dev, elem, what, hd, hkv, h, n, side):
    """One value that is not finite, in a tile without masked keys, in the last one behind the drafted rows'
    or in the first: every node's heads over its KV head are NaN, the other KV head's are untouched; one split and many."""
    note(f"tree ranges, bad row {elem} {what} {side} {h}/{hkv}x{hd} n {n}")
    rng = np.random.default_rng(5)
    pos = 900
    nodes = Nodes(dev, random_parents(n, rng))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    k, v = rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd)
    clean = {cus: launch(dev, Cache(dev, elem, pos + n, hkv, hd, k, v), elem, q, nodes, pos, 0.1, 0, cus)[0]
             for cus in (1, 256)}
    for at, dim in ((0, hd - 1), (413, 5), (pos - 1, 0)):
        x = (k if side == "k" else v).copy()
        x[at, 0, dim] = what
        c = Cache(dev, elem, pos + n, hkv, hd, x if side == "k" else k, x if side == "v" else v)
        for cus in (1, 256):
            got = launch(dev, c, elem, q, nodes, pos, 0.1, 0, cus)[0]
            assert np.isnan(got[:, :h // hkv]).all(), (at, cus, np.isnan(got[:, :h // hkv]).mean())
            assert got[:, h // hkv:].tobytes() == clean[cus][:, h // hkv:].tobytes()


@pytest.mark.parametrize("elem", ["f32", "f16"])
@pytest.mark.parametrize("size", [-2.2e38, 2.2e38, -2.3e38])
def test_scores_at_the_ends(dev, elem, size):
    """All keys alike, their scores' log2 units just inside f32's range: V's average."""
    note(f"tree ranges, scores of {size} {elem}")
    rng = np.random.default_rng(4)
    h, hkv, hd, n, pos = 4, 2, 64, 5, 700
    nodes = Nodes(dev, random_parents(n, rng))
    k = np.broadcast_to(np.sign(rng.standard_normal((1, hkv, hd))), (pos + n, hkv, hd)).astype(np.float32) * np.float32(64)
    v = rng.standard_normal((pos + n, hkv, hd)).astype(np.float32)
    c = Cache(dev, elem, pos + n, hkv, hd, k, v)
    q = np.repeat(k[:n], h // hkv, 1) * np.float32(size / 64 ** 3)
    got = c.attend(dev, q, nodes, pos, 1.0)
    want, bound = attention(np.zeros_like(q), c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), 1.0)
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("elem,k_power,q_power,scale_power", [
    ("f32", -130, 120, 10), ("f32", -120, 100, 20), ("f32", 120, -130, 10), ("f32", 0, -100, 100), ("f32", 0, 100, -100),
    ("f32", 100, 15, -115), ("f16", 0, 100, -100), ("f16", -10, -100, 110), ("f16", 0, -126, 126), ("f16", -10, 120, -110)])
@pytest.mark.parametrize("n", [3, 40])
def test_scales_of_any_size(dev, elem, k_power, q_power, scale_power, n):
    """Ordinary scores of queries whose product with the scale f32 does not hold, or only in part."""
    note(f"tree ranges, {elem} K 2^{k_power} q 2^{q_power} scale 2^{scale_power} n {n}")
    rng = np.random.default_rng(7)
    h, hkv, hd, pos = 8, 2, 64, 400
    nodes = Nodes(dev, random_parents(n, rng))
    # Multiples of 2^-4 and 2^-6 below 2^6 and 2^2: exact at either end, down to 2^-149 (half: 2^-24).
    k = np.clip(np.round(rows(rng, pos + n, hkv, hd) * 16), -1024, 1024) / 16 * 2.0 ** k_power
    q = np.clip(np.round(rng.standard_normal((n, h, hd)) * 64), -256, 256) / 64 * 2.0 ** q_power
    k, q, scale = k.astype(np.float32), q.astype(np.float32), np.float32(0.1 * 2.0 ** scale_power)
    c = Cache(dev, elem, pos + n, hkv, hd, k, rows(rng, pos + n, hkv, hd))
    assert np.array_equal(c.k, k)
    got = c.attend(dev, q, nodes, pos, float(scale))
    want, bound = attention(q, c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), np.float64(scale))
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()
