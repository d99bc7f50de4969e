"""Attention of a drafted tree however its columns and keys are dealt out: every width of a workgroup, one
split and many, for any number of compute units; and calls at the same time."""
import threading

import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._tree import Cache, Nodes, attention, check, random_parents, rows, visible

pytestmark = pytest.mark.gpu

DTYPES = {"f32": eb.DType.F32, "f16": eb.DType.F16, "e4m3": eb.DType.F8E4M3, "i8": eb.DType.I8}
GUARD = 64


def launch(dev, c, elem, q, nodes, pos, scale, window, cus):
    """The raw form in a workspace of just the floats it asks for, and none behind them written."""
    n, h, hd = q.shape
    need = eb.attn_tree_workspace_floats(h, c.hkv, pos, n, hd, DTYPES[elem], cus)
    ws = eb.Tensor.from_f32(dev, (need + GUARD,), np.full(need + GUARD, np.nan, np.float32))
    qt = eb.Tensor.from_f32(dev, q.shape, q)
    ot = eb.Tensor.from_f32(dev, q.shape, np.full(q.shape, 7.0, np.float32))
    tail = (nodes.masks.data_ptr, nodes.masks.numel(), nodes.depths.data_ptr, n, ot.data_ptr, q.size)
    k, v = c.kv.k[0], c.kv.v[0]
    if elem == "i8":
        ke, ve = c.kv.k_scale[0], c.kv.v_scale[0]
        cache = eb.CacheI8(k.data_ptr, ke.data_ptr, v.data_ptr, ve.data_ptr, k.numel(), ke.numel(), c.max_seq, c.hkv, hd,
                           64)
        eb.launch_attn_tree_i8(dev.stream, qt.data_ptr, q.size, cache, *tail, h, pos, n, scale, window, ws.data_ptr,
                               need, cus)
    else:
        eb.launch_attn_tree(dev.stream, qt.data_ptr, q.size, k.data_ptr, k.numel(), v.data_ptr, v.numel(), DTYPES[elem],
                            *tail, h, c.hkv, pos, n, hd, c.max_seq, scale, window, ws.data_ptr, need, cus)
    assert np.isnan(ws.to_f32()[need:]).all()
    return ot.to_f32().reshape(q.shape), need


# Up to 16, 64 and more columns per KV head, keys of a few tiles and of many, with and without a window.
@pytest.mark.parametrize("elem", ["f32", "f16", "e4m3", "i8"])
@pytest.mark.parametrize("h,hkv,hd,n,pos,window", [
    (4, 2, 128, 7, 1200, 0), (8, 2, 128, 15, 900, 0), (8, 2, 128, 33, 1100, 300), (6, 1, 64, 50, 700, 0),
    (2, 1, 256, 24, 800, 0), (4, 1, 256, 37, 500, 100), (2, 2, 32, 130, 3, 0),
])
def test_any_number_of_compute_units(dev, elem, h, hkv, hd, n, pos, window):
    rng = np.random.default_rng(17 * n + pos)
    nodes = Nodes(dev, random_parents(n, rng))
    c = Cache(dev, elem, pos + n + 3, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    want, bound = attention(q, c.k, c.v, visible(nodes.seen, nodes.depth, pos, window), hd ** -0.5)
    needs = []
    for cus in (1, 5, 24, 100, 256, 100000):
        note(f"tree plans {elem} {h}/{hkv}x{hd} n {n} pos {pos} window {window}, {cus} compute units")
        got, need = launch(dev, c, elem, q, nodes, pos, hd ** -0.5, window, cus)
        check(got, want, bound, f"{cus} compute units")
        needs.append(need)
    assert needs == sorted(needs)


def test_most_columns(dev):
    """256 heads on one KV head and 256 nodes: 65536 columns of 296 keys."""
    rng = np.random.default_rng(3)
    h, hkv, hd, n, pos = 256, 1, 32, 256, 40
    nodes = Nodes(dev, random_parents(n, rng))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    for elem in ("f32", "i8"):
        note(f"tree plans, most columns {elem}")
        c = Cache(dev, elem, pos + n, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
        got = c.attend(dev, q, nodes, pos, 0.2)
        want, bound = attention(q, c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), 0.2)
        check(got, want, bound, elem)


def test_threads_share_the_device(dev):
    """Two threads on one device: their splits' sums lie in the same workspace, one after the other."""
    rng = np.random.default_rng(4)
    jobs = []
    for elem, h, hkv, hd, n, pos in (("f16", 16, 8, 128, 20, 3000), ("f32", 8, 2, 64, 64, 2100)):
        c = Cache(dev, elem, pos + n, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
        nodes = Nodes(dev, random_parents(n, rng))
        q = rng.standard_normal((n, h, hd)).astype(np.float32)
        jobs.append((c, q, nodes, pos, c.attend(dev, q, nodes, pos, 0.1).tobytes()))
    wrong = []

    def work(c, q, nodes, pos, want):
        try:
            for _ in range(12):
                if c.attend(dev, q, nodes, pos, 0.1).tobytes() != want:
                    wrong.append(c.elem)
        except Exception as e:  # (a thread's failure is the test's)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_same_call_same_bits(dev):
    rng = np.random.default_rng(5)
    h, hkv, hd, n, pos = 32, 8, 128, 21, 5000
    for elem in DTYPES:
        c = Cache(dev, elem, pos + n, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
        nodes = Nodes(dev, random_parents(n, rng))
        q = rng.standard_normal((n, h, hd)).astype(np.float32)
        first = c.attend(dev, q, nodes, pos, 0.1).tobytes()
        for _ in range(3):
            assert c.attend(dev, q, nodes, pos, 0.1).tobytes() == first, elem


@pytest.mark.parametrize("elem", ["f32", "f16", "e4m3", "i8"])
@pytest.mark.parametrize("n,pos", [(9, 0), (9, 2500), (70, 300)])
def test_queries_that_are_not_finite(dev, elem, n, pos):
    """They make their own head of their node NaN, where it sees a key, and change no other bit."""
    note(f"tree plans, queries {elem} {n} {pos}")
    rng = np.random.default_rng(6)
    h, hkv, hd = 8, 2, 128
    seen = Nodes(dev, random_parents(n, rng)).seen
    seen[4] = False
    nodes = Nodes(dev, seen=seen, depths=seen.sum(1))
    c = Cache(dev, elem, pos + n, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    want = c.attend(dev, q, nodes, pos, 0.1)
    q[0, 1, 5], q[3, 7, 127], q[n - 1, 2, 0], q[4, 0, 3] = np.nan, np.inf, -np.inf, np.nan
    got = c.attend(dev, q, nodes, pos, 0.1)
    bad = np.zeros((n, h), bool)
    bad[0, 1] = bad[3, 7] = bad[n - 1, 2] = True
    bad[4, 0] = pos > 0  # (otherwise it sees nothing: zeros)
    assert np.isnan(got[bad]).all()
    assert got[~bad].tobytes() == want[~bad].tobytes()


@pytest.mark.parametrize("elem", ["f32", "f16", "e4m3", "i8"])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30, 30.0])
def test_scales(dev, elem, scale):
    """All keys alike, the least alike key first, all nearly alike, one key with all the weight; and a node of zeros."""
    note(f"tree plans, scale {elem} {scale}")
    rng = np.random.default_rng(7)
    h, hkv, hd, n, pos = 8, 2, 64, 11, 1300
    nodes = Nodes(dev, random_parents(n, rng))
    c = Cache(dev, elem, pos + n, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    q[2] = 0
    got = c.attend(dev, q, nodes, pos, scale)
    want, bound = attention(q, c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), np.float64(np.float32(scale)))
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("size", [1e-41, 1e-30, 1e30, 3e37])
def test_sizes_of_rows(dev, size):
    """f32 rows at the ends of their range, in K (against queries of the other end) and in V."""
    note(f"tree plans, rows of {size}")
    rng = np.random.default_rng(8)
    h, hkv, hd, n, pos = 4, 2, 64, 9, 500
    nodes = Nodes(dev, random_parents(n, rng))
    k = rows(rng, pos + n, hkv, hd)
    v = np.clip(rng.standard_normal((pos + n, hkv, hd)), -3, 3).astype(np.float32)
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    plain = Cache(dev, "f32", pos + n, hkv, hd, k, v)
    c = Cache(dev, "f32", pos + n, hkv, hd, k, (v.astype(np.float64) * size).astype(np.float32))
    got = c.attend(dev, q, nodes, pos, 0.1)
    want, bound = attention(q, c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), 0.1)
    # (a value or a result below 2^-126 may be taken for zero)
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound + 2 * 2.0 ** -126).all()
    if size > 1e-40:
        c = Cache(dev, "f32", pos + n, hkv, hd, (k * np.float32(2.0 ** np.round(np.log2(size) / 2))).astype(np.float32), v)
        small = (q * np.float32(2.0 ** -np.round(np.log2(size) / 2))).astype(np.float32)
        assert c.attend(dev, small, nodes, pos, 0.1).tobytes() == plain.attend(dev, q, nodes, pos, 0.1).tobytes()


@pytest.mark.parametrize("elem", ["f32", "f16"])
@pytest.mark.parametrize("size", [1e25, -1e25, -1e31, 1e31])
def test_large_scores(dev, elem, size):
    """All keys alike, with scores near the ends of f32's range: V's average."""
    note(f"tree plans, scores of {size} {elem}")
    rng = np.random.default_rng(9)
    h, hkv, hd, n, pos = 4, 2, 64, 5, 700
    nodes = Nodes(dev, random_parents(n, rng))
    k = np.broadcast_to(np.sign(rng.standard_normal((1, hkv, hd))), (pos + n, hkv, hd)).astype(np.float32) * np.float32(64)
    v = rng.standard_normal((pos + n, hkv, hd)).astype(np.float32)
    c = Cache(dev, elem, pos + n, hkv, hd, k, v)
    q = np.repeat(k[:n], h // hkv, 1) * np.float32(size / 64 ** 2)
    got = c.attend(dev, q, nodes, pos, 1.0)
    # (alike keys have the same score to the bit, so the weights are alike whatever the scores' error)
    want, bound = attention(np.zeros_like(q), c.k, c.v, visible(nodes.seen, nodes.depth, pos, 0), 1.0)
    check(got, want, bound, f"{elem} {size}")
