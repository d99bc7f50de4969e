"""Attention of a drafted tree against its definition in 64 bits."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._tree import Cache, Nodes, attention, check, random_parents, rows, u32, visible

pytestmark = pytest.mark.gpu


def run(dev, elem, h, hkv, hd, n, pos, window=0, seed=0, scale=None, spare=0, nodes=None, block=64):
    rng = np.random.default_rng(seed + 7 * n + pos)
    nodes = nodes or Nodes(dev, random_parents(n, rng))
    scale = hd ** -0.5 if scale is None else scale
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    c = Cache(dev, elem, pos + n + spare, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd), block)
    got = c.attend(dev, q, nodes, pos, scale, window)
    want, bound = attention(q, c.k, c.v, visible(nodes.seen, nodes.depth, pos, window), scale)
    check(got, want, bound, f"{elem} {h}/{hkv}x{hd} n {n} pos {pos} window {window}")


# Column counts on both sides of 16, 64 and 128 per KV head, head dims of every padded width, tiles
# that end inside the cached and the drafted keys, one split and many.
SHAPES = [
    (4, 2, 8, 1, 0, 0), (4, 2, 8, 1, 1, 0), (4, 4, 24, 5, 31, 0), (2, 1, 64, 16, 32, 0), (6, 2, 96, 7, 33, 0),
    (16, 8, 128, 8, 100, 0), (16, 8, 128, 9, 700, 0), (14, 2, 64, 10, 1000, 0), (32, 8, 128, 17, 515, 0),
    (32, 8, 128, 33, 1500, 0), (8, 1, 128, 16, 257, 0), (16, 8, 256, 8, 300, 0), (16, 8, 256, 40, 999, 0),
    (3, 3, 144, 65, 64, 0), (8, 8, 32, 200, 90, 0), (2, 2, 128, 256, 40, 0), (64, 1, 64, 3, 400, 0),
    (16, 8, 128, 12, 640, 1), (16, 8, 128, 12, 640, 3), (32, 8, 128, 30, 2000, 100), (4, 2, 64, 64, 50, 20),
    (16, 8, 256, 25, 3000, 700), (12, 4, 80, 21, 128, 129), (16, 8, 128, 20, 4096, 5000),
]


@pytest.mark.parametrize("elem", ["f32", "f16", "e4m3", "i8"])
@pytest.mark.parametrize("h,hkv,hd,n,pos,window", SHAPES)
def test_attn_tree(dev, elem, h, hkv, hd, n, pos, window):
    if elem == "i8" and (hd % 16 or hd < 32):
        hd = 32
    note(f"attn_tree {elem} {h}/{hkv}x{hd} n {n} pos {pos} window {window}")
    run(dev, elem, h, hkv, hd, n, pos, window, spare=5)


def test_head_dim_4(dev):
    run(dev, "f32", 4, 2, 4, 9, 77)


@pytest.mark.parametrize("block", [16, 256])
def test_blocks(dev, block):
    run(dev, "i8", 8, 4, 64, 11, 301, block=block)


def test_larger_scale(dev):
    """Scores of some hundred: one key takes nearly all of a node's weight."""
    run(dev, "f32", 16, 8, 128, 12, 500, scale=1.0)
    run(dev, "f16", 16, 8, 256, 12, 500, scale=1.0)


@pytest.mark.parametrize("elem", ["f32", "f16", "e4m3", "i8"])
def test_long(dev, elem):
    note(f"attn_tree long {elem}")
    run(dev, elem, 8, 2, 128, 20, 30011)


@pytest.mark.parametrize("elem", ["f32", "f16", "e4m3", "i8"])
@pytest.mark.parametrize("pos", [0, 3, 200])
def test_any_masks(dev, elem, pos):
    """Masks that are no tree's: bits above the diagonal, rows without any, bits past n."""
    note(f"any masks {elem} {pos}")
    rng = np.random.default_rng(pos)
    n, h, hkv, hd = 37, 4, 2, 64
    seen = rng.random((n, n)) < 0.3
    seen[5] = seen[36] = False
    nodes = Nodes(dev, seen=seen, depths=rng.integers(0, 9, n))
    nodes.masks = eb.Tensor.from_array(dev, u32(nodes.masks) | np.array([0, 0xFFFFFFFF << 5 & 0xFFFFFFFF], np.uint32))
    for window in (0, 4):
        q = rng.standard_normal((n, h, hd)).astype(np.float32)
        c = Cache(dev, elem, pos + n, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
        got = c.attend(dev, q, nodes, pos, 0.125, window)
        vis = visible(seen, nodes.depth, pos, window)
        want, bound = attention(q, c.k, c.v, vis, 0.125)
        check(got, want, bound, f"any masks {elem} {pos} {window}")
        assert pos > 0 or not vis[5].any()
        assert (got[~vis.any(1)] == 0).all()


BAD = {"nan": np.nan, "inf": np.inf, "-inf": -np.inf, "huge": 1e30, "lowest": -3.4028235e38}


@pytest.mark.parametrize("elem", ["f32", "f16", "e4m3"])
@pytest.mark.parametrize("what", sorted(BAD))
@pytest.mark.parametrize("side", ["k", "v"])
def test_unseen_rows_do_not_count(dev, elem, what, side):
    """A drafted row, and rows behind the window and behind the tree, whose values are not finite or
    very large: the nodes that do not see them answer as without them; those that do, with NaN (huge
    finite values apart)."""
    note(f"unseen {elem} {what} {side}")
    if elem != "f32" and what in ("huge", "lowest"):
        what = "inf"  # (what those values are stored as)
    rng = np.random.default_rng(3)
    n, pos, h, hkv, hd, window = 21, 150, 8, 4, 64, 60
    nodes = Nodes(dev, random_parents(n, rng))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    k, v = rows(rng, pos + n + 3, hkv, hd), rows(rng, pos + n + 3, hkv, hd)
    bad = 2
    clean_k, clean_v = k.copy(), v.copy()
    x = k if side == "k" else v
    x[pos + bad, :, 17] = BAD[what]
    x[20, :, 3] = BAD[what]  # behind every window
    x[pos + n:, :, 0] = BAD[what]  # behind the tree
    c = Cache(dev, elem, pos + n + 3, hkv, hd, k, v)
    clean = Cache(dev, elem, pos + n + 3, hkv, hd, clean_k, clean_v)
    got = c.attend(dev, q, nodes, pos, 0.125, window)
    vis = visible(nodes.seen, nodes.depth, pos, window)
    free = ~vis[:, pos + bad]
    assert free.sum() > 3 and (~free).sum() > 1
    want, bound = attention(q, clean.k[:pos + n], clean.v[:pos + n], vis, 0.125)
    check(got[free], want[free], bound[free], f"unseen {elem} {what} {side}")
    if what in ("nan", "inf", "-inf"):
        assert np.isnan(got[~free]).all()
    elif side == "v" and what == "huge":
        want, bound = attention(q, k[:pos + n], v[:pos + n], vis, 0.125)
        check(got[~free], want[~free], bound[~free], "huge value seen")


def test_unseen_rows_i8(dev):
    """A NaN block reaches the nodes that see one of its keys."""
    rng = np.random.default_rng(4)
    n, pos, h, hkv, hd, window = 21, 160, 4, 2, 64, 24
    nodes = Nodes(dev, random_parents(n, rng, width=3))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    for side in range(2):
        kv = [rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd)]
        clean = Cache(dev, "i8", pos + n, hkv, hd, kv[0], kv[1], 16)
        kv[side][pos - 20, 1, 5] = np.nan  # keys pos - 32 .. pos - 17, KV head 1
        c = Cache(dev, "i8", pos + n, hkv, hd, kv[0], kv[1], 16)
        got = c.attend(dev, q, nodes, pos, 0.125, window)
        vis = visible(nodes.seen, nodes.depth, pos, window)
        hit = vis[:, pos - 32:pos - 16].any(1)
        assert hit.any() and not hit.all()
        want, bound = attention(q, clean.k, clean.v, vis, 0.125)
        check(got[:, :2], want[:, :2], bound[:, :2], "the other KV head")
        check(got[~hit], want[~hit], bound[~hit], "nodes past the block")
        assert np.isnan(got[hit][:, 2:]).all()


def test_rows_of_unlike_size(dev):
    """f32 rows from 1e-30 to 1e30 beside ordinary ones: values whose weight is large keep theirs."""
    rng = np.random.default_rng(5)
    n, pos, h, hkv, hd = 9, 300, 4, 2, 128
    nodes = Nodes(dev, random_parents(n, rng))
    for lo, hi in ((-30, 0), (0, 30), (-18, -12)):
        q = rng.standard_normal((n, h, hd)).astype(np.float32)
        k = rows(rng, pos + n, hkv, hd)
        v = (rows(rng, pos + n, hkv, hd) * 10.0 ** rng.uniform(lo, hi, (pos + n, hkv, 1))).astype(np.float32)
        c = Cache(dev, "f32", pos + n, hkv, hd, k, v)
        got = c.attend(dev, q, nodes, pos, 0.2)
        want, bound = attention(q, k, v, visible(nodes.seen, nodes.depth, pos, 0), 0.2)
        check(got, want, bound, f"rows of 1e{lo} to 1e{hi}")


@pytest.mark.parametrize("elem,rows_", [("f32", 600000), ("f16", 1200000), ("i8", 2200000)])
def test_offsets_past_32_bits(dev, elem, rows_):
    """The last rows of a cache of more than 2^31 bytes, through a window."""
    note(f"long offsets {elem}")
    rng = np.random.default_rng(6)
    n, h, hkv, hd, window = 10, 16, 8, 128, 90
    pos = rows_ - n
    nodes = Nodes(dev, random_parents(n, rng))
    new = window + n
    k, v = rows(rng, new, hkv, hd), rows(rng, new, hkv, hd)
    if elem == "f16":  # (values the cache holds exactly)
        k, v = (x.astype(np.float16).astype(np.float32) for x in (k, v))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    qt, kt, vt = (eb.Tensor.from_f32(dev, x.shape, x) for x in (q, k, v))
    ot = eb.Tensor.empty(dev, q.shape)
    rec = eb.Recorder(dev)
    if elem == "i8":
        kv = eb.KvCache.new_i8(dev, 1, rows_, hkv, hd, 64)
        eb.kv_write_i8(rec, kv, 0, kt, vt, new, rows_ - new)
        eb.attn_tree_i8(rec, qt, kv, 0, nodes.masks, nodes.depths, ot, h, pos, n, 0.1, window)
        eb.kv_read_i8(rec, kv, 0, kt, vt, new, rows_ - new)
    else:
        kv = eb.KvCache.new(dev, 1, rows_, hkv, hd, eb.DType.F32 if elem == "f32" else eb.DType.F16)
        for x, to in ((kt, kv.k[0]), (vt, kv.v[0])):
            eb.kv_write(rec, to, x, hkv, new, hd, rows_, rows_ - new)
        eb.attn_tree(rec, qt, kv.k[0], kv.v[0], nodes.masks, nodes.depths, ot, h, hkv, pos, n, hd, rows_, 0.1, window)
    rec.submit()
    k, v = (t.to_f32().reshape(k.shape) for t in (kt, vt))
    want, bound = attention(q, k, v, visible(nodes.seen, nodes.depth, window, window), 0.1)
    check(ot.to_f32().reshape(q.shape), want, bound, f"long offsets {elem}")


def test_chain_is_a_chunk(dev):
    """A tree without branches is the next rows of a prompt, and one node is a decode step."""
    rng = np.random.default_rng(8)
    h, hkv, hd, pos, n = 16, 8, 128, 333, 24
    c = Cache(dev, "f32", pos + n, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    got = c.attend(dev, q, Nodes(dev, list(range(-1, n - 1))), pos, 0.1)
    qt, ot = eb.Tensor.from_f32(dev, q.shape, q), eb.Tensor.empty(dev, q.shape)
    rec = eb.Recorder(dev)
    eb.attn_prefill_chunk(rec, qt, c.kv.k[0], c.kv.v[0], ot, h, hkv, pos, n, hd, pos + n, 0.1)
    rec.submit()
    assert np.abs(got - ot.to_f32().reshape(q.shape)).max() < 1e-5


@pytest.mark.parametrize("elem", ["f32", "i8"])
def test_raw_launch_is_the_recorders(dev, elem):
    rng = np.random.default_rng(9)
    h, hkv, hd, pos, n, seq = 16, 8, 128, 3000, 20, 3050
    c = Cache(dev, elem, seq, hkv, hd, rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd))
    nodes = Nodes(dev, random_parents(n, rng))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    want = c.attend(dev, q, nodes, pos, 0.1, 2000)
    dt = eb.DType.F32 if elem == "f32" else eb.DType.I8
    need = eb.attn_tree_workspace_floats(h, hkv, pos, n, hd, dt, dev.cu_count)
    assert need > 0
    ws = eb.Tensor.from_f32(dev, (need,), np.full(need, np.nan, np.float32))
    qt, ot = eb.Tensor.from_f32(dev, q.shape, q), eb.Tensor.empty(dev, q.shape)
    tail = (nodes.masks.data_ptr, n, nodes.depths.data_ptr, n, ot.data_ptr, q.size)
    if elem == "f32":
        eb.launch_attn_tree(dev.stream, qt.data_ptr, q.size, c.kv.k[0].data_ptr, c.kv.k[0].numel(),
                            c.kv.v[0].data_ptr, c.kv.v[0].numel(), dt, *tail, h, hkv, pos, n, hd, seq, 0.1, 2000,
                            ws.data_ptr, need, dev.cu_count)
    else:
        k, v, ke, ve = c.kv.k[0], c.kv.v[0], c.kv.k_scale[0], c.kv.v_scale[0]
        cache = eb.CacheI8(k.data_ptr, ke.data_ptr, v.data_ptr, ve.data_ptr, k.numel(), ke.numel(), seq, hkv, hd, 64)
        eb.launch_attn_tree_i8(dev.stream, qt.data_ptr, q.size, cache, *tail, h, pos, n, 0.1, 2000, ws.data_ptr, need,
                               dev.cu_count)
    got = ot.to_f32().reshape(q.shape)
    assert got.tobytes() == want.tobytes()
