"""A drafted tree's plan, rows, walk and moved cache rows against their definitions."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import CacheModel
from tests._textbook import rmsnorm_f64
from tests._tree import NOBODY, Nodes, accept, e4m3_values, plan, random_parents, rows, u32, words

pytestmark = pytest.mark.gpu


def device_plan(dev, parents):
    n = len(parents)
    pt = eb.Tensor.from_array(dev, np.asarray(parents, np.int32))
    masks = eb.Tensor.from_u32(dev, (n, -(-n // 32)), np.full(n * -(-n // 32), 5, np.uint32))
    depths = eb.Tensor.from_u32(dev, (n,), np.full(n, 5, np.uint32))
    rec = eb.Recorder(dev)
    eb.tree_plan(rec, pt, masks, depths, n)
    rec.submit()
    return u32(masks), u32(depths)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 100, 255, 256])
def test_plan(dev, n):
    rng = np.random.default_rng(n)
    trees = [random_parents(n, rng), random_parents(n, rng, width=200), list(range(-1, n - 1)), [-1] + [0] * (n - 1),
             [-1] * n, random_parents(n, rng, roots=3)]
    odd = random_parents(n, rng)  # entries that are no earlier node count as none
    for i, p in ((0, 0), (n - 1, n - 1), (n // 2, n), (n // 3, -77), (n // 4, 2 ** 31 - 1)):
        odd[i] = p
    for parents in trees + [odd]:
        masks, depths = device_plan(dev, parents)
        seen, depth = plan(parents)
        assert np.array_equal(masks, words(seen)) and np.array_equal(depths, depth)


def device_accept(dev, tokens, parents, sampled):
    n = len(tokens)
    t, s = (eb.Tensor.from_u32(dev, (n,), x) for x in (tokens, sampled))
    p = eb.Tensor.from_array(dev, np.asarray(parents, np.int32))
    path, emitted = (eb.Tensor.from_u32(dev, (n,), np.full(n, 3, np.uint32)) for _ in range(2))
    count = eb.Tensor.from_u32(dev, (1,), [99])
    rec = eb.Recorder(dev)
    eb.tree_accept(rec, t, p, s, path, emitted, count, n)
    rec.submit()
    return u32(path), u32(emitted), int(u32(count)[0])


@pytest.mark.parametrize("n", [1, 2, 5, 32, 63, 64, 65, 200, 256])
def test_accept(dev, n):
    rng = np.random.default_rng(n)
    for kind in range(6):
        vocab = (3, 3, 2, 1, 1, 2 ** 32)[kind]  # (few tokens: siblings alike, long paths)
        parents = random_parents(n, rng, width=(2, 8, 3, 4, 1, 5)[kind], roots=(1, 1, 2, 1, 1, 1)[kind])
        if kind == 3 and n > 4:
            parents[2], parents[4] = 2, -9
        tokens = rng.integers(0, vocab, n).astype(np.uint32)
        sampled = rng.integers(0, vocab, n).astype(np.uint32)
        path, emitted, count = device_accept(dev, tokens, parents, sampled)
        want = accept(tokens, parents, sampled)
        assert count == len(want) and path[:count].tolist() == want
        assert emitted[:count].tolist() == sampled[want].tolist()
        assert (path[count:] == NOBODY).all() and (emitted[count:] == NOBODY).all()
    if n > 1:  # a whole chain
        tokens = rng.integers(0, 9, n).astype(np.uint32)
        sampled = np.append(tokens[1:], 4).astype(np.uint32)
        path, emitted, count = device_accept(dev, tokens, list(range(-1, n - 1)), sampled)
        assert count == n and path.tolist() == list(range(n)) and np.array_equal(emitted, sampled)


# ---- rows at their positions ---------------------------------------------------------------

def cache_values(t, elem, shape):
    raw = t.read_bytes()
    if elem == eb.DType.F32:
        return np.frombuffer(raw, np.float32).reshape(shape).astype(np.float64)
    if elem == eb.DType.F16:
        return np.frombuffer(raw, np.float16).reshape(shape).astype(np.float64)
    return e4m3_values(np.frombuffer(raw, np.uint8)).reshape(shape)


@pytest.mark.parametrize("elem", [eb.DType.F32, eb.DType.F16, eb.DType.F8E4M3])
@pytest.mark.parametrize("h,hkv,hd,n,pos,norms", [
    (4, 2, 8, 1, 0, True), (16, 8, 128, 17, 30, True), (6, 2, 96, 33, 5, False), (3, 3, 256, 70, 1000, True),
    (5, 5, 10, 6, 9, True), (2, 1, 4, 256, 3, False),
])
def test_prologue_tree(dev, elem, h, hkv, hd, n, pos, norms):
    note(f"prologue {elem.name} {h}/{hkv}x{hd} n {n} pos {pos}")
    rng = np.random.default_rng(n)
    max_seq = pos + n + 2
    nodes = Nodes(dev, random_parents(n, rng))
    q, k, v = (rng.standard_normal((n, a, hd)).astype(np.float32) for a in (h, hkv, hkv))
    gains = [rng.uniform(0.5, 1.5, hd).astype(np.float32) if norms else None for _ in range(3)]
    up = lambda x: None if x is None else eb.Tensor.from_f32(dev, x.shape, x)  # noqa: E731
    rope = eb.Rope.build(dev, max_seq, hd, 1e4)
    kv = eb.KvCache.new(dev, 1, max_seq, hkv, hd, elem)
    for t in (kv.k[0], kv.v[0]):
        t.write(b"\x11" * t.byte_len())
    before = cache_values(kv.k[0], elem, (max_seq, hkv, hd))
    qo = eb.Tensor.empty(dev, q.shape)
    rec = eb.Recorder(dev)
    eb.attn_prologue_tree(rec, up(q), up(k), up(v), nodes.depths, qo, kv.k[0], kv.v[0], n, h, hkv, hd, pos, max_seq,
                          up(gains[0]), up(gains[1]), up(gains[2]), 1e-6, rope.cos, rope.sin)
    rec.submit()
    c, s = (t.to_f32().reshape(max_seq, 1, hd // 2).astype(np.float64)[pos + nodes.depth] for t in (rope.cos, rope.sin))

    def expect(x, gain, turn):
        x = x.astype(np.float64)
        if gain is not None:
            x = rmsnorm_f64(x, gain, hd, 1e-6).reshape(x.shape)
        if not turn:
            return x
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return np.concatenate((a * c - b * s, b * c + a * s), -1)

    # f32: the norm's sum (hd / 8 terms per lane and few steps), root, quotient and two products, two
    # products and a sum of the rotation: 2^-24 each, of a pair's length; then the store's half step.
    step = {eb.DType.F32: 0.0, eb.DType.F16: 2.0 ** -11, eb.DType.F8E4M3: 2.0 ** -4}[elem]
    least = {eb.DType.F32: 0.0, eb.DType.F16: 2.0 ** -25, eb.DType.F8E4M3: 2.0 ** -10}[elem]

    def close(got, want, extra, floor):
        size = np.hypot(want[..., :hd // 2], want[..., hd // 2:])
        size = np.concatenate((size, size), -1)
        err = (hd + 12) * 2.0 ** -24 * size
        assert (np.abs(got - want) <= err + extra * (np.abs(want) + err) + floor + 1e-37).all()

    close(qo.to_f32().reshape(q.shape), expect(q, gains[0], True), 0.0, 0.0)
    kc, vc = (cache_values(t, elem, (max_seq, hkv, hd)) for t in (kv.k[0], kv.v[0]))
    close(kc[pos:pos + n], expect(k, gains[1], True), step, least)
    close(vc[pos:pos + n], expect(v, gains[2], False), step, least)
    for x in (kc, vc):  # the other rows
        assert np.array_equal(x[:pos], before[:pos]) and np.array_equal(x[pos + n:], before[pos + n:])


def test_chain_rows_are_the_prologues(dev):
    """Without branches the positions are the rows': bit for bit what a prompt's rows get; a depth no
    tree has makes its node's q and K NaN, and nothing else."""
    rng = np.random.default_rng(1)
    h, hkv, hd, n, pos, seq = 8, 4, 64, 19, 40, 64
    q, k, v = (rng.standard_normal((n, a, hd)).astype(np.float32) for a in (h, hkv, hkv))
    gain = eb.Tensor.from_f32(dev, (hd,), rng.uniform(0.5, 1.5, hd))
    rope = eb.Rope.build(dev, seq, hd, 1e4)
    qt, kt, vt = (eb.Tensor.from_f32(dev, x.shape, x) for x in (q, k, v))
    depth = np.arange(n)
    got = []
    for how in range(3):
        kv = eb.KvCache.new(dev, 1, seq, hkv, hd)
        qo = eb.Tensor.empty(dev, q.shape)
        if how == 2:
            depth = depth.copy()
            depth[7], depth[11] = n, 2 ** 32 - 1
        depths = eb.Tensor.from_array(dev, depth.astype(np.uint32))
        head = (dev.stream, qt.data_ptr, q.size, kt.data_ptr, k.size, vt.data_ptr, v.size, n, h, hkv, hd, gain.data_ptr,
                gain.data_ptr, 0, 1e-6, rope.cos.data_ptr, rope.sin.data_ptr, rope.cos.numel(), pos)
        tail = (qo.data_ptr, q.size, kv.k[0].data_ptr, kv.k[0].numel(), kv.v[0].data_ptr, kv.v[0].numel(), seq,
                eb.DType.F32)
        if how == 0:
            eb.launch_attn_prologue(*head, *tail)
        else:
            eb.launch_attn_prologue_tree(*head, depths.data_ptr, n, *tail)
        k_rows, v_rows = (t.to_f32().reshape(seq, hkv, hd)[pos:pos + n] for t in (kv.k[0], kv.v[0]))
        got.append((qo.to_f32().reshape(q.shape), k_rows, v_rows))
    for a, b, c in zip(*got):
        assert a.tobytes() == b.tobytes()
    keep = np.delete(np.arange(n), [7, 11])
    for i in range(2):
        assert np.isnan(got[2][i][[7, 11]]).all()
        assert got[2][i][keep].tobytes() == got[0][i][keep].tobytes()
    assert got[2][2].tobytes() == got[0][2].tobytes()


# ---- moved rows ------------------------------------------------------------------------------

SIZES = {eb.DType.F32: 4, eb.DType.F16: 2, eb.DType.F8E4M3: 1}


def compact(dev, kv, path, count, n, pos):
    padded = np.full(n, 0xDEADBEEF, np.uint32)
    padded[:len(path)] = path
    pt, ct = eb.Tensor.from_u32(dev, (n,), padded), eb.Tensor.from_u32(dev, (1,), [count])
    rec = eb.Recorder(dev)
    eb.kv_compact(rec, kv, pt, ct, n, pos)
    rec.submit()


PATHS = [  # (path, count, how many rows count)
    ([0], 1, 1), ([0, 1, 2], 3, 3), ([0, 3, 4, 9], 4, 4), ([2, 3, 5], 3, 3), ([0, 1, 4, 5, 6, 11, 17], 7, 7),
    ([0, 3, 9], 2, 2), ([0, 3, 9], 0, 0), ([0, 3, 3, 5], 4, 2), ([0, 7, 4, 8], 4, 2), ([0, 2, 30, 31], 4, 2),
    (list(range(0, 20, 1)), 500, 20), (list(range(2, 20)), 18, 18),
]


@pytest.mark.parametrize("elem", list(SIZES))
@pytest.mark.parametrize("dims,hkv", [((64, 64), 2), ((8, 24, 8), 3), ((256,), 8)])
def test_compact(dev, elem, dims, hkv):
    note(f"compact {elem.name} {dims} {hkv}")
    rng = np.random.default_rng(2)
    n, pos, seq = 20, 13, 40
    for path, count, kept in PATHS:
        kv = eb.KvCache.new_per_layer(dev, list(dims), seq, hkv, elem)
        want = []
        for hd, k, v in zip(dims, kv.k, kv.v):
            for t in (k, v):
                x = rng.integers(0, 256, (seq, hkv * hd * SIZES[elem])).astype(np.uint8)
                t.write(x)
                y = x.copy()
                y[pos:pos + kept] = x[[pos + p for p in path[:kept]]]
                want.append(y)
        compact(dev, kv, path, count, n, pos)
        got = [t.read_bytes() for k, v in zip(kv.k, kv.v) for t in (k, v)]
        assert [y.tobytes() for y in want] == got, (path, count)


def test_compact_wide_path(dev):
    """The widest tree, with the deepest path, over more layers than a launch takes."""
    rng = np.random.default_rng(3)
    n, hkv, hd, seq, layers = 256, 1, 32, 300, 70
    path = np.sort(rng.choice(n, 200, replace=False))
    kv = eb.KvCache.new(dev, layers, seq, hkv, hd)
    x = rng.standard_normal((2 * layers, seq, hkv, hd)).astype(np.float32)
    for l in range(layers):
        kv.k[l].write(x[2 * l])
        kv.v[l].write(x[2 * l + 1])
    compact(dev, kv, path, 200, n, 44)
    want = x.copy()
    want[:, 44:244] = x[:, 44 + path]
    for l in range(layers):
        assert kv.k[l].read_bytes() == want[2 * l].tobytes() and kv.v[l].read_bytes() == want[2 * l + 1].tobytes()


@pytest.mark.parametrize("block,hd,pos", [(16, 32, 13), (16, 64, 16), (64, 128, 100), (32, 256, 37), (256, 48, 20)])
def test_compact_i8(dev, block, hd, pos):
    """As the branch's rows read as values and written at pos."""
    note(f"compact i8 {block} {hd} {pos}")
    rng = np.random.default_rng(block)
    n, hkv, layers = 50, 3, 2
    seq = pos + n + 5
    for path in ([0], [0, 1, 2], [0, 4, 5, 20, 33], sorted(rng.choice(n, 30, replace=False)), list(range(n))):
        kv = eb.KvCache.new_i8(dev, layers, seq, hkv, hd, block)
        models = []
        for l in range(layers):
            for codes, exps in ((kv.k[l], kv.k_scale[l]), (kv.v[l], kv.v_scale[l])):
                m = CacheModel(seq, hkv, hd, block, rng)
                x = rows(rng, pos + n, hkv, hd) * 2.0 ** rng.integers(-20, 20, (pos + n, 1, 1))
                if l == 1:
                    x[pos + 9, 0, 1] = np.nan
                m.write(x.astype(np.float32), 0)
                codes.write(m.codes)
                exps.write(m.exps)
                models.append(m)
        compact(dev, kv, path, len(path), n, pos)
        for i, m in enumerate(models):
            m.write(m.values(pos, pos + n)[path].astype(np.float32), pos)
            codes, exps = ((kv.k, kv.k_scale), (kv.v, kv.v_scale))[i % 2]
            assert codes[i // 2].read_bytes() == m.codes.tobytes(), (path, i)
            assert exps[i // 2].read_bytes() == m.exps.tobytes(), (path, i)


def test_compact_i8_widest(dev):
    rng = np.random.default_rng(7)
    n, pos, hkv, hd, block = 256, 70, 2, 256, 64
    seq = pos + n
    kv = eb.KvCache.new_i8(dev, 1, seq, hkv, hd, block)
    path = np.sort(rng.choice(n, 180, replace=False))
    models = []
    for codes, exps in ((kv.k[0], kv.k_scale[0]), (kv.v[0], kv.v_scale[0])):
        m = CacheModel(seq, hkv, hd, block)
        m.write(rows(rng, seq, hkv, hd), 0)
        codes.write(m.codes)
        exps.write(m.exps)
        models.append(m)
    compact(dev, kv, path, 180, n, pos)
    for m, codes, exps in zip(models, (kv.k[0], kv.v[0]), (kv.k_scale[0], kv.v_scale[0])):
        m.write(m.values(pos, pos + n)[path].astype(np.float32), pos)
        assert codes.read_bytes() == m.codes.tobytes() and exps.read_bytes() == m.exps.tobytes()


@pytest.mark.parametrize("elem", list(SIZES) + [eb.DType.I8])
@pytest.mark.parametrize("count", [0, 1, 17, 64, 333])
def test_fork(dev, elem, count):
    note(f"fork {elem.name} {count}")
    rng = np.random.default_rng(count)
    dims, hkv = [32, 48, 96], 3
    if elem == eb.DType.I8:
        src = eb.KvCache.new_i8_per_layer(dev, dims, 333, hkv, 32)
        dst = eb.KvCache.new_i8_per_layer(dev, dims, 400, hkv, 32)
        pairs = [(a, b, hkv * d, 1) for s, t in ((src.k, dst.k), (src.v, dst.v)) for a, b, d in zip(s, t, dims)]
        pairs += [(a, b, hkv, 32) for s, t in ((src.k_scale, dst.k_scale), (src.v_scale, dst.v_scale))
                  for a, b in zip(s, t)]
    else:
        src = eb.KvCache.new_per_layer(dev, dims, 333, hkv, elem)
        dst = eb.KvCache.new_per_layer(dev, dims, 400, hkv, elem)
        pairs = [(a, b, hkv * d * SIZES[elem], 1) for s, t in ((src.k, dst.k), (src.v, dst.v))
                 for a, b, d in zip(s, t, dims)]
    want = []
    for a, b, width, per in pairs:
        x, y = (rng.integers(0, 256, t.byte_len()).astype(np.uint8) for t in (a, b))
        a.write(x)
        b.write(y)
        y[:-(-count // per) * width] = x[:-(-count // per) * width]
        want.append((x.tobytes(), y.tobytes()))
    rec = eb.Recorder(dev)
    eb.kv_fork(rec, dst, src, count)
    rec.submit()
    assert [(a.read_bytes(), b.read_bytes()) for a, b, _, _ in pairs] == want


def test_fork_many_layers(dev):
    rng = np.random.default_rng(1)
    src, dst = (eb.KvCache.new(dev, 67, 700, 2, 64, eb.DType.F16) for _ in range(2))
    data = rng.integers(0, 256, (134, 700 * 256)).astype(np.uint8)
    for l in range(67):
        src.k[l].write(data[2 * l])
        src.v[l].write(data[2 * l + 1])
    rec = eb.Recorder(dev)
    eb.kv_fork(rec, dst, src, 700)
    rec.submit()
    for l in range(67):
        assert dst.k[l].read_bytes() == data[2 * l].tobytes() and dst.v[l].read_bytes() == data[2 * l + 1].tobytes()
