"""A drafted tree's operators as a model uses them: whole steps, captured steps, refusals of handles."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._tree import Nodes, accept, check, attention, random_parents, rows, u32, visible

pytestmark = pytest.mark.gpu

H, HKV, HD, HIDDEN, VOCAB, LAYERS, SEQ = 8, 2, 64, 128, 96, 3, 160


class Model:
    """Embedding, attention layers, head; the cache is its argument."""

    def __init__(self, dev, seed=0, window=0):
        rng = np.random.default_rng(seed)
        self.dev = dev

        def weight(out_f, in_f):
            w = (rng.standard_normal((out_f, in_f)) / np.sqrt(in_f)).astype(np.float32)
            return eb.Tensor.from_f16_packed(dev, (out_f, in_f), w)

        def gain():
            return eb.Tensor.from_f32(dev, (HD,), rng.uniform(0.7, 1.3, HD))

        self.emb = rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32)
        self.layers = [eb.Attention(H, HKV, HD, 0.4, gain(), gain(), None, 1e-6, window if l == 1 else 0,
                                    weight(H * HD, HIDDEN), weight(HKV * HD, HIDDEN), weight(HKV * HD, HIDDEN),
                                    weight(HIDDEN, H * HD), HIDDEN) for l in range(LAYERS)]
        self.head = eb.Linear(weight(VOCAB, HIDDEN), HIDDEN, VOCAB)
        self.rope = eb.Rope.build(dev, SEQ, HD, 1e4)

    def cache(self, elem):
        if elem == "i8":
            return eb.KvCache.new_i8(self.dev, LAYERS, SEQ, HKV, HD, 16)
        return eb.KvCache.new(self.dev, LAYERS, SEQ, HKV, HD, eb.DType[elem])

    def tokens(self, rec, logits, n):
        """The largest logit of each row."""
        u, cold = (eb.Tensor.from_f32(self.dev, (n,), np.zeros(n, np.float32)) for _ in range(2))
        out = eb.Tensor.empty(self.dev, (n,), eb.DType.U32)
        eb.sample(rec, logits, u, out, n, VOCAB, temperature=cold)
        return out

    def forward(self, kv, tokens, pos):
        n = len(tokens)
        rec = eb.Recorder(self.dev)
        x = eb.Tensor.from_f32(self.dev, (n, HIDDEN), self.emb[tokens])
        for l, a in enumerate(self.layers):
            x = a.forward(rec, x, self.rope, kv, l, n, pos)
        out = self.tokens(rec, self.head.forward(rec, x, n), n)
        rec.submit()
        return u32(out)

    def step(self, rec, kv, x, tokens, parents, n, pos):
        """Everything of one drafted step that runs on the device: (path, emitted, count)."""
        dev = self.dev
        masks, depths = (eb.Tensor.empty(dev, s, eb.DType.U32) for s in ((n, -(-n // 32)), (n,)))
        path, emitted = (eb.Tensor.empty(dev, (n,), eb.DType.U32) for _ in range(2))
        count = eb.Tensor.empty(dev, (1,), eb.DType.U32)
        u, cold = self.zeros(n)
        sampled = eb.Tensor.empty(dev, (n,), eb.DType.U32)
        eb.tree_plan(rec, parents, masks, depths, n)
        for l, a in enumerate(self.layers):
            x = a.forward_tree(rec, x, self.rope, kv, l, masks, depths, n, pos)
        eb.sample(rec, self.head.forward(rec, x, n), u, sampled, n, VOCAB, temperature=cold)
        eb.tree_accept(rec, tokens, parents, sampled, path, emitted, count, n)
        eb.kv_compact(rec, kv, path, count, n, pos)
        return path, emitted, count

    def zeros(self, n):
        if not hasattr(self, "_zeros"):
            self._zeros = {}
        if n not in self._zeros:
            self._zeros[n] = tuple(eb.Tensor.from_f32(self.dev, (n,), np.zeros(n, np.float32)) for _ in range(2))
        return self._zeros[n]


def draft(rng, n, root, right):
    """A tree that holds the coming tokens `right` on some branch, up to where it ends or guesses wrong."""
    parents = random_parents(n, rng, width=4)
    tokens = rng.integers(0, VOCAB, n).astype(np.uint32)
    tokens[0] = root
    line = [int(rng.integers(0, n))]
    while parents[line[-1]] >= 0:
        line.append(parents[line[-1]])
    for node, t in zip(reversed(line[:-1]), right):
        tokens[node] = t
    return parents, tokens


@pytest.mark.parametrize("elem,window", [("F32", 0), ("F32", 9), ("F16", 0), ("F8E4M3", 9)])
def test_drafted_answer_is_the_plain_one(dev, elem, window):
    """Trees of many sizes, verified step after step, give the tokens that decoding one by one gives,
    and leave the same cache."""
    note(f"drafted answer {elem} {window}")
    rng = np.random.default_rng(11)
    m = Model(dev, window=window)
    prompt = rng.integers(0, VOCAB, 20)
    plain = m.cache(elem)
    want = [int(m.forward(plain, prompt, 0)[-1])]
    while len(want) < 90:
        want.append(int(m.forward(plain, [want[-1]], len(prompt) + len(want) - 1)[0]))
    kv = m.cache(elem)
    got = [int(m.forward(kv, prompt, 0)[-1])]
    steps = 0
    while len(got) < 80:
        n, pos = int(rng.integers(1, 40)), len(prompt) + len(got) - 1
        parents, tokens = draft(rng, n, got[-1], want[len(got):])
        x = eb.Tensor.from_f32(dev, (n, HIDDEN), m.emb[tokens])
        rec = eb.Recorder(dev)
        tt, pt = eb.Tensor.from_u32(dev, (n,), tokens), eb.Tensor.from_array(dev, np.asarray(parents, np.int32))
        path, emitted, count = m.step(rec, kv, x, tt, pt, n, pos)
        rec.submit()
        c = int(u32(count)[0])
        assert 1 <= c <= n and u32(path)[0] == 0
        got += u32(emitted)[:c].tolist()
        steps += 1
    assert got == want[:len(got)]
    assert steps < len(got) - 20  # (branches were taken)
    width = HKV * HD
    for l in range(LAYERS):
        for a, b in ((kv.k[l], plain.k[l]), (kv.v[l], plain.v[l])):
            x, y = (np.frombuffer(t.read_bytes(), np.uint8).reshape(SEQ, -1)[:len(prompt) + len(got) - 1] for t in (a, b))
            if elem == "F32":
                x, y = x.copy().view(np.float32), y.copy().view(np.float32)
                assert x.shape[1] == width and np.abs(x - y).max() < 1e-4
            elif elem == "F16":
                x, y = x.copy().view(np.float16).astype(np.float32), y.copy().view(np.float16).astype(np.float32)
                assert np.abs(x - y).max() <= 2.0 ** -9 * max(1.0, np.abs(y).max())


@pytest.mark.parametrize("elem", ["F32", "F16", "F8E4M3", "i8"])
@pytest.mark.parametrize("n,window", [(1, 0), (23, 0), (23, 7), (70, 30)])
def test_layer_is_its_parts(dev, elem, n, window):
    """forward_tree_qkv = the rows at their positions, their cache rows, the attention."""
    note(f"layer {elem} {n} {window}")
    rng = np.random.default_rng(n)
    pos, rope = 60, eb.Rope.build(dev, SEQ, HD, 1e4)
    nodes = Nodes(dev, random_parents(n, rng))
    gains = [eb.Tensor.from_f32(dev, (HD,), rng.uniform(0.7, 1.3, HD)) for _ in range(3)]
    a = eb.Attention(H, HKV, HD, 0.2, *gains, window=window)
    q, k, v = (rng.standard_normal((n, w * HD)).astype(np.float32) for w in (H, HKV, HKV))
    qt, kt, vt = (eb.Tensor.from_f32(dev, x.shape, x) for x in (q, k, v))
    old = [eb.Tensor.from_f32(dev, (pos, HKV, HD), rows(rng, pos, HKV, HD)) for _ in range(2)]

    def cache():
        rec = eb.Recorder(dev)
        if elem == "i8":
            kv = eb.KvCache.new_i8(dev, 1, SEQ, HKV, HD, 16)
            eb.kv_write_i8(rec, kv, 0, *old, pos, 0)
        else:
            kv = eb.KvCache.new(dev, 1, SEQ, HKV, HD, eb.DType[elem])
            for x, t in zip(old, (kv.k[0], kv.v[0])):
                eb.kv_write(rec, t, x, HKV, pos, HD, SEQ, 0)
        rec.submit()
        return kv

    kv, parts = cache(), cache()
    rec = eb.Recorder(dev)
    out = a.forward_tree_qkv(rec, qt, kt, vt, rope, kv, 0, nodes.masks, nodes.depths, n, pos)
    qo, o = eb.Tensor.empty(dev, (n, H, HD)), eb.Tensor.empty(dev, (n, H, HD))
    if elem == "i8":
        f32 = eb.KvCache.new(dev, 1, SEQ, HKV, HD)
        eb.attn_prologue_tree(rec, qt, kt, vt, nodes.depths, qo, f32.k[0], f32.v[0], n, H, HKV, HD, pos, SEQ, *gains, 1e-6,
                              rope.cos, rope.sin)
        rec.submit()
        new = [t.to_f32().reshape(SEQ, HKV, HD)[pos:pos + n] for t in (f32.k[0], f32.v[0])]
        new = [eb.Tensor.from_f32(dev, x.shape, x) for x in new]
        rec = eb.Recorder(dev)
        eb.kv_write_i8(rec, parts, 0, *new, n, pos)
        eb.attn_tree_i8(rec, qo, parts, 0, nodes.masks, nodes.depths, o, H, pos, n, 0.2, window)
    else:
        eb.attn_prologue_tree(rec, qt, kt, vt, nodes.depths, qo, parts.k[0], parts.v[0], n, H, HKV, HD, pos, SEQ, *gains,
                              1e-6, rope.cos, rope.sin)
        eb.attn_tree(rec, qo, parts.k[0], parts.v[0], nodes.masks, nodes.depths, o, H, HKV, pos, n, HD, SEQ, 0.2, window)
    rec.submit()
    assert out.shape == (n, H * HD) and out.read_bytes() == o.read_bytes()
    if elem == "F32":
        kk, vv = (t.to_f32().reshape(SEQ, HKV, HD)[:pos + n] for t in (kv.k[0], kv.v[0]))
        want, bound = attention(qo.to_f32().reshape(n, H, HD), kk, vv, visible(nodes.seen, nodes.depth, pos, window), 0.2)
        check(out.to_f32().reshape(n, H, HD), want, bound, "layer")


@pytest.mark.parametrize("elem", ["F32", "i8"])
def test_captured_step(dev, elem):
    """One graph of a whole step: replays with other trees and tokens equal the eager step, with eager
    work between the replays."""
    note(f"captured step {elem}")
    rng = np.random.default_rng(5)
    m = Model(dev, seed=3, window=11)
    n, pos = 26, 40
    base = m.cache(elem)
    m.forward(base, rng.integers(0, VOCAB, pos), 0)
    kv, eager = m.cache(elem), m.cache(elem)
    x = eb.Tensor.empty(dev, (n, HIDDEN))
    tt, pt = eb.Tensor.empty(dev, (n,), eb.DType.U32), eb.Tensor.empty(dev, (n,), eb.DType.I32)

    def trees():
        parents, tokens = draft(rng, n, int(rng.integers(0, VOCAB)), [])
        x.write(m.emb[tokens])
        tt.write(tokens)
        pt.write(np.asarray(parents, np.int32))
        return tokens, parents

    def whole(cache):
        rec = eb.Recorder(dev)
        eb.kv_fork(rec, cache, base, pos)
        out = m.step(rec, cache, x, tt, pt, n, pos)
        rec.submit()
        return out

    trees()
    whole(eager)  # (the workspace is there)
    dev.synchronize()
    dev.begin_capture()
    outs = whole(kv)
    graph = dev.end_capture()
    for i in range(6):
        tokens, parents = trees()
        if i % 2:  # (what the root's answer will be, drafted behind it: at least two nodes accepted)
            first = u32(whole(eager)[1])[0]
            tokens[1] = first
            x.write(m.emb[tokens])
            tt.write(tokens)
        graph.launch()
        want = [t.read_bytes() for t in whole(eager)]
        dev.synchronize()
        assert [t.read_bytes() for t in outs] == want
        count = int(u32(outs[2])[0])
        assert count >= 1 + i % 2
        for l in range(LAYERS):
            for a, b in ((kv.k[l], eager.k[l]), (kv.v[l], eager.v[l])):
                row = a.byte_len() // SEQ
                assert a.read_bytes()[:row * (pos + count)] == b.read_bytes()[:row * (pos + count)]
    graph.release()


def test_two_graphs_share_the_workspace(dev):
    """Two captured attentions of unlike size, replayed in turn beside eager work that grows it."""
    rng = np.random.default_rng(6)
    cases = []
    for n, pos, h, hkv, hd in ((20, 3000, 16, 8, 128), (64, 900, 8, 2, 64)):
        kt, vt = (eb.Tensor.from_f32(dev, (pos + n, hkv, hd), rows(rng, pos + n, hkv, hd)) for _ in range(2))
        qt = eb.Tensor.from_f32(dev, (n, h, hd), rng.standard_normal((n, h, hd)))
        nodes = Nodes(dev, random_parents(n, rng))
        cases.append((n, pos, h, hkv, hd, kt, vt, qt, nodes, eb.Tensor.empty(dev, (n, h, hd))))

    def call(c):
        n, pos, h, hkv, hd, kt, vt, qt, nodes, o = c
        rec = eb.Recorder(dev)
        eb.attn_tree(rec, qt, kt, vt, nodes.masks, nodes.depths, o, h, hkv, pos, n, hd, pos + n, 0.1)
        rec.submit()

    want, graphs = [], []
    for c in cases:
        call(c)
        want.append(c[-1].read_bytes())
        dev.begin_capture()
        call(c)
        graphs.append(dev.end_capture())
    for i in range(4):
        for g in graphs:
            g.launch()
        if i == 1:  # (an eager call that may outgrow the workspace)
            seq = 40000
            kv = eb.KvCache.new(dev, 1, seq, 1, 128, eb.DType.F16)
            nodes = Nodes(dev, [-1] + [0] * 255)
            q, o = (eb.Tensor.from_f32(dev, (256, 4, 128), np.zeros((256, 4, 128), np.float32)) for _ in range(2))
            rec = eb.Recorder(dev)
            eb.attn_tree(rec, q, kv.k[0], kv.v[0], nodes.masks, nodes.depths, o, 4, 1, seq - 256, 256, 128, seq, 0.1)
            rec.submit()
        dev.synchronize()
        for c, w in zip(cases, want):
            assert c[-1].read_bytes() == w
            c[-1].write(np.zeros(c[-1].numel(), np.float32))


def test_refused_handles(dev):
    """Tensors and caches of other types, shapes or devices."""
    n = 4
    nodes = Nodes(dev, [-1, 0, 0, 1])
    kv, kv8 = eb.KvCache.new(dev, 2, 32, 2, 64), eb.KvCache.new_i8(dev, 2, 32, 2, 64, 16)
    q, o = (eb.Tensor.empty(dev, (n, 4, 64)) for _ in range(2))
    rec = eb.Recorder(dev)
    ids = eb.Tensor.empty(dev, (n,), eb.DType.U32)
    f = eb.Tensor.empty(dev, (n,))
    for bad in (lambda: eb.attn_tree(rec, q, kv8.k[0], kv8.v[0], nodes.masks, None, o, 4, 2, 8, n, 64, 32, 0.1),
                lambda: eb.attn_tree(rec, q, kv.k[0], kv.v[0], f, None, o, 4, 2, 8, n, 64, 32, 0.1),
                lambda: eb.attn_tree(rec, q, kv.k[0], kv.v[0], nodes.masks, None, o, 4, 2, 8, n, 64, 32, 0.1, 5),
                lambda: eb.attn_tree(rec, ids, kv.k[0], kv.v[0], nodes.masks, None, o, 4, 2, 8, n, 64, 32, 0.1),
                lambda: eb.attn_tree(rec, q, kv.k[0], kv.v[0], nodes.masks, None, o, 4, 2, 29, n, 64, 32, 0.1),
                lambda: eb.attn_tree_i8(rec, q, kv, 0, nodes.masks, None, o, 4, 8, n, 0.1),
                lambda: eb.attn_tree_i8(rec, q, kv8, 2, nodes.masks, None, o, 4, 8, n, 0.1),
                lambda: eb.tree_plan(rec, ids, nodes.masks, nodes.depths, n),
                lambda: eb.tree_accept(rec, ids, ids, ids, ids, ids, ids, n),
                lambda: eb.kv_compact(rec, kv, ids, f, n, 8),
                lambda: eb.kv_compact(rec, kv, ids, ids, n, 29),
                lambda: eb.kv_compact(rec, kv, ids, ids, 5, 8),
                lambda: eb.kv_fork(rec, kv, kv, 4),
                lambda: eb.kv_fork(rec, kv, kv8, 4),
                lambda: eb.kv_fork(rec, kv, eb.KvCache.new(dev, 1, 32, 2, 64), 4),
                lambda: eb.kv_fork(rec, kv, eb.KvCache.new(dev, 2, 32, 1, 64), 4),
                lambda: eb.kv_fork(rec, kv, eb.KvCache.new(dev, 2, 32, 2, 32), 4),
                lambda: eb.kv_fork(rec, kv, eb.KvCache.new(dev, 2, 32, 2, 64, eb.DType.F16), 4),
                lambda: eb.kv_fork(rec, kv8, eb.KvCache.new_i8(dev, 2, 32, 2, 64, 32), 4),
                lambda: eb.kv_fork(rec, kv, eb.KvCache.new(dev, 2, 16, 2, 64), 17)):
        with pytest.raises(eb.ShapeMismatch):
            bad()
    other = eb.Device.new(0)
    far = eb.KvCache.new(other, 2, 32, 2, 64)
    for bad in (lambda: eb.kv_fork(rec, kv, far, 4), lambda: eb.kv_compact(rec, far, ids, ids, n, 8),
                lambda: eb.attn_tree(rec, q, far.k[0], far.v[0], nodes.masks, None, o, 4, 2, 8, n, 64, 32, 0.1)):
        with pytest.raises(eb.EyebrowseError, match="another device"):
            bad()
    a = eb.Attention(4, 2, 64, 0.1)
    rope = eb.Rope.build(dev, 32, 64, 1e4)
    k, v = (eb.Tensor.empty(dev, (n, 2, 64)) for _ in range(2))
    with pytest.raises(eb.ShapeMismatch):  # rows past the cache
        a.forward_tree_qkv(rec, q, k, v, rope, kv, 0, nodes.masks, nodes.depths, n, 29)
    with pytest.raises(eb.ShapeMismatch):  # rows past the tables
        a.forward_tree_qkv(rec, q, k, v, eb.Rope.build(dev, 10, 64, 1e4), kv, 0, nodes.masks, nodes.depths, n, 8)
    with pytest.raises(eb.ShapeMismatch):
        a.forward_tree_qkv(rec, q, k, v, eb.Rope.build(dev, 10, 64, 1e4), kv8, 0, nodes.masks, nodes.depths, n, 8)
    with pytest.raises(eb.ShapeMismatch):  # another cache's heads
        a.forward_tree_qkv(rec, q, k, v, rope, eb.KvCache.new(dev, 1, 32, 1, 128), 0, nodes.masks, nodes.depths, n, 8)
    rec.submit()


def test_accept_follows_the_plan(dev):
    """Plan and walk of one tree agree: the path is the accepted leaf's own ancestors."""
    rng = np.random.default_rng(9)
    for n in (3, 40, 256):
        parents, tokens = draft(rng, n, 1, rng.integers(0, VOCAB, 50))
        nodes = Nodes(dev, parents)
        sampled = np.asarray([tokens[i + 1] if i + 1 < n else 0 for i in range(n)], np.uint32)
        want = accept(tokens, parents, sampled)
        assert nodes.depth[want[-1]] == len(want) - 1
        assert np.flatnonzero(nodes.seen[want[-1]]).tolist() == want
