"""Drafts over a block-scaled cache: what they leave in it, and whom a draft that is not finite reaches."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._tree import Nodes, random_parents, rows

pytestmark = pytest.mark.gpu

EPS = 1e-6


class Layer:
    """One attention layer over block-scaled caches of `pos` rows, and a tree of n nodes behind them."""

    def __init__(self, dev, block, hd, pos, n, seed=0, h=4, hkv=2, window=0):
        self.dev, self.h, self.hkv, self.hd, self.pos, self.n, self.block = dev, h, hkv, hd, pos, n, block
        rng = np.random.default_rng(seed + 31 * block + pos)
        self.rng, self.seq = rng, pos + n + 40
        self.nodes = Nodes(dev, random_parents(n, rng))
        self.rope = eb.Rope.build(dev, self.seq, hd, 1e4)
        # (K has a norm and V has none: V rows keep their sizes)
        self.gains = [eb.Tensor.from_f32(dev, (hd,), rng.uniform(0.7, 1.3, hd)) for _ in range(2)] + [None]
        self.attn = eb.Attention(h, hkv, hd, 0.2, *self.gains, EPS, window)
        self.old = [rows(rng, pos, hkv, hd) for _ in range(2)]
        self.q, self.k, self.v = (rng.standard_normal((n, w, hd)).astype(np.float32) for w in (h, hkv, hkv))

    def cache(self):
        kv = eb.KvCache.new_i8(self.dev, 1, self.seq, self.hkv, self.hd, self.block)
        if self.pos:
            self.write(kv, *self.old, 0)
        return kv

    def write(self, kv, k, v, at):
        rec = eb.Recorder(self.dev)
        kt, vt = (eb.Tensor.from_f32(self.dev, x.shape, x) for x in (k, v))
        eb.kv_write_i8(rec, kv, 0, kt, vt, len(k), at)
        rec.submit()

    def forward(self, kv):
        rec = eb.Recorder(self.dev)
        qt, kt, vt = (eb.Tensor.from_f32(self.dev, x.shape, x) for x in (self.q, self.k, self.v))
        out = self.attn.forward_tree_qkv(rec, qt, kt, vt, self.rope, kv, 0, self.nodes.masks, self.nodes.depths,
                                         self.n, self.pos)
        rec.submit()
        return out.to_f32().reshape(self.n, self.h, self.hd)

    def final_rows(self):
        """The nodes' K and V as the row pass makes them."""
        f32 = eb.KvCache.new(self.dev, 1, self.seq, self.hkv, self.hd)
        qt, kt, vt = (eb.Tensor.from_f32(self.dev, x.shape, x) for x in (self.q, self.k, self.v))
        rec = eb.Recorder(self.dev)
        eb.attn_prologue_tree(rec, qt, kt, vt, self.nodes.depths, eb.Tensor.empty(self.dev, self.q.shape), f32.k[0],
                              f32.v[0], self.n, self.h, self.hkv, self.hd, self.pos, self.seq, *self.gains, EPS,
                              self.rope.cos, self.rope.sin)
        rec.submit()
        return [t.to_f32().reshape(self.seq, self.hkv, self.hd)[self.pos:self.pos + self.n] for t in (f32.k[0], f32.v[0])]

    def compact(self, kv, path, n=None):
        n = n or self.n
        padded = np.full(n, 0xFFFFFFFF, np.uint32)
        padded[:len(path)] = path
        pt, ct = eb.Tensor.from_u32(self.dev, (n,), padded), eb.Tensor.from_u32(self.dev, (1,), [len(path)])
        rec = eb.Recorder(self.dev)
        eb.kv_compact(rec, kv, pt, ct, n, self.pos)
        rec.submit()

    def bytes(self, kv, rows_):
        """Codes of the first rows and the exponents of their blocks."""
        out = []
        for codes, exps in ((kv.k[0], kv.k_scale[0]), (kv.v[0], kv.v_scale[0])):
            out.append(codes.read_bytes()[:rows_ * self.hkv * self.hd])
            out.append(exps.read_bytes()[:-(-rows_ // self.block) * self.hkv])
        return out


def branch(nodes, leaf):
    return np.flatnonzero(nodes.seen[leaf]).tolist()


@pytest.mark.parametrize("block,hd,pos,n", [(16, 32, 13, 20), (16, 64, 16, 40), (64, 128, 40, 20), (256, 96, 100, 200),
                                            (32, 256, 0, 9), (64, 64, 700, 256), (16, 48, 5, 1)])
@pytest.mark.parametrize("rejected", [1.0, 1e4, np.inf])
def test_rejected_drafts_leave_no_trace(dev, block, hd, pos, n, rejected):
    """After a step the cache holds what writing the accepted rows alone would have left there, whatever
    the others held; between the pass and the compaction it holds what it did before."""
    note(f"i8 drafts, block {block} hd {hd} pos {pos} n {n} rejected {rejected}")
    x = Layer(dev, block, hd, pos, n)
    for leaf in {0, n // 2, n - 1}:
        path = branch(x.nodes, leaf)
        v = x.v.copy()
        out = np.setdiff1d(np.arange(n), path)
        if len(out):
            x.v[out[::2], :, 3] *= np.float32(rejected)
        kv, plain = x.cache(), x.cache()
        x.forward(kv)
        assert x.bytes(kv, pos) == x.bytes(plain, pos)
        k_new, v_new = x.final_rows()
        x.compact(kv, path)
        x.write(plain, k_new[path], v_new[path], pos)
        assert x.bytes(kv, pos + len(path)) == x.bytes(plain, pos + len(path)), path
        x.v = v


def test_nothing_accepted_and_abandoned(dev):
    """A draft that is dropped (an empty path, or no compaction) leaves the cache to plain decoding."""
    note("i8 drafts, abandoned")
    x = Layer(dev, 64, 64, 40, 20)
    x.v[5] *= 1e6
    plain = x.cache()
    for compacted in (False, True):
        kv = x.cache()
        x.forward(kv)
        if compacted:
            x.compact(kv, [])
        assert x.bytes(kv, x.pos) == x.bytes(plain, x.pos)
        outs = []
        for c in (kv, x.cache()):
            rec = eb.Recorder(dev)
            q, k, v = (eb.Tensor.from_f32(dev, t[:1].shape, t[:1]) for t in (x.q, x.k, x.v))
            o = x.attn.forward_qkv(rec, q, k, v, x.rope, c, 0, 1, x.pos)
            rec.submit()
            outs.append((o.read_bytes(), *x.bytes(c, x.pos + 1)))
        assert outs[0] == outs[1]


@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("window", [0, 9])
def test_draft_that_is_not_finite(dev, side, what, window):
    """It makes the heads of the nodes that see it NaN and no others: the rest answer as if its row were
    zeros; accepted, its block becomes NaN as in any write."""
    note(f"i8 drafts, {side} {what} window {window}")
    for block, hd, pos, n in ((64, 64, 40, 30), (16, 128, 500, 70), (32, 256, 33, 21)):
        x = Layer(dev, block, hd, pos, n, window=window)
        bad, head = 2, 1
        kin = x.nodes.seen[:, bad] & ((x.nodes.depth - x.nodes.depth[bad] < window) | (window == 0))
        assert 1 <= kin.sum() < n
        a = x.v if side == "v" else x.k
        a[bad, head] = 0
        want = x.forward(x.cache())
        a[bad, head, 7] = what
        kv = x.cache()
        got = x.forward(kv)
        mine = slice(head * 2, head * 2 + 2)
        assert np.isnan(got[kin][:, mine]).all()
        hit = np.zeros(got.shape, bool)
        hit[np.ix_(kin, [2, 3])] = True
        assert got[~hit].tobytes() == want[~hit].tobytes()
        path, plain = branch(x.nodes, bad), x.cache()
        k_new, v_new = x.final_rows()
        x.compact(kv, path)
        x.write(plain, k_new[path], v_new[path], pos)
        assert x.bytes(kv, pos + len(path)) == x.bytes(plain, pos + len(path))


def test_graphs_apart(dev):
    """Pass and compaction captured as graphs of their own, replayed with other rows, beside an eager draft
    over the same cache."""
    note("i8 drafts, graphs apart")
    x = Layer(dev, 64, 64, 40, 24)
    kv = x.cache()
    path = branch(x.nodes, 23)
    ins = [eb.Tensor.from_f32(dev, t.shape, t) for t in (x.q, x.k, x.v)]
    padded = np.full(x.n, 0xFFFFFFFF, np.uint32)
    padded[:len(path)] = path
    pt, ct = eb.Tensor.from_u32(dev, (x.n,), padded), eb.Tensor.from_u32(dev, (1,), [len(path)])

    def step():
        rec = eb.Recorder(dev)
        x.attn.forward_tree_qkv(rec, *ins, x.rope, kv, 0, x.nodes.masks, x.nodes.depths, x.n, x.pos)
        rec.submit()

    def move():
        rec = eb.Recorder(dev)
        eb.kv_compact(rec, kv, pt, ct, x.n, x.pos)
        rec.submit()

    def again():
        rec = eb.Recorder(dev)
        eb.kv_fork(rec, kv, base, x.pos)
        rec.submit()

    base = x.cache()
    step()
    dev.synchronize()
    graphs = []
    for f in (step, move):
        dev.begin_capture()
        f()
        graphs.append(dev.end_capture())
    for i in range(4):
        again()
        x.v = x.rng.standard_normal(x.v.shape).astype(np.float32) * np.float32(10.0 ** (i - 1))
        ins[2].write(x.v)
        graphs[0].launch()
        if i == 2:  # (an eager pass of the same rows and its own compaction come first)
            dev.synchronize()
            x.compact(kv, [0])
            again()
            graphs[0].launch()
        graphs[1].launch()
        dev.synchronize()
        plain = x.cache()
        k_new, v_new = x.final_rows()
        x.write(plain, k_new[path], v_new[path], x.pos)
        assert x.bytes(kv, x.pos + len(path)) == x.bytes(plain, x.pos + len(path)), i
    for g in graphs:
        g.release()


@pytest.mark.parametrize("how", ["write", "prompt", "step", "raw"])
def test_rows_written_after_a_draft(dev, how):
    """Rows that the caller puts into the cache are what a compaction moves from then on: written, as a
    prompt's chunk, one by one, and one by one without the layer."""
    note(f"i8 drafts, rows written after one: {how}")
    x = Layer(dev, 16, 64, 40, 12)
    kv, other = x.cache(), x.cache()
    x.forward(kv)
    k, v = (rows(x.rng, x.n, x.hkv, x.hd) for _ in range(2))
    q = x.rng.standard_normal((x.n, x.h, x.hd)).astype(np.float32)
    for c in (kv, other):
        rec = eb.Recorder(dev)
        if how == "write":
            x.write(c, k, v, x.pos)
        elif how == "prompt":
            qt, kt, vt = (eb.Tensor.from_f32(dev, t.shape, t) for t in (q, k, v))
            x.attn.forward_qkv(rec, qt, kt, vt, x.rope, c, 0, x.n, x.pos)
        else:
            for i in range(x.n):
                qt, kt, vt = (eb.Tensor.from_f32(dev, t[i:i + 1].shape, t[i:i + 1]) for t in (q, k, v))
                if how == "step":
                    x.attn.forward_qkv(rec, qt, kt, vt, x.rope, c, 0, 1, x.pos + i)
                else:
                    eb.attn_decode_step_i8(rec, qt, kt, vt, c, 0, eb.Tensor.empty(dev, (x.h, x.hd)), x.h, x.pos + i, 0.1)
        rec.submit()
        x.compact(c, [0, 3, 7])
    assert x.bytes(kv, x.pos + x.n) == x.bytes(other, x.pos + x.n)


def test_many_layers(dev):
    """More layers than a launch of the compaction takes, of unlike head dims, each with its own draft; a
    draft of another pos, and one that a fork replaced, are not what is moved."""
    note("i8 drafts, many layers")
    rng = np.random.default_rng(7)
    dims, hkv, h, n, pos, block = [32, 96, 64] * 23, 2, 4, 18, 45, 32
    seq = pos + n + 3
    kv, plain = (eb.KvCache.new_i8_per_layer(dev, dims, seq, hkv, block) for _ in range(2))
    nodes = Nodes(dev, random_parents(n, rng))
    ropes = {hd: eb.Rope.build(dev, seq, hd, 1e4) for hd in set(dims)}
    attns = {hd: eb.Attention(h, hkv, hd, 0.2) for hd in set(dims)}
    path = branch(nodes, n - 1)
    pt, ct = (eb.Tensor.from_u32(dev, (len(x),), x) for x in (path + [0xFFFFFFFF] * (n - len(path)), [len(path)]))

    def up(x):
        return eb.Tensor.from_f32(dev, x.shape, x)

    def draft(at, layers):
        """A tree pass; the rows it makes."""
        made = []
        rec = eb.Recorder(dev)
        for l in layers:
            hd = dims[l]
            q, k, v = (up(rng.standard_normal((n, w, hd)).astype(np.float32)) for w in (h, hkv, hkv))
            attns[hd].forward_tree_qkv(rec, q, k, v, ropes[hd], kv, l, nodes.masks, nodes.depths, n, at)
            f32 = eb.KvCache.new(dev, 1, seq, hkv, hd)
            eb.attn_prologue_tree(rec, q, k, v, nodes.depths, eb.Tensor.empty(dev, (n, h, hd)), f32.k[0], f32.v[0], n, h,
                                  hkv, hd, at, seq, None, None, None, 1e-6, ropes[hd].cos, ropes[hd].sin)
            made.append(f32)
        rec.submit()
        return [[t.to_f32().reshape(seq, hkv, dims[l])[at:at + n] for t in (m.k[0], m.v[0])] for l, m in zip(layers, made)]

    rec = eb.Recorder(dev)
    for l, hd in enumerate(dims):
        x = [up(rows(rng, pos, hkv, hd)) for _ in range(2)]
        for c in (kv, plain):
            eb.kv_write_i8(rec, c, l, *x, pos, 0)
    rec.submit()
    draft(pos - 3, range(0, len(dims), 2))  # (dropped: another pos)
    made = draft(pos, range(len(dims)))
    rec = eb.Recorder(dev)
    eb.kv_compact(rec, kv, pt, ct, n, pos)
    for l, new in enumerate(made):
        eb.kv_write_i8(rec, plain, l, *(up(x[path]) for x in new), len(path), pos)
    rec.submit()

    def same(rows_):
        for l, hd in enumerate(dims):
            for a, b, e, f in ((kv.k, plain.k, kv.k_scale, plain.k_scale), (kv.v, plain.v, kv.v_scale, plain.v_scale)):
                assert a[l].read_bytes()[:rows_ * hkv * hd] == b[l].read_bytes()[:rows_ * hkv * hd], l
                assert e[l].read_bytes()[:-(-rows_ // block) * hkv] == f[l].read_bytes()[:-(-rows_ // block) * hkv], l

    same(pos + len(path))
    # A draft, then all rows of another cache: its rows at pos are the ones that a compaction moves.
    draft(pos, range(len(dims)))
    rec = eb.Recorder(dev)
    eb.kv_fork(rec, kv, plain, seq)
    for c in (kv, plain):
        eb.kv_compact(rec, c, pt, ct, n, pos)
    rec.submit()
    same(seq)


@pytest.mark.parametrize("block", [64, 256])
@pytest.mark.parametrize("pos", [64, 69, 200])
def test_pass_rounds_sixteen_rows_together(dev, block, pos):
    """What the nodes see: the cache's rows as they are, but those of pos's aligned 16, and the nodes' own,
    coded as by a cache whose blocks are 16 rows."""
    note(f"i8 drafts, sixteen rows together, block {block} pos {pos}")
    x = Layer(dev, block, 64, pos, 40)
    x.v[20] *= 300  # (its neighbours only are rounded to its exponent)
    got = x.forward(x.cache())
    # The same codes, in a cache of blocks of 16.
    kv, fine = x.cache(), eb.KvCache.new_i8(dev, 1, x.seq, x.hkv, x.hd, 16)
    for a, b, e, f in ((kv.k, fine.k, kv.k_scale, fine.k_scale), (kv.v, fine.v, kv.v_scale, fine.v_scale)):
        b[0].write(a[0].read_bytes())
        exps = np.frombuffer(e[0].read_bytes(), np.uint8).reshape(-1, x.hkv)
        f[0].write(np.repeat(exps, block // 16, 0)[:-(-x.seq // 16)].copy())
    k_new, v_new = x.final_rows()
    x.write(fine, k_new, v_new, pos)
    f32 = eb.KvCache.new(dev, 1, x.seq, x.hkv, x.hd)
    qo, o = (eb.Tensor.empty(dev, x.q.shape) for _ in range(2))
    qt, kt, vt = (eb.Tensor.from_f32(dev, t.shape, t) for t in (x.q, x.k, x.v))
    rec = eb.Recorder(dev)
    eb.attn_prologue_tree(rec, qt, kt, vt, x.nodes.depths, qo, f32.k[0], f32.v[0], x.n, x.h, x.hkv, x.hd, pos, x.seq,
                          *x.gains, EPS, x.rope.cos, x.rope.sin)
    eb.attn_tree_i8(rec, qo, fine, 0, x.nodes.masks, None, o, x.h, pos, x.n, 0.2)
    rec.submit()
    assert got.tobytes() == o.read_bytes()
