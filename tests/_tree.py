"""A drafted tree's operators written from their definitions in 64 bits, with numpy."""
import numpy as np

import eyebrowse_amd as eb

NOBODY = 0xFFFFFFFF


def random_parents(n, rng, width=6, roots=1):
    """Parents of a tree of n nodes; the first `roots` have none."""
    return [-1] * min(n, roots) + [max(0, i - int(rng.integers(1, width + 1))) for i in range(roots, n)]


def plan(parents):
    """(masks as booleans [n, n], depths [n])."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen, seen.sum(1) - 1


def words(seen):
    """Boolean masks [n, n] as u32 words [n, ceil(n / 32)]."""
    n = seen.shape[1]
    w = -(-n // 32)
    bits = np.zeros((seen.shape[0], 32 * w), np.uint64)
    bits[:, :n] = seen
    return (bits.reshape(-1, w, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def accept(tokens, parents, sampled):
    """The accepted path."""
    path = [0]
    while True:
        at = path[-1]
        fit = [i for i in range(at + 1, len(tokens)) if parents[i] == at and tokens[i] == sampled[at]]
        if not fit:
            return path
        path.append(fit[0])


def visible(seen, depths, pos, window):
    """Which of the keys 0 .. pos + n - 1 each node sees: [n, pos + n]."""
    n = len(seen)
    at = np.concatenate((np.arange(pos), pos + np.asarray(depths, np.int64)))
    mine = at[pos:, None]
    vis = np.concatenate((np.ones((n, pos), bool), np.asarray(seen, bool)), 1)
    return vis & (at[None] > mine - window) if window else vis


def attention(q, k, v, vis, scale):
    """(output, bound on its error) of q [n, h, hd] over keys k, v [pos + n, hkv, hd] in 64 bits.

    A value split into two f16 halves, each rounded to nearest (half a step, 2^-11 relative), keeps
    2^-22 of itself; q, k, v and the weights are such pairs (narrow caches' k and v are exact), and the
    product of two low halves, up to 2^-22 of the product, is left out. A score in log2 units is a sum
    of 3 hd products in f32 (2^-24 each) and three exact or once-rounded factors: it is off by at most
    (3 2^-22 + (3 hd + 4) 2^-24) S, S = the largest sum of |q k| scale log2(e). x - m is rounded once
    and 2^x is good to 2^-22: with |x| <= 2 S a weight is off by ln 2 times all that, relative to
    itself. Numerator and denominator carry it, then the numerator 3 2^-22 (the split of weight and
    value), the sums 3 n + 64 roundings of 2^-24 each (64: rescales and the merge), and the quotient
    2^-22. The smallest half is a step of 2^-24, where the column's largest term is at least 2^6 times
    its value's scale of 2^13: 2^-24 / 2 / 2^19 of it, less than 2^-40 for each key and half."""
    n, h, hd = q.shape
    keys, hkv = k.shape[:2]
    g = h // hkv
    qd = np.asarray(q, np.float64)
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    some = vis.any(1)
    for j in range(hkv):
        kj, vj = np.asarray(k[:, j], np.float64), np.asarray(v[:, j], np.float64)
        for a in range(j * g, (j + 1) * g):
            x = np.where(vis, (qd[:, a] @ kj.T) * scale, -np.inf)
            size = np.where(vis, (np.abs(qd[:, a]) @ np.abs(kj).T) * abs(scale) * np.log2(np.e), 0).max(1)
            p = np.exp(x - np.where(some, x.max(1, initial=-np.inf), 0)[:, None])
            p /= np.where(some, p.sum(1), 1)[:, None]
            out[:, a] = p @ vj
            mass = p @ np.abs(vj)
            score = (3 * 2.0 ** -22 + (3 * hd + 4) * 2.0 ** -24) * size
            weight = np.log(2) * (score + 2.0 ** -24 * 2 * size) + 2.0 ** -22
            rel = 2 * weight + 4 * 2.0 ** -22 + 2 * (3 * keys + 64) * 2.0 ** -24
            largest = (p * np.abs(vj).max(1)).max(1)
            bound[:, a] = rel[:, None] * mass + (keys * 2.0 ** -39 * largest)[:, None] + 1e-35
    return out, bound


class Nodes:
    """A tree's arrays on the device."""

    def __init__(self, dev, parents=None, seen=None, depths=None):
        if parents is not None:
            seen, depths = plan(parents)
            self.parents = eb.Tensor.from_array(dev, np.asarray(parents, np.int32))
        self.n = len(seen)
        self.seen, self.depth = np.asarray(seen, bool), np.asarray(depths)
        self.masks = eb.Tensor.from_array(dev, words(self.seen))
        self.depths = eb.Tensor.from_array(dev, self.depth.astype(np.uint32))


def u32(t):
    return np.frombuffer(t.read_bytes(), np.uint32).reshape(t.shape)


# ---- caches of every element type, by their values ---------------------------------------

def e4m3_values(codes):
    """OCP E4M3 patterns as float64."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    e, f = (c >> 3) & 15, c & 7
    x = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    x = np.where((c & 0x7F) == 0x7F, np.nan, x)
    return np.where(c & 0x80, -x, x)


def rows(rng, n, hkv, hd):
    """n rows of unlike size, and the same for channels."""
    x = rng.standard_normal((n, hkv, hd)) * np.exp(0.4 * rng.standard_normal((1, hkv, hd)))
    return (x * np.exp(0.3 * rng.standard_normal((n, 1, 1)))).astype(np.float32)


class Cache:
    """One layer's K and V on the device with `have` rows written, and their values."""

    def __init__(self, dev, elem, max_seq, hkv, hd, k, v, block=64):
        self.elem, self.hkv, self.hd, self.max_seq = elem, hkv, hd, max_seq
        have = len(k)
        rec = eb.Recorder(dev)
        if elem == "i8":
            self.kv = eb.KvCache.new_i8(dev, 1, max_seq, hkv, hd, block)
            kt, vt = (eb.Tensor.from_f32(dev, x.shape, x) for x in (k, v))
            eb.kv_write_i8(rec, self.kv, 0, kt, vt, have, 0)
            ko, vo = eb.Tensor.empty(dev, k.shape), eb.Tensor.empty(dev, v.shape)
            eb.kv_read_i8(rec, self.kv, 0, ko, vo, have, 0)
            rec.submit()
            self.k, self.v = (t.to_f32().reshape(k.shape) for t in (ko, vo))
        else:
            dt = {"f32": eb.DType.F32, "f16": eb.DType.F16, "e4m3": eb.DType.F8E4M3}[elem]
            self.kv = eb.KvCache.new(dev, 1, max_seq, hkv, hd, dt)
            for x, to in ((k, self.kv.k[0]), (v, self.kv.v[0])):
                eb.kv_write(rec, to, eb.Tensor.from_f32(dev, x.shape, x), hkv, have, hd, max_seq, 0)
            rec.submit()
            self.k, self.v = (self.read(t, have) for t in (self.kv.k[0], self.kv.v[0]))

    def read(self, t, have):
        raw = t.read_bytes()
        shape = (self.max_seq, self.hkv, self.hd)
        if self.elem == "f32":
            x = np.frombuffer(raw, np.float32)
        elif self.elem == "f16":
            x = np.frombuffer(raw, np.float16).astype(np.float32)
        else:
            x = e4m3_values(np.frombuffer(raw, np.uint8))
        return x.reshape(shape)[:have]

    def attend(self, dev, q, nodes, pos, scale, window=0, o=None):
        n, h, hd = q.shape
        qt = eb.Tensor.from_f32(dev, q.shape, q)
        ot = eb.Tensor.from_f32(dev, q.shape, np.full(q.shape, 7.0, np.float32))
        rec = eb.Recorder(dev)
        depths = nodes.depths if window else None
        if self.elem == "i8":
            eb.attn_tree_i8(rec, qt, self.kv, 0, nodes.masks, depths, ot, h, pos, n, scale, window)
        else:
            eb.attn_tree(rec, qt, self.kv.k[0], self.kv.v[0], nodes.masks, depths, ot, h, self.hkv, pos, n, hd,
                         self.max_seq, scale, window)
        rec.submit()
        return ot.to_f32().reshape(q.shape)


def check(got, want, bound, what):
    assert np.isfinite(got).all(), f"{what}: not finite"
    bad = np.abs(got - want) > bound
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} past the bound, worst "
                           f"{(np.abs(got - want) / bound).max():.2f} of it, largest error {np.abs(got - want).max():.2e}")
    rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert rel <= 2e-5, f"{what}: rel-L2 {rel:.2e}"
