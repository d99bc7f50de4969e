"""The quantised operators written from their definitions in 64 bits, with numpy."""
import numpy as np

from tests._textbook import attention_f64


# ---- block-scaled caches ----------------------------------------------------------------

class CacheModel:
    """One of a layer's two block-scaled caches: int8 codes and exponent bytes."""

    def __init__(self, max_seq, hkv, hd, block, rng=None):
        self.block = block
        nb = -(-max_seq // block)
        self.codes = np.zeros((max_seq, hkv, hd), np.int8)
        self.exps = np.ones((nb, hkv), np.uint8)
        if rng is not None:  # (stale rows, as a recycled buffer holds)
            self.codes[:] = rng.integers(-128, 128, self.codes.shape)

    def write(self, x, dst):
        x = np.asarray(x, np.float32)
        n, hkv, _ = x.shape
        bl = self.block
        for b in range(dst // bl, -(-(dst + n) // bl)):
            lo, hi = max(b * bl, dst), min((b + 1) * bl, dst + n)
            for h in range(hkv):
                new = x[lo - dst:hi - dst, h].astype(np.float64)
                top = np.abs(new).max()
                if not np.isfinite(new).all():
                    e = 255
                else:
                    e = 1
                    while top > 127 * 2.0 ** (e - 127):
                        e += 1
                if lo > b * bl:
                    old = int(self.exps[b, h])
                    e = max(e, old)
                    if old < e < 255:
                        kept = self.codes[b * bl:lo, h].astype(np.float64)
                        self.codes[b * bl:lo, h] = np.rint(kept * 2.0 ** (old - e))
                self.exps[b, h] = e
                self.codes[lo:hi, h] = 0 if e == 255 else np.rint(new * 2.0 ** (127 - e))

    def values(self, lo, hi):
        e = self.exps[np.arange(lo, hi) // self.block].astype(np.float64)
        f = np.where(e == 255, np.nan, 2.0 ** (e - 127))
        return self.codes[lo:hi].astype(np.float64) * f[..., None]


def attention_bound(q, k, v, scale, pos, window=0):
    """(output, bound on its error) of rows q at pos.. over keys k, v (row 0 is token 0) in 64 bits.

    The kernels keep 22 bits of q (2^-22 of each element) and sum hd products in f32, so a score in
    log2 units is off by at most (2^-22 + hd 2^-24) S, S = the largest sum of |q k| scale log2(e);
    x - m and 2^x add 2^-23 (|x| + 2); the weights keep 20 bits (two halves rounded toward zero), and
    n terms are summed in f32. Numerator and denominator each carry that, relative to the sum of
    p |v|. A weight's halves end at f16's 2^-24, and the largest term p |v| (v: its row's largest) of
    a column lies between a half and 2^9 of the unit they are in: each of the n terms is off by at
    most 2^-24 of twice the largest, besides."""
    hd, n = q.shape[-1], k.shape[0]
    out = attention_f64(q, k, v, scale, q_offset=pos, window=window)
    mass = attention_f64(q, k, np.abs(v), scale, q_offset=pos, window=window)
    g = q.shape[1] // k.shape[1]
    qd, kr = np.asarray(q, np.float64), np.repeat(np.asarray(k, np.float64), g, axis=1)
    s = float(np.einsum("thd,shd->ths", np.abs(qd), np.abs(kr)).max()) * abs(scale) * np.log2(np.e)
    x = np.einsum("thd,shd->ths", qd, kr) * scale
    at, key = pos + np.arange(len(q))[:, None, None], np.arange(n)[None, None]
    x = np.where((key > at) | ((window > 0) & (key <= at - window)), -np.inf, x)
    p = np.exp(x - x.max(-1, keepdims=True))
    largest = (p / p.sum(-1, keepdims=True) * np.repeat(np.abs(v).max(-1), g, axis=1).T[None]).max(-1)
    weight = np.log(2) * ((2.0 ** -22 + hd * 2.0 ** -24) * s + 2.0 ** -23 * (2 * s + 2))
    return out, (2 * weight + 2.0 ** -20 + 2 * n * 2.0 ** -24) * mass + 2 * n * 2.0 ** -24 * largest[..., None]


# ---- 4-bit projections ------------------------------------------------------------------

def pack_q4(codes):
    out_f, in_f = codes.shape
    c = codes.astype(np.uint32).reshape(out_f, in_f // 8, 8)
    return np.bitwise_or.reduce(c << (4 * np.arange(8, dtype=np.uint32)), axis=-1).astype(np.uint32)


def unpack_q4(packed, in_f, out_f, group, zeros):
    """(codes, scales, zero points or None) of a packed weight's bytes, and whether its padding (to
    16 features, 128 of the contraction) is zeros."""
    nt, nb, ng = -(-out_f // 16), -(-in_f // 128), 128 // group
    b = np.frombuffer(packed, np.uint8)
    planes = np.split(b, np.cumsum([nt * nb * 1024, nt * nb * 16 * ng * 2]))
    w = planes[0].view(np.uint32).reshape(nt, nb, 4, 16, 4)  # tile, block, g, n, j
    at = [16 * (i % 2) + 4 * (i // 2) for i in range(8)]
    c = np.stack([(w >> np.uint32(a)) & 15 for a in at], -1)  # tile, block, g, n, j, k
    codes = c.transpose(0, 3, 1, 4, 2, 5).reshape(nt * 16, nb * 128)
    s = planes[1].view(np.float16).reshape(nt, nb, 16, ng).transpose(0, 2, 1, 3).reshape(nt * 16, nb * ng)
    ngr = in_f // group
    padding = s[out_f:].any() or s[:, ngr:].any() or codes[out_f:].any() or codes[:, in_f:].any()
    z = None
    if zeros:
        z = planes[2].reshape(nt, nb, 16, ng).transpose(0, 2, 1, 3).reshape(nt * 16, nb * ng)[:out_f, :ngr]
    assert planes[2].size == (nt * nb * 16 * ng if zeros else 0)
    return codes[:out_f, :in_f].astype(np.int64), s[:out_f, :ngr], z, not padding


def linear_q4_bound(a, codes, scales, zeros, group):
    """(a . W^T, bound on its error) in 64 bits: a keeps 22 bits, a group's products are summed in
    f32 and scaled, and the groups' sums added in f32 (the waves of a workgroup adding eight more)."""
    a = np.asarray(a, np.float64)
    z = np.repeat(np.full(scales.shape, 8.0) if zeros is None else zeros.astype(np.float64), group, 1)
    w = (codes.astype(np.float64) - z) * np.repeat(scales.astype(np.float64), group, 1)
    adds = group + scales.shape[1] + 16
    return a @ w.T, (2.0 ** -22 + adds * 2.0 ** -24) * (np.abs(a) @ np.abs(w).T) + 1e-37


# ---- sampling ---------------------------------------------------------------------------

def sample_f64(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row."""
    x = np.asarray(logits, np.float64)
    ok = ~np.isnan(x)
    if not ok.any() or x[ok].max() == -np.inf:
        return 0
    top = x[ok].max()
    greedy = not temperature > 0 or min_p > 1
    t = float(temperature) if temperature > 0 else 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))
    w[~ok] = 0
    ranks = [i for i in np.lexsort((np.arange(len(x)), -np.where(ok, x, -np.inf))) if ok[i]]
    if greedy:
        return int(ranks[0])
    if 0 < top_k < len(x):
        ranks = ranks[:int(top_k)]
    ranks = np.array(ranks)
    if top_p < 1:
        sums = np.cumsum(w[ranks])
        before = np.concatenate(([0.0], sums[:-1]))
        keep = before < float(top_p) * sums[-1]
        keep[0] = True
        ranks = ranks[keep]
    if min_p > 0:
        ranks = ranks[w[ranks] >= float(min_p)]
    ranks = np.sort(ranks)
    ranks = ranks[w[ranks] > 0]
    cdf = np.cumsum(w[ranks])
    if u >= 1:
        return int(ranks[-1])
    at = float(u) * cdf[-1] if u > 0 else 0.0
    return int(ranks[min(np.searchsorted(cdf, at, "right"), len(ranks) - 1)])
