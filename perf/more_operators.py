"""The operators that verify a tree of drafted tokens, as cases that can be timed and compared.

A draft proposes several continuations at once, as a tree: node 0 is the last token that is
certain, every other node names its parent. One pass over the cache then answers for all nodes.
A case is one call of such a program:

- ``attend``: attention of the nodes over a cache that holds their rows: each sees the cached
  keys and its own ancestors, within the layer's window;
- ``rows``: RMSNorm and rotation of q and k for each head, v stored beside k, every node at the
  position of its depth;
- ``accept``: the tree's depths and ancestor masks from its parents, and the branch that the
  model's own tokens follow;
- ``compact``: the accepted branch's rows moved together, in every layer of the cache;
- ``fork``: the first rows of every layer copied into another cache.

With ``own`` false the operators run in their plain form, elementary torch operations in 32 bits;
with ``own`` true, as the library's calls. The shapes are this repository's three model shapes, and
generic ones with 64 and 96 dims a head.
"""
import math
import random

import torch

own = False

SHAPES = {
    # h query heads, hkv KV heads, head dim, scale
    "qwen": (16, 8, 128, 128 ** -0.5),
    "mistral": (32, 8, 128, 128 ** -0.5),
    "gemma": (16, 8, 256, 1.0),
    "narrow": (14, 2, 64, 64 ** -0.5),
    "odd": (6, 2, 96, 96 ** -0.5),
}
EPS = 1e-6
VOCAB = 151936


# ------------------------------------------------------------------------------ the cases

def _attend(shape, nodes, pos, cache, window=0):
    return dict(kind="attend", shape=shape, nodes=nodes, pos=pos, cache=cache, window=window)


def _rows(shape, nodes, pos, cache, norms):
    return dict(kind="rows", shape=shape, nodes=nodes, pos=pos, cache=cache, norms=norms)


def _move(kind, shape, layers, rows, pos, cache):
    return dict(kind=kind, shape=shape, layers=layers, rows=rows, pos=pos, cache=cache)


def listed():
    return [
        # A short chat's first drafts: latency counts.
        dict(name="attend, qwen 8 nodes at 100, f32", **_attend("qwen", 8, 100, "f32")),
        # An ordinary tree behind a long answer, in 8-bit codes.
        dict(name="attend, mistral 21 nodes at 8191, i8", **_attend("mistral", 21, 8191, "i8")),
        # A local layer of a model with wide heads.
        dict(name="attend, gemma 30 nodes at 6001, e4m3", **_attend("gemma", 30, 6001, "e4m3", 1024)),
        # A wide tree at the longest context of the 7B shape.
        dict(name="attend, mistral 64 nodes at 32000, f16", **_attend("mistral", 64, 32000, "f16")),
        # The rows of an ordinary tree into the small model's cache.
        dict(name="rows, qwen 16 nodes, f32", **_rows("qwen", 16, 1000, "f32", True)),
        # The widest tree, without norms.
        dict(name="rows, mistral 256 nodes, f16", **_rows("mistral", 256, 4000, "f16", False)),
        # An ordinary tree's plan and walk.
        dict(name="accept, 21 nodes", kind="accept", nodes=21),
        # The widest one's.
        dict(name="accept, 256 nodes", kind="accept", nodes=256),
        # Five accepted tokens of 21 in every layer of the small model.
        dict(name="compact, qwen 28 layers, 5 of 21, f32", **_move("compact", "qwen", 28, 21, 1000, "f32")),
        # The same in the 7B shape's half cache, with a wide tree.
        dict(name="compact, mistral 32 layers, 64, f16", **_move("compact", "mistral", 32, 64, 1900, "f16")),
        # A short prompt's cache continued twice.
        dict(name="fork, qwen 28 layers, 333 rows, f32", **_move("fork", "qwen", 28, 333, 0, "f32")),
        # A long one: the largest case.
        dict(name="fork, mistral 32 layers, 8000 rows, f16", **_move("fork", "mistral", 32, 8000, 0, "f16")),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(("attend", "attend", "attend", "attend", "rows", "accept", "compact", "fork"))
    shape = rng.choice(sorted(SHAPES))
    if what == "accept":
        return dict(kind="accept", nodes=_spread(rng, 1, 256))
    if what == "attend":
        nodes = _spread(rng, 1, 128)
        most = min(32000, 2048000 // nodes)
        pos = rng.choice((0, _spread(rng, 1, most), _spread(rng, 1, most)))
        window = rng.choice((0, 0, _spread(rng, 3, 4000)))
        return _attend(shape, nodes, pos, rng.choice(("f32", "f16", "e4m3", "i8")), window)
    if what == "rows":
        return _rows(shape, _spread(rng, 1, 256), _spread(rng, 1, 8000), rng.choice(("f32", "f16")),
                     rng.random() < 0.5)
    layers = rng.randint(1, 40)
    if what == "compact":
        return _move("compact", shape, layers, _spread(rng, 2, 128), _spread(rng, 1, 1900),
                     rng.choice(("f32", "f16")))
    return _move("fork", shape, layers, _spread(rng, 1, 3000), 0, rng.choice(("f32", "f16")))


# ---------------------------------------------------------------------------- the inputs

BLOCK = 64  # tokens that share a scale in a cache of 8-bit codes
DTYPES = {"f32": torch.float32, "f16": torch.float16, "e4m3": torch.uint8, "i8": torch.int8}


def _tree(nodes, seed):
    """Parents of a drafted tree: a few wide levels, then long branches; node 0 is the root."""
    rng = random.Random(seed)
    width = rng.randint(2, 12)
    return [-1] + [max(0, i - rng.randint(1, width)) for i in range(1, nodes)]


def _branch(rows, seed):
    """An accepted branch of a tree of `rows` nodes: its first nodes were drafted first, the rest lie
    behind, as the rows of a branch that was not the likeliest do."""
    rng = random.Random(seed + 1)
    count = min(rows, max(1, min(rows // 4, 8)))
    first = rng.randint(1, count)
    rest = sorted(rng.sample(range(count, rows), min(count - first, rows - count)))
    return list(range(first)) + rest


def _cached(g, n, hkv, hd, k):
    """n rows of K or V: channels of unlike size (K's outliers) and tokens of unlike size."""
    x = torch.randn(n, hkv, hd, generator=g, device="cuda")
    if k:
        x *= torch.exp(0.5 * torch.randn(1, hkv, hd, generator=g, device="cuda"))
    return x * torch.exp(0.3 * torch.randn(n, 1, 1, generator=g, device="cuda"))


def _as_i8(x, block):
    """Codes and exponents of rows x: a block's exponent is the least E with |x| <= 127 * 2^E."""
    n, hkv, hd = x.shape
    nb = -(-n // block)
    pad = torch.zeros(nb * block, hkv, hd, device=x.device)
    pad[:n] = x
    top = pad.view(nb, block, hkv, hd).abs().amax((1, 3))
    e = torch.ceil(torch.log2(top.double() / 127)).clamp(min=-126)
    codes = torch.round(x.double() * torch.exp2(-e).repeat_interleave(block, 0)[:n, :, None]).clamp(-127, 127)
    return codes.to(torch.int8), (e + 127).to(torch.uint8)


def _inputs(case, seed):
    """The case's inputs as torch tensors, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    if kind == "accept":
        n = case["nodes"]
        parents = _tree(n, seed)
        rng = random.Random(seed + 2)
        tokens = [rng.randrange(VOCAB) for _ in range(n)]
        for i in range(2, n, 7):  # (a token drafted twice behind one parent)
            if parents[i] == parents[i - 1]:
                tokens[i] = tokens[i - 1]
        sampled = [rng.randrange(VOCAB) for _ in range(n)]
        node = rng.randrange(n)
        while node > 0 and parents[node] >= 0:
            sampled[parents[node]] = tokens[node]
            node = parents[node]
        return dict(parents=ints(parents), tokens=ints(tokens), sampled=ints(sampled))
    h, hkv, hd, _ = SHAPES[case["shape"]]
    if kind == "attend":
        n, pos = case["nodes"], case["pos"]
        d = dict(q=normal(n, h, hd), parents=_tree(n, seed))
        seen = [[False] * n for _ in range(n)]
        for i, p in enumerate(d["parents"]):
            if p >= 0:
                seen[i] = list(seen[p])
            seen[i][i] = True
        words = [[sum(1 << b for b in range(32) if 32 * w + b < n and row[32 * w + b])
                  for w in range(-(-n // 32))] for row in seen]
        d["masks"] = ints([[w - (1 << 32) if w >> 31 else w for w in row] for row in words])
        d["depths"] = ints([sum(row) - 1 for row in seen])
        for name in "kv":
            x = _cached(g, pos + n, hkv, hd, name == "k")
            if case["cache"] == "i8":
                d[name], d[name + "s"] = _as_i8(x, BLOCK)
            elif case["cache"] == "e4m3":
                d[name] = x.to(torch.float8_e4m3fn).view(torch.uint8)
            else:
                d[name] = x.to(DTYPES[case["cache"]])
        return d
    if kind == "rows":
        n = case["nodes"]
        depth = []
        for p in _tree(n, seed):
            depth.append(depth[p] + 1 if p >= 0 else 0)
        at = torch.arange(case["pos"] + n, device="cuda", dtype=torch.float64)
        angle = at[:, None] * 1e6 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))
        d = dict(q=normal(n, h, hd), k=normal(n, hkv, hd), v=normal(n, hkv, hd), depths=ints(depth),
                 cos=torch.cos(angle).float(), sin=torch.sin(angle).float())
        if case["norms"]:
            d["q_norm"], d["k_norm"] = 1 + 0.2 * normal(hd), 1 + 0.2 * normal(hd)
        for name in ("kc", "vc"):
            d[name] = torch.zeros(case["pos"] + n, hkv, hd, device="cuda", dtype=DTYPES[case["cache"]])
        return d
    rows = case["pos"] + case["rows"]
    layers = [normal(rows, hkv, hd).to(DTYPES[case["cache"]]) for _ in range(2 * case["layers"])]
    d = dict(layers=layers)
    if kind == "compact":
        path = _branch(case["rows"], seed)
        d["count"] = ints([len(path)])
        d["path"] = ints(path + [-1] * (case["rows"] - len(path)))
        d["kept"] = len(path)
    else:
        d["into"] = [torch.zeros_like(x) for x in layers]
    return d


# -------------------------------------------------------------------------- the plain forms

def _values(d, name, cache):
    if cache == "i8":
        scale = torch.exp2(d[name + "s"].float() - 127).repeat_interleave(BLOCK, 0)[:len(d[name])]
        return d[name].float() * scale[..., None]
    if cache == "e4m3":
        return d[name].view(torch.float8_e4m3fn).float()
    return d[name].float()


def _seen(case, d):
    """[nodes, pos + nodes]: which keys each node sees."""
    n, pos, w = case["nodes"], case["pos"], case["window"]
    bit = torch.arange(n, device="cuda")
    drafted = (d["masks"][:, bit // 32] >> (bit % 32)) & 1 == 1
    key = torch.arange(pos, device="cuda")[None]
    at = pos + d["depths"].long()
    cached = torch.ones(n, pos, dtype=torch.bool, device="cuda")
    if w:
        cached = key > at[:, None] - w
        drafted = drafted & (at[None] > at[:, None] - w)
    return torch.cat((cached, drafted), 1)


def _plain_attend(case, d):
    h, hkv, hd, scale = SHAPES[case["shape"]]
    n, g = case["nodes"], h // hkv
    k, v = _values(d, "k", case["cache"]), _values(d, "v", case["cache"])
    hidden = ~_seen(case, d)
    out = torch.empty_like(d["q"])
    for j in range(hkv):
        q = d["q"][:, j * g:(j + 1) * g].transpose(0, 1).reshape(g * n, hd)
        s = (q @ k[:, j].t().contiguous()) * scale
        s = s.view(g, n, -1).masked_fill(hidden, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = (p.view(g * n, -1) @ v[:, j].contiguous()).view(g, n, hd) / p.sum(-1, keepdim=True)
        out[:, j * g:(j + 1) * g] = o.transpose(0, 1)
    return {"out": out}


def _plain_rows(case, d):
    n, pos = case["nodes"], case["pos"]
    at = pos + d["depths"].long()
    c, s = d["cos"][at][:, None], d["sin"][at][:, None]

    def rotated(x, gain):
        if gain is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    d["kc"][pos:pos + n] = rotated(d["k"], d.get("k_norm")).to(d["kc"].dtype)
    d["vc"][pos:pos + n] = d["v"].to(d["vc"].dtype)
    return {"q": rotated(d["q"], d.get("q_norm")), "k": d["kc"][pos:pos + n], "v": d["vc"][pos:pos + n]}


def _plain_accept(d):
    parents, tokens, sampled = d["parents"].long(), d["tokens"], d["sampled"]
    n = len(parents)
    node = torch.arange(n, device="cuda")
    seen = torch.eye(n, dtype=torch.bool, device="cuda")
    up = torch.where(parents < 0, node, parents)
    for _ in range(max(1, (n - 1).bit_length())):  # ancestors within 2, 4, 8, .. steps
        seen = seen | seen[up]
        up = up[up]
    depths = seen.int().sum(1) - 1
    words = -(-n // 32)
    bits = torch.zeros(n, 32 * words, dtype=torch.int64, device="cuda")
    bits[:, :n] = seen.long()
    masks = (bits.view(n, words, 32) << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    # A node is taken if it is the first of its parent's children that has the model's token.
    fits = (node > 0) & (parents >= 0) & (tokens == sampled[parents.clamp(min=0)])
    earlier = fits[None] & (parents[None] == parents[:, None]) & (node[None] < node[:, None])
    taken = (fits & ~earlier.any(1)) | (node == 0)
    accepted = (taken[None] | ~seen).all(1) & seen[:, 0]
    slot = torch.where(accepted, depths.long(), torch.full_like(depths, n).long())
    path = torch.full((n + 1,), -1, dtype=torch.int32, device="cuda")
    path.scatter_(0, slot, node.int())
    emitted = torch.full((n + 1,), -1, dtype=torch.int32, device="cuda")
    emitted.scatter_(0, slot, sampled)
    return {"depths": depths.int(), "masks": masks, "path": path[:n], "emitted": emitted[:n],
            "count": accepted.sum().int()[None]}


def _plain_move(case, d):
    pos, n = case["pos"], case["rows"]
    if case["kind"] == "fork":
        for x, y in zip(d["layers"], d["into"]):
            y[:n] = x[:n]
        return d["into"]
    j = torch.arange(n, device="cuda")
    src = pos + torch.where(j < d["count"], d["path"], j.int()).long()  # (the others stay)
    for x in d["layers"]:
        x[pos:pos + n] = x[src]
    return [x[pos:pos + n] for x in d["layers"]]


def _plain(case, d):
    kind = case["kind"]
    if kind == "attend":
        return _plain_attend(case, d)
    if kind == "rows":
        return _plain_rows(case, d)
    if kind == "accept":
        return _plain_accept(d)
    return _plain_move(case, d)


# ------------------------------------------------------------------- the library's tensors

class _Memory:
    """A library tensor's memory as torch reads it. It does not own it: the state does."""

    def __init__(self, t):
        typestr = {"F32": "<f4", "F16": "<f2", "U32": "<i4", "I32": "<i4", "I8": "|i1", "U8": "|u1",
                   "F8E4M3": "|u1"}[t.dtype.name]
        self.__cuda_array_interface__ = dict(data=(t.data_ptr, False), shape=t.shape, strides=None,
                                             typestr=typestr, version=2)


def _view(t):
    return torch.as_tensor(_Memory(t), device="cuda")


_devices = []


def _device():
    import eyebrowse_amd as eb
    if not _devices:
        _devices.append(eb.Device.new(0))
    return _devices[0]


def _tensor(x, dtype):
    """x (a torch tensor) in a library tensor."""
    import eyebrowse_amd as eb
    t = eb.Tensor.empty(_device(), tuple(x.shape), dtype)
    _view(t).copy_(x)
    return t


def _library_state(case, d):
    """The case's inputs in the library's tensors, and its outputs' tensors."""
    import eyebrowse_amd as eb
    dev = _device()
    dev.synchronize()  # pooled buffers may still be read by an earlier call
    T = eb.DType
    types = {"f32": T.F32, "f16": T.F16, "e4m3": T.F8E4M3, "i8": T.I8}
    kind = case["kind"]
    s = {"case": case, "dev": dev}
    if kind == "accept":
        n = case["nodes"]
        s.update(parents=_tensor(d["parents"], T.I32), tokens=_tensor(d["tokens"], T.U32),
                 sampled=_tensor(d["sampled"], T.U32), masks=eb.Tensor.empty(dev, (n, -(-n // 32)), T.U32),
                 depths=eb.Tensor.empty(dev, (n,), T.U32), path=eb.Tensor.empty(dev, (n,), T.U32),
                 emitted=eb.Tensor.empty(dev, (n,), T.U32), count=eb.Tensor.empty(dev, (1,), T.U32))
        s["result"] = {name: _view(s[name]) for name in ("depths", "masks", "path", "emitted", "count")}
        torch.cuda.synchronize()
        return s
    h, hkv, hd, _ = SHAPES[case["shape"]]
    if kind == "attend":
        s.update(q=_tensor(d["q"], T.F32), masks=_tensor(d["masks"], T.U32), depths=_tensor(d["depths"], T.U32),
                 out=eb.Tensor.empty(dev, tuple(d["q"].shape)))
        seq = case["pos"] + case["nodes"]
        if case["cache"] == "i8":
            kv = eb.KvCache.new_i8(dev, 1, seq, hkv, hd, BLOCK)
            for name, t in (("ks", kv.k_scale[0]), ("vs", kv.v_scale[0])):
                _view(t).copy_(d[name])
        else:
            kv = eb.KvCache.new(dev, 1, seq, hkv, hd, types[case["cache"]])
        _view(kv.k[0]).copy_(d["k"])
        _view(kv.v[0]).copy_(d["v"])
        s.update(kv=kv, result={"out": _view(s["out"])})
    elif kind == "rows":
        n, pos = case["nodes"], case["pos"]
        s["kv"] = kv = eb.KvCache.new(dev, 1, pos + n, hkv, hd, types[case["cache"]])
        s.update((name, _tensor(d[name], T.U32 if name == "depths" else T.F32))
                 for name in d if name not in ("kc", "vc"))
        s["out"] = eb.Tensor.empty(dev, (n, h, hd))
        s["result"] = {"q": _view(s["out"]), "k": _view(kv.k[0])[pos:pos + n], "v": _view(kv.v[0])[pos:pos + n]}
    else:
        pos, n = case["pos"], case["rows"]

        def cache(layers):
            kv = eb.KvCache.new(dev, case["layers"], pos + n, hkv, hd, types[case["cache"]])
            for i, x in enumerate(layers):
                _view((kv.v if i % 2 else kv.k)[i // 2]).copy_(x)
            return kv, [_view((kv.v if i % 2 else kv.k)[i // 2]) for i in range(len(layers))]

        s["kv"], views = cache(d["layers"])
        if kind == "fork":
            s["into"], s["result"] = cache(d["into"])
        else:
            s.update(path=_tensor(d["path"], T.U32), count=_tensor(d["count"], T.U32))
            s["result"] = [x[pos:pos + n] for x in views]
    torch.cuda.synchronize()
    return s


def _library(s):
    import eyebrowse_amd as eb
    case = s["case"]
    kind = case["kind"]
    rec = eb.Recorder(s["dev"])
    if kind == "accept":
        eb.tree_plan(rec, s["parents"], s["masks"], s["depths"], case["nodes"])
        eb.tree_accept(rec, s["tokens"], s["parents"], s["sampled"], s["path"], s["emitted"], s["count"],
                       case["nodes"])
    elif kind == "fork":
        eb.kv_fork(rec, s["into"], s["kv"], case["rows"])
    elif kind == "compact":
        eb.kv_compact(rec, s["kv"], s["path"], s["count"], case["rows"], case["pos"])
    else:
        h, hkv, hd, scale = SHAPES[case["shape"]]
        n, pos, kv = case["nodes"], case["pos"], s["kv"]
        if kind == "rows":
            eb.attn_prologue_tree(rec, s["q"], s["k"], s["v"], s["depths"], s["out"], kv.k[0], kv.v[0], n, h, hkv,
                                  hd, pos, pos + n, s.get("q_norm"), s.get("k_norm"), None, EPS, s["cos"], s["sin"])
        elif case["cache"] == "i8":
            eb.attn_tree_i8(rec, s["q"], kv, 0, s["masks"], s["depths"], s["out"], h, pos, n, scale, case["window"])
        else:
            eb.attn_tree(rec, s["q"], kv.k[0], kv.v[0], s["masks"], s["depths"], s["out"], h, hkv, pos, n, hd,
                         pos + n, scale, case["window"])
    rec.submit()
    return s["result"]


# ------------------------------------------------------------------------ prepare and run

def prepare(case, seed):
    d = _inputs(case, seed)
    return _library_state(case, d) if own else {"case": case, "inputs": d}


def run(s):
    return _library(s) if own else _plain(s["case"], s["inputs"])


# -------------------------------------------------------------------- what a pass has to do

def work(case):
    kind = case["kind"]
    if kind == "accept":
        n = case["nodes"]
        # parents twice, tokens, sampled; depths, masks, path, emitted, count
        return {"bytes": 4 * (4 * n + 3 * n + n * -(-n // 32) + 1), "flops": 0}
    h, hkv, hd, _ = SHAPES[case["shape"]]
    size = torch.empty(0, dtype=DTYPES[case["cache"]]).element_size()
    row = 2 * hkv * hd * size
    if kind == "attend":
        n, pos = case["nodes"], case["pos"]
        keys = min(pos, case["window"] - 1) if case["window"] else pos
        scales = 2 * hkv * -(-keys // BLOCK) if case["cache"] == "i8" else 0
        # Of the drafted keys each node sees itself and some ancestors: counted as half of them.
        return {"bytes": row * (keys + n) + scales + 8 * n * h * hd, "flops": 4 * h * hd * n * (keys + (n + 1) // 2)}
    if kind == "rows":
        n = case["nodes"]
        return {"bytes": 4 * n * (2 * h + 2 * hkv) * hd + n * row + 4 * n * hd, "flops": 8 * n * (h + hkv) * hd}
    if kind == "fork":
        return {"bytes": 2 * case["layers"] * case["rows"] * row, "flops": 0}
    moved = max(1, min(case["rows"] // 4, 8))
    return {"bytes": 2 * case["layers"] * moved * row + 4 * moved + 4, "flops": 0}


# ------------------------------------------------------------------------- 64-bit results

def _exact_attend(case, d):
    h, hkv, hd, scale = SHAPES[case["shape"]]
    n, pos, w = case["nodes"], case["pos"], case["window"]
    parents = d["parents"]
    value = {}
    for name in "kv":
        x = d[name]
        if case["cache"] == "e4m3":
            x = x.view(torch.float8_e4m3fn)
        x = x.double()
        if case["cache"] == "i8":
            for b in range(d[name + "s"].shape[0]):
                x[b * BLOCK:(b + 1) * BLOCK] *= (2.0 ** (d[name + "s"][b].double() - 127))[:, None]
        value[name] = x
    out = torch.empty(n, h, hd, dtype=torch.float64, device="cuda")
    for i in range(n):
        line = [i]
        while parents[line[-1]] >= 0:
            line.append(parents[line[-1]])
        line.reverse()  # (line[t] is drafted at position pos + t)
        at = pos + len(line) - 1
        lo = max(0, at - w + 1) if w else 0
        rows = torch.tensor(list(range(lo, pos)) + [pos + j for t, j in enumerate(line) if pos + t >= lo],
                            device="cuda")
        for j in range(hkv):
            kk, vv = value["k"][rows, j], value["v"][rows, j]
            g = h // hkv
            s = (d["q"][i, j * g:(j + 1) * g].double() @ kk.t().contiguous()) * scale
            out[i, j * g:(j + 1) * g] = torch.softmax(s, 1) @ vv
    return {"out": out}


def _exact_rows(case, d):
    n, pos = case["nodes"], case["pos"]
    half = d["q"].shape[-1] // 2

    def turned(x, gain):
        x = x.double()
        if gain is not None:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / (2 * half) + EPS) * gain.double()
        y = torch.empty_like(x)
        for i, depth in enumerate(d["depths"].tolist()):
            c, s = d["cos"][pos + depth].double(), d["sin"][pos + depth].double()
            y[i, :, :half] = x[i, :, :half] * c - x[i, :, half:] * s
            y[i, :, half:] = x[i, :, half:] * c + x[i, :, :half] * s
        return y

    return {"q": turned(d["q"], d.get("q_norm")), "k": turned(d["k"], d.get("k_norm")), "v": d["v"].double()}


def _exact_accept(d):
    parents, tokens, sampled = (d[name].tolist() for name in ("parents", "tokens", "sampled"))
    n = len(parents)
    words = -(-n // 32)
    depths, masks = [], []
    for i in range(n):
        line, mask = i, 0
        depth = -1
        while line >= 0:
            mask |= 1 << line
            depth += 1
            line = parents[line]
        depths.append(depth)
        parts = [(mask >> (32 * w)) & 0xFFFFFFFF for w in range(words)]
        masks.append([p - (1 << 32) if p >> 31 else p for p in parts])
    path = [0]
    while True:
        fit = [i for i in range(1, n) if parents[i] == path[-1] and tokens[i] == sampled[path[-1]]]
        if not fit:
            break
        path.append(fit[0])
    rest = [-1] * (n - len(path))
    out = {"depths": depths, "masks": masks, "path": path + rest, "emitted": [sampled[i] for i in path] + rest,
           "count": [len(path)]}
    return {name: torch.tensor(x, dtype=torch.int32) for name, x in out.items()}


def exact(case, seed):
    d = _inputs(case, seed)
    kind = case["kind"]
    if kind == "attend":
        return _exact_attend(case, d)
    if kind == "rows":
        return _exact_rows(case, d)
    if kind == "accept":
        return _exact_accept(d)
    if kind == "fork":
        return [torch.cat((x[:case["rows"]], y[case["rows"]:])) for x, y in zip(d["layers"], d["into"])]
    pos, out = case["pos"], []
    for x in d["layers"]:
        y = x[pos:pos + case["rows"]].clone()
        for j, i in enumerate(d["path"].tolist()[:d["kept"]]):
            y[j] = x[pos + i]
        out.append(y)
    return out
