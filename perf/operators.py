"""The operators of a quantised model's token, as cases that can be timed and compared.

A case is one call of a serving program:

- ``linear``: a projection (or the LM head) with 4-bit weights and group scales;
- ``write``: a prompt's or a chunk's K and V rows into a cache of 8-bit codes with one
  power-of-two scale for each block of tokens and head, and the rows it changed read back as
  the values they stand for;
- ``step``: one token against such a cache: its K and V appended, its attention, and the
  token's block read back;
- ``chunk``: causal attention of a prompt, or of a prompt's next rows, over such a cache;
- ``sample``: the next tokens from their logits and given random numbers.

With ``own`` false the operators run in their plain form, elementary torch operations in 32 bits
(64 where a token's choice lies next to a border); with ``own`` true, as the library's calls.
The shapes are this repository's three model shapes, and generic ones with 64 and 96 dims a head.
"""
import math

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


# ------------------------------------------------------------------------------ the cases

def _linear(rows, in_f, out_f, group, zeros):
    return dict(kind="linear", rows=rows, in_f=in_f, out_f=out_f, group=group, zeros=zeros)


def _cache(kind, shape, rows, pos, block=64, window=0):
    return dict(kind=kind, shape=shape, rows=rows, pos=pos, block=block, window=window,
                max_seq=max(256, 1 << (pos + rows - 1).bit_length()))


def _sample(rows, vocab, top_k, top_p, min_p):
    return dict(kind="sample", rows=rows, vocab=vocab, top_k=top_k, top_p=top_p, min_p=min_p)


def listed():
    return [
        # A token's query projection in the small model: latency counts.
        dict(name="linear, token 1024 to 2048", **_linear(1, 1024, 2048, 128, False)),
        # The LM head of every token, with fine groups and zero points.
        dict(name="linear, head 1024 to 151936", **_linear(1, 1024, 151936, 32, True)),
        # Three answers generated together, through a wide projection of odd size.
        dict(name="linear, 3 rows 4096 to 14335", **_linear(3, 4096, 14335, 64, True)),
        # An ordinary prompt through the 7B shape's output projection.
        dict(name="linear, prompt 1000, 4096 to 4096", **_linear(1000, 4096, 4096, 128, False)),
        # A long prompt enters the cache.
        dict(name="write, mistral prompt 4096", **_cache("write", "mistral", 4096, 0)),
        # The next turn's rows start inside a block whose tokens keep their values.
        dict(name="write, gemma 37 rows at 1000", **_cache("write", "gemma", 37, 1000, 32)),
        # A chat's first answer tokens.
        dict(name="step, qwen token 100", **_cache("step", "qwen", 1, 100)),
        # The longest context of the 7B shape.
        dict(name="step, mistral token 32767", **_cache("step", "mistral", 1, 32767)),
        # A long prompt's next chunk.
        dict(name="chunk, mistral 256 rows at 8192", **_cache("chunk", "mistral", 256, 8192)),
        # A whole long prompt: the largest case.
        dict(name="chunk, mistral prompt 4096", **_cache("chunk", "mistral", 4096, 0)),
        # One answer's next token from the small model's vocabulary.
        dict(name="sample, 1 row of 151936", **_sample(1, 151936, 50, 0.9, 0.0)),
        # A batch's next tokens, with the nucleus alone and a floor below the best token.
        dict(name="sample, 64 rows of 32768", **_sample(64, 32768, 0, 0.95, 0.02)),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(("linear", "linear", "write", "step", "step", "chunk", "chunk", "sample"))
    if what == "linear":
        group = rng.choice((32, 64, 128))
        in_f = 128 * rng.randint(4, 48)
        rows = rng.choice((1, 1, _spread(rng, 2, 1200)))
        most = min(160000, 160000000 // in_f, 17000000000 // (rows * in_f))
        return _linear(rows, in_f, _spread(rng, 64, most), group, rng.random() < 0.5)
    if what == "sample":
        rows = _spread(rng, 1, 64)
        vocab = _spread(rng, 100, min(200000, 2097152 // rows))
        return _sample(rows, vocab, rng.choice((0, 1, _spread(rng, 2, 400))),
                       rng.choice((1.0, round(rng.uniform(0.3, 0.99), 2))),
                       rng.choice((0.0, round(rng.uniform(0.001, 0.2), 3))))
    shape = rng.choice(sorted(SHAPES))
    block = rng.choice((16, 32, 64, 128, 256))
    window = rng.choice((0, 0, _spread(rng, 100, 4000)))
    if what == "write":
        return _cache("write", shape, _spread(rng, 1, 2000), rng.choice((0, _spread(rng, 1, 2000))), block)
    if what == "step":
        return _cache("step", shape, 1, _spread(rng, 1, 32000), block, window)
    return _cache("chunk", shape, _spread(rng, 2, 1500), rng.choice((0, _spread(rng, 1, 7000))), block, window)


# ---------------------------------------------------------------------------- the inputs

def _rows(g, n, hkv, hd, outliers):
    """n rows of K or V: channels of unlike size (K's outliers) and tokens of unlike size."""
    x = torch.randn(n, hkv, hd, generator=g, device="cuda")
    if outliers:
        x *= torch.exp(0.5 * torch.randn(1, hkv, hd, generator=g, device="cuda"))
    return x * torch.exp(0.3 * torch.randn(n, 1, 1, generator=g, device="cuda"))


def _quantise(w, group, zeros):
    """Round-to-nearest 4-bit codes of w [out_f, in_f] with a half scale (and a whole zero point)
    for each group of a row."""
    out_f, in_f = w.shape
    x = w.view(out_f, in_f // group, group)
    if zeros:
        lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).half()
        z = torch.round(-lo / s.float()).clamp(0, 15)
    else:
        s = (x.abs().amax(-1) / 7).half()
        z = torch.full_like(s, 8, dtype=torch.float32)
    c = torch.round(x / s.float()[..., None] + z[..., None]).clamp(0, 15).to(torch.int32)
    c = c.view(out_f, in_f // 8, 8)
    words = torch.zeros(out_f, in_f // 8, dtype=torch.int32, device=w.device)
    for i in range(8):
        words |= c[..., i] << (4 * i)
    return words, s, z.to(torch.uint8) if zeros else None


def _inputs(case, seed):
    """The case's inputs as torch tensors, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind == "linear":
        w = normal(case["out_f"], case["in_f"]) / math.sqrt(case["in_f"])
        words, scales, zeros = _quantise(w, case["group"], case["zeros"])
        return dict(a=normal(case["rows"], case["in_f"]), w=words, scales=scales, zeros=zeros)
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # A few likely tokens above a wide floor, as a language model's logits are.
        x = 2.0 * normal(rows, vocab)
        x[:, : max(1, vocab // 500)] += 6.0 + 2.0 * normal(rows, max(1, vocab // 500))
        x = torch.gather(x, 1, torch.argsort(normal(rows, vocab), 1))
        temperature = 0.6 + 0.8 * torch.rand(rows, generator=g, device="cuda")
        temperature[5::8] = 0.0  # (some rows ask for the best token)
        return dict(logits=x, temperature=temperature,
                    top_k=torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda"),
                    top_p=torch.full((rows,), case["top_p"], device="cuda"),
                    min_p=torch.full((rows,), case["min_p"], device="cuda"),
                    u=torch.rand(rows, generator=g, device="cuda"))
    h, hkv, hd, _ = SHAPES[case["shape"]]
    rows, pos, block, max_seq = case["rows"], case["pos"], case["block"], case["max_seq"]
    # The cache as `pos` earlier tokens left it (all rows of it for a chunk, whose own rows are
    # written before it attends); what lies behind them is stale.
    have = pos + rows if kind == "chunk" else pos
    d = {}
    for n in "kv":
        codes = torch.randint(-127, 128, (max_seq, hkv, hd), generator=g, device="cuda", dtype=torch.int8)
        exps = torch.randint(100, 140, (-(-max_seq // block), hkv), generator=g, device="cuda").to(torch.uint8)
        if have:
            _append(codes, exps, _rows(g, have, hkv, hd, n == "k"), 0, block)
        d[n + "c"], d[n + "s"] = codes, exps
    if kind != "chunk":
        d["k"], d["v"] = _rows(g, rows, hkv, hd, True), _rows(g, rows, hkv, hd, False)
    if kind != "write":
        d["q"] = normal(rows, h, hd) if kind == "chunk" else normal(h, hd)
    return d


# -------------------------------------------------------------------------- the plain forms

def _pow2(e):
    """2^e for whole e from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _append(codes, exps, x, pos, block):
    """Rows x [n, hkv, hd] at row pos.. of a block-scaled cache, in place: a block's exponent is
    the least E with every |x| <= 127 * 2^E, at least that of the rows before pos in its block,
    whose codes are rounded again where it grew."""
    n, hkv, hd = x.shape
    first = pos // block
    last = (pos + n - 1) // block
    start, lead = first * block, pos - first * block
    pad = torch.zeros((last + 1) * block - start, hkv, hd, device=x.device)
    pad[lead:lead + n] = x
    amax = pad.view(-1, block, hkv, hd).abs().amax((1, 3))
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 7 + (m * 128 > 127).int(), torch.full_like(e, -126)).clamp(min=-126)
    if lead:
        old = exps[first].int() - 127
        e[0] = torch.maximum(e[0], old)
        kept = codes[start:pos].float() * _pow2((old - e[0]).clamp(min=-126))[:, None]
        codes[start:pos] = torch.round(kept).to(torch.int8)
    per_row = e.repeat_interleave(block, 0)[lead:lead + n]
    codes[pos:pos + n] = torch.round(x * _pow2(-per_row)[..., None]).to(torch.int8)
    exps[first:last + 1] = (e + 127).to(torch.uint8)


def _values(codes, exps, lo, hi, block):
    """Rows lo..hi of a block-scaled cache as the values they stand for."""
    rows = torch.arange(lo, hi, device=codes.device) // block
    return codes[lo:hi].float() * _pow2(exps[rows].int() - 127)[..., None]


def _attend(q, k, v, pos, scale, window):
    """Rows of q [rows, h, hd] at pos.. over keys k, v [keys, hkv, hd]; key 0 is token 0."""
    rows, h, hd = q.shape
    hkv = k.shape[1]
    g = h // hkv
    lo = max(0, pos - window + 1) if window else 0
    at = torch.arange(pos, pos + rows, device=q.device)[:, None]
    key = torch.arange(lo, pos + rows, device=q.device)[None]
    seen = key <= at
    if window:
        seen = seen & (key > at - window)
    out = torch.empty_like(q)
    for j in range(hkv):
        qj = q[:, j * g:(j + 1) * g].transpose(0, 1).reshape(g * rows, hd)
        s = (qj @ k[lo:, j].t().contiguous()) * scale
        s = s.view(g, rows, -1).masked_fill(~seen, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = (p.view(g * rows, -1) @ v[lo:, j].contiguous()).view(g, rows, hd) / p.sum(-1, keepdim=True)
        out[:, j * g:(j + 1) * g] = o.transpose(0, 1)
    return out


def _unpack(words, scales, zeros):
    c = torch.stack([(words >> (4 * i)) & 15 for i in range(8)], -1).view(*scales.shape, -1)
    z = zeros.float()[..., None] if zeros is not None else 8.0
    return ((c.float() - z) * scales.float()[..., None]).view(words.shape[0], -1)


def _choose(d):
    """The sampled tokens. A token's weight is exp((x - max) / temperature); kept are the top_k
    largest, of those the fewest largest that hold top_p of their sum, of those the ones with at
    least min_p of the largest weight; the token is the first, in the vocabulary's order, at
    which the kept weights' sum exceeds u times their total. Equal logits rank by index."""
    x = d["logits"].double()
    rows, vocab = x.shape
    cold = d["temperature"] <= 0
    t = torch.where(cold, torch.ones_like(d["temperature"]), d["temperature"]).double()[:, None]
    w = torch.exp((x - x.amax(1, keepdim=True)) / t)
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    ws = torch.gather(w, 1, order)
    rank = torch.arange(vocab, device=x.device)[None]
    k = d["top_k"].long()[:, None]
    k = torch.where((k <= 0) | cold[:, None], torch.where(cold[:, None], 1, vocab), k)
    ws = torch.where(rank < k, ws, torch.zeros_like(ws))
    cum = torch.cumsum(ws, 1)
    p = d["top_p"].double()[:, None]
    keep = (rank < k) & ((p >= 1) | (rank == 0) | (cum - ws < p * cum[:, -1:]))
    keep &= ws >= d["min_p"].double()[:, None]
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    cdf = torch.cumsum(torch.where(kept, w, torch.zeros_like(w)), 1)
    over = cdf > d["u"].double()[:, None] * cdf[:, -1:]
    return torch.argmax(over.int(), 1).int()


def _plain(case, d):
    kind = case["kind"]
    if kind == "linear":
        return {"out": d["a"] @ _unpack(d["w"], d["scales"], d["zeros"]).t()}
    if kind == "sample":
        return {"token": _choose(d)}
    h, hkv, hd, scale = SHAPES[case["shape"]]
    rows, pos, block = case["rows"], case["pos"], case["block"]
    out = {}
    start = pos // block * block
    if kind != "chunk":
        for n in "kv":
            _append(d[n + "c"], d[n + "s"], d[n], pos, block)
            out[n] = _values(d[n + "c"], d[n + "s"], start, pos + rows, block)
    if kind != "write":
        k, v = (_values(d[n + "c"], d[n + "s"], 0, pos + rows, block) for n in "kv")
        q = d["q"].view(rows, h, hd)
        out["out"] = _attend(q, k, v, pos, scale, case["window"]).view(d["q"].shape)
    return out


# ------------------------------------------------------------------- the library's tensors

class _Memory:
    """A library tensor's memory as torch reads it. It does not own it: the state does."""

    def __init__(self, t):
        typestr = {"F32": "<f4", "F16": "<f2", "U32": "<i4", "I8": "|i1", "U8": "|u1"}[t.dtype.name]
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
    f32, u32 = eb.DType.F32, eb.DType.U32
    kind = case["kind"]
    s = {"case": case, "dev": dev}
    if kind == "linear":
        s["a"] = _tensor(d["a"], f32)
        s["proj"] = eb.LinearQ4(_tensor(d["w"], u32), _tensor(d["scales"], eb.DType.F16),
                                None if d["zeros"] is None else _tensor(d["zeros"], eb.DType.U8),
                                case["in_f"], case["out_f"], case["group"])
        s["out"] = eb.Tensor.empty(dev, (case["rows"], case["out_f"]))
        s["result"] = {"out": _view(s["out"])}
    elif kind == "sample":
        s.update((n, _tensor(d[n], u32 if n == "top_k" else f32)) for n in d)
        s["token"] = eb.Tensor.empty(dev, (case["rows"],), u32)
        s["result"] = {"token": _view(s["token"])}
    else:
        h, hkv, hd, _ = SHAPES[case["shape"]]
        rows, pos, block = case["rows"], case["pos"], case["block"]
        kv = eb.KvCache.new_i8(dev, 1, case["max_seq"], hkv, hd, block)
        for n, t in (("kc", kv.k[0]), ("ks", kv.k_scale[0]), ("vc", kv.v[0]), ("vs", kv.v_scale[0])):
            _view(t).copy_(d[n])
        s.update((n, _tensor(d[n], f32)) for n in "kvq" if n in d)
        s.update(kv=kv, result={})
        if kind != "chunk":
            changed = pos + rows - pos // block * block
            for n in "kv":
                s[n + "_out"] = eb.Tensor.empty(dev, (changed, hkv, hd))
                s["result"][n] = _view(s[n + "_out"])
        if kind != "write":
            s["out"] = eb.Tensor.empty(dev, tuple(d["q"].shape))
            s["result"]["out"] = _view(s["out"])
    torch.cuda.synchronize()
    return s


def _library(s):
    import eyebrowse_amd as eb
    case = s["case"]
    kind = case["kind"]
    rec = eb.Recorder(s["dev"])
    if kind == "linear":
        eb.linear_q4(rec, s["a"], s["proj"], s["out"], case["rows"])
    elif kind == "sample":
        eb.sample(rec, s["logits"], s["u"], s["token"], case["rows"], case["vocab"],
                  temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    else:
        h, hkv, hd, scale = SHAPES[case["shape"]]
        rows, pos, block, kv = case["rows"], case["pos"], case["block"], s["kv"]
        start = pos // block * block
        if kind == "write":
            eb.kv_write_i8(rec, kv, 0, s["k"], s["v"], rows, pos)
        elif kind == "step":
            eb.attn_decode_step_i8(rec, s["q"], s["k"], s["v"], kv, 0, s["out"], h, pos, scale, case["window"])
        else:
            eb.attn_prefill_chunk_i8(rec, s["q"], kv, 0, s["out"], h, pos, rows, scale, case["window"])
        if kind != "chunk":
            eb.kv_read_i8(rec, kv, 0, s["k_out"], s["v_out"], pos + rows - start, start)
    rec.submit()
    return s["result"]


# ------------------------------------------------------------------------ prepare and run

def prepare(case, seed):
    d = _inputs(case, seed)
    return _library_state(case, d) if own else {"case": case, "inputs": d}


def run(s):
    return _library(s) if own else _plain(s["case"], s["inputs"])


# -------------------------------------------------------------------- what a pass has to do

def _span(case):
    """(first key any row reads, visible query-key pairs) of an attention case."""
    rows, pos = case["rows"], case["pos"]
    w = case["window"] or pos + rows
    return max(0, pos - w + 1), sum(min(w, p + 1) for p in range(pos, pos + rows))


def work(case):
    kind = case["kind"]
    if kind == "linear":
        rows, in_f, out_f, group = case["rows"], case["in_f"], case["out_f"], case["group"]
        weights = out_f * in_f // 2 + out_f * in_f // group * (3 if case["zeros"] else 2)
        return {"bytes": weights + 4 * rows * (in_f + out_f), "flops": 2 * rows * in_f * out_f}
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": 4 * rows * vocab + 24 * rows, "flops": 4 * rows * vocab}
    h, hkv, hd, _ = SHAPES[case["shape"]]
    rows, pos, block = case["rows"], case["pos"], case["block"]
    lead = pos % block
    # New rows in 32 bits read and stored as codes; the changed rows given back in 32 bits.
    new = 2 * hkv * hd * (5 * rows + 4 * (lead + rows))
    if kind == "write":
        return {"bytes": new + 2 * hkv * hd * 2 * lead, "flops": 4 * hkv * hd * (lead + rows)}
    first, pairs = _span(case)
    flops = 4 * h * hd * pairs
    if kind == "step":
        return {"bytes": 2 * hkv * hd * (pos - first) + new + 8 * h * hd, "flops": flops}
    return {"bytes": 2 * hkv * hd * (pos + rows - first) + 8 * rows * h * hd, "flops": flops}


# ------------------------------------------------------------------------- 64-bit results

def _exact_linear(d, group):
    w, s = d["w"].long(), d["scales"].double()
    parts = []
    for o in range(0, w.shape[0], 8192):
        q = torch.empty(w[o:o + 8192].shape[0], w.shape[1] * 8, dtype=torch.float64, device=w.device)
        for i in range(8):
            q[:, i::8] = ((w[o:o + 8192] >> (4 * i)) % 16).double()
        z = 8.0 if d["zeros"] is None else d["zeros"][o:o + 8192].double().repeat_interleave(group, 1)
        parts.append(d["a"].double() @ ((q - z) * s[o:o + 8192].repeat_interleave(group, 1)).t().contiguous())
    return torch.cat(parts, 1)


def _step(e):
    """2^e in 64 bits, for whole e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rows(codes, exps, x, pos, block):
    """The cache's values, rows 0..pos + n, after x's rows: block by block in 64 bits."""
    n = x.shape[0]
    x = x.double()
    end = pos + n
    val = torch.empty(end, *x.shape[1:], dtype=torch.float64, device=x.device)
    for b in range(-(-end // block)):
        lo, hi = b * block, min(end, (b + 1) * block)
        step = _step(exps[b].long() - 127)[:, None]  # [hkv, 1]
        old = codes[lo:min(hi, pos)].double() if lo < pos else None
        if hi <= pos:
            val[lo:hi] = old * step
            continue
        new = x[max(lo, pos) - pos:hi - pos]
        top = new.abs().amax((0, 2))
        e = torch.ceil(torch.log2(top / 127))
        e = e.clamp(min=-126)
        e = torch.where(top > 127 * _step(e), e + 1, e)  # (log2 rounds either way)
        e = torch.where(top <= 127 * _step(e - 1), e - 1, e).clamp(min=-126)
        grown = _step(e)[:, None]
        if old is not None:
            grown = torch.maximum(grown, step)
            val[lo:pos] = torch.round(old * (step / grown)) * grown
        val[max(lo, pos):hi] = torch.round(new / grown) * grown
    return val


def _exact_attention(q, k, v, pos, scale, window):
    rows, h, hd = q.shape
    g = h // k.shape[1]
    out = torch.empty(rows, h, hd, dtype=torch.float64, device=q.device)
    for head in range(h):
        kh, vh = k[:, head // g].t().contiguous(), v[:, head // g].contiguous()
        for r0 in range(0, rows, 1024):
            r1 = min(rows, r0 + 1024)
            at = torch.arange(pos + r0, pos + r1, device=q.device)[:, None]
            key = torch.arange(0, pos + r1, device=q.device)[None]
            hidden = key > at
            if window:
                hidden = hidden | (key <= at - window)
            s = (q[r0:r1, head].double() @ kh[:, :pos + r1].contiguous()) * scale
            out[r0:r1, head] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ vh[:pos + r1]
    return out


def _exact_choice(d):
    import numpy as np
    x = d["logits"].cpu().numpy().astype(np.float64)
    t, k, p, m, u = (d[n].cpu().numpy().astype(np.float64)
                     for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    tokens = []
    for r in range(len(x)):
        if t[r] <= 0:
            tokens.append(int(np.argmax(x[r])))
            continue
        w = np.exp((x[r] - x[r].max()) / t[r])
        best = np.lexsort((np.arange(len(w)), -x[r]))
        if k[r] > 0:
            best = best[:int(k[r])]
        if p[r] < 1:
            sums = np.cumsum(w[best])
            best = best[:1 + int(np.searchsorted(sums[:-1], p[r] * sums[-1], "left"))]
        best = np.sort(best[w[best] >= m[r]])
        sums = np.cumsum(w[best])
        tokens.append(int(best[np.searchsorted(sums, u[r] * sums[-1], "right")]))
    return torch.tensor(tokens, dtype=torch.int32)


def exact(case, seed):
    d = _inputs(case, seed)
    kind = case["kind"]
    if kind == "linear":
        return {"out": _exact_linear(d, case["group"])}
    if kind == "sample":
        return {"token": _exact_choice(d)}
    h, hkv, hd, scale = SHAPES[case["shape"]]
    rows, pos, block = case["rows"], case["pos"], case["block"]
    none = torch.zeros(0, hkv, hd, device="cuda")
    val = {}
    for n in "kv":
        x, at = (none, pos + rows) if kind == "chunk" else (d[n], pos)
        val[n] = _exact_rows(d[n + "c"], d[n + "s"], x, at, block)
    start = pos // block * block
    out = {} if kind == "chunk" else {n: val[n][start:] for n in "kv"}
    if kind != "write":
        o = _exact_attention(d["q"].view(rows, h, hd), val["k"], val["v"], pos, scale, case["window"])
        out["out"] = o.view(d["q"].shape)
    return out
