"""The quantised operators together, as a model's layer and a token's end use them: 4-bit projections,
per-head norms and RoPE, the block-scaled cache and its attention, the head and the choice."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import CacheModel, sample_f64, unpack_q4
from tests._textbook import attention_f64, rel_l2_f64, rmsnorm_f64, rope_f64

pytestmark = pytest.mark.gpu
EPS, THETA = 1e-6, 1e4


def dequantised(p):
    codes, s, z, _ = unpack_q4(p.packed.read_bytes(), p.in_f, p.out_f, p.group, p.zeros)
    z = np.full(s.shape, 8.0) if z is None else z.astype(np.float64)
    return (codes - np.repeat(z, p.group, 1)) * np.repeat(s.astype(np.float64), p.group, 1)


class Model:
    """A layer on the device and its definition in 64 bits."""

    def __init__(self, dev, h, hkv, hd, hidden, max_seq, block, window=0, norms=True, group=64, seed=0):
        rng = np.random.default_rng(seed)
        self.dev, self.h, self.hkv, self.hd, self.window = dev, h, hkv, hd, window
        shapes = ((h * hd, hidden), (hkv * hd, hidden), (hkv * hd, hidden), (hidden, h * hd))
        self.q4 = tuple(eb.LinearQ4.from_f32(dev, rng.standard_normal(s) / np.sqrt(s[1]), group, symmetric=False) for s in shapes)
        self.w = [dequantised(p) for p in self.q4]
        self.gains = [1 + 0.1 * rng.standard_normal(hd).astype(np.float32) for _ in range(3)] if norms else [None] * 3
        self.tensors = [None if g is None else eb.Tensor.from_array(dev, g.astype(np.float32)) for g in self.gains]
        self.attn = eb.Attention(h, hkv, hd, hd ** -0.5, *self.tensors, norm_eps=EPS, window=window, hidden=hidden, q4=self.q4)
        self.rope = eb.Rope.build(dev, max_seq, hd, THETA)
        self.kv = eb.KvCache.new_i8(dev, 1, max_seq, hkv, hd, block)
        self.model = [CacheModel(max_seq, hkv, hd, block) for _ in range(2)]

    def forward(self, x, pos):
        rec = eb.Recorder(self.dev)
        y = self.attn.forward(rec, eb.Tensor.from_array(self.dev, x), self.rope, self.kv, 0, len(x), pos)
        rec.submit()
        return y.to_f32().reshape(x.shape)

    def definition(self, x, pos):
        n = len(x)
        q, k, v = (np.asarray(x, np.float64) @ w.T for w in self.w[:3])
        rows = []
        for t, heads, g in zip((q, k, v), (self.h, self.hkv, self.hkv), self.gains):
            t = t.reshape(n, heads, self.hd)
            rows.append(t if g is None else rmsnorm_f64(t, g.astype(np.float32), self.hd, EPS).reshape(t.shape))
        q, k = (rope_f64(t, n, t.shape[1], self.hd, THETA, base_pos=pos) for t in rows[:2])
        for m, t in zip(self.model, (k, rows[2])):
            m.write(t.astype(np.float32), pos)
        kk, vv = (m.values(0, pos + n) for m in self.model)
        o = attention_f64(q, kk, vv, self.hd ** -0.5, q_offset=pos, window=self.window)
        return o.reshape(n, -1) @ self.w[3].T

    def check_cache(self, n):
        """The codes' rows come from projections in f32: those next to a border round either way, by
        one step. A projected value is off by about 1e-6 of the block's largest at most, a step is
        1/127 of it at least, so up to 2 * 127e-6 of the codes may differ; ten times that is allowed."""
        for t, e, m in ((self.kv.k[0], self.kv.k_scale[0], self.model[0]), (self.kv.v[0], self.kv.v_scale[0], self.model[1])):
            codes = np.frombuffer(t.read_bytes(), np.int8).reshape(m.codes.shape)[:n].astype(int)
            exps = np.frombuffer(e.read_bytes(), np.uint8).reshape(m.exps.shape)
            assert (exps[:-(-n // m.block)] == m.exps[:-(-n // m.block)]).all()
            d = np.abs(codes - m.codes[:n])
            assert d.max() <= 1 and (d > 0).mean() <= 2.5e-3, (d.max(), (d > 0).mean())


@pytest.mark.parametrize("h,hkv,hd,hidden", [(8, 2, 64, 256), (4, 4, 128, 512), (6, 2, 96, 384), (34, 2, 32, 128), (4, 1, 256, 256)])
@pytest.mark.parametrize("window", [0, 48])
@pytest.mark.parametrize("norms", [True, False])
def test_layer(dev, h, hkv, hd, hidden, window, norms):
    """A prompt, its next chunk, a short one, and tokens, against the definition. A differing code is
    a step of its value, at most 2.5e-3 of them: rel-L2 1/127 * sqrt(2.5e-3) = 4e-4, through the
    softmax up to a few times that."""
    note(f"quant layer {h}/{hkv}x{hd} window {window} norms {norms}")
    m = Model(dev, h, hkv, hd, hidden, 256, 32, window, norms, seed=hd)
    rng = np.random.default_rng(1)
    pos = 0
    for n in (70, 45, 3, 1, 1, 1, 16, 1):
        x = rng.standard_normal((n, hidden)).astype(np.float32)
        want = m.definition(x, pos)
        got = m.forward(x, pos)
        assert rel_l2_f64(got, want) <= 2e-3, (n, pos, rel_l2_f64(got, want))
        pos += n
        m.check_cache(pos)


def test_tokens_from_a_graph(dev):
    """Head and choice captured once and replayed: a sampling loop whose tokens are the definition's."""
    rng = np.random.default_rng(3)
    hidden, vocab = 256, 5000
    head = eb.LinearQ4.from_f32(dev, rng.standard_normal((vocab, hidden)) / 8, 32)
    x, logits = eb.Tensor.empty(dev, (1, hidden)), eb.Tensor.empty(dev, (1, vocab))
    u, token = eb.Tensor.empty(dev, (1,)), eb.Tensor.empty(dev, (1,), eb.DType.U32)
    k, p = eb.Tensor.from_array(dev, np.array([200], np.uint32)), eb.Tensor.from_array(dev, np.array([0.9], np.float32))

    def step():
        rec = eb.Recorder(dev)
        eb.linear_q4(rec, x, head, logits, 1)
        eb.sample(rec, logits, u, token, 1, vocab, top_k=k, top_p=p)
        rec.submit()

    x.write(np.zeros((1, hidden), np.float32))
    u.write(np.zeros(1, np.float32))
    step()
    dev.begin_capture()
    step()
    graph = dev.end_capture()
    for _ in range(6):
        r = np.float32(rng.random())
        x.write(rng.standard_normal((1, hidden)).astype(np.float32))
        u.write(np.array([r], np.float32))
        graph.launch()
        dev.synchronize()
        want = sample_f64(logits.to_f32(), float(r), 1.0, 200, float(np.float32(0.9)), 0.0)
        assert int(np.frombuffer(token.read_bytes(), np.uint32)[0]) == want


def test_layer_step_from_a_graph(dev):
    """A captured token replays to the eager call's bits, at each position a capture of its own."""
    rng = np.random.default_rng(4)
    a, b = (Model(dev, 8, 2, 64, 256, 128, 16, seed=9) for _ in range(2))
    x0 = rng.standard_normal((40, 256)).astype(np.float32)
    a.forward(x0, 0)
    b.forward(x0, 0)
    xt = eb.Tensor.empty(dev, (1, 256))
    b.forward(x0[:1], 40)  # (fills the pool and the workspace)
    a.forward(x0[:1], 40)
    graph = None
    for pos in range(41, 46):
        x = rng.standard_normal((1, 256)).astype(np.float32)
        want = a.forward(x, pos)
        dev.begin_capture()
        rec = eb.Recorder(dev)
        y = b.attn.forward(rec, xt, b.rope, b.kv, 0, 1, pos)
        rec.submit()
        graph = dev.end_capture(graph)
        for _ in range(3):
            xt.write(x)
            graph.launch()
            dev.synchronize()
            assert y.to_f32().tobytes() == want.tobytes()
        written = (pos + 1) * 2 * 64  # (rows behind it are as the pool left them)
        assert a.kv.k[0].read_bytes()[:written] == b.kv.k[0].read_bytes()[:written]


def test_other_calls_refuse_a_block_scaled_cache(dev):
    kv = eb.KvCache.new_i8(dev, 1, 64, 2, 64, 16)
    src = eb.Tensor.empty(dev, (1, 2, 64))
    rec = eb.Recorder(dev)
    with pytest.raises(eb.ShapeMismatch):
        eb.kv_write(rec, kv.k[0], src, 2, 1, 64, 64, 0)
    with pytest.raises(eb.ShapeMismatch):
        eb.attn_decode(rec, src, kv.k[0], kv.v[0], src, 2, 2, 0, 64, 64, 0.1)
    plain = eb.KvCache.new(dev, 1, 64, 2, 64)
    with pytest.raises(eb.ShapeMismatch):
        eb.kv_write_i8(rec, plain, 0, src, src, 1, 0)
    with pytest.raises(eb.ShapeMismatch):
        eb.attn_decode_i8(rec, src, kv, 1, src, 2, 0, 0.1)
    for bad in ((48, 64), (512, 64), (16, 40), (16, 16)):
        with pytest.raises(eb.UnsupportedConfig):
            eb.KvCache.new_i8(dev, 1, 64, 2, bad[1], bad[0])
    rec.submit()


@pytest.mark.parametrize("hkv,hd", [(2, 128), (8, 32)])
@pytest.mark.parametrize("rows", [1, 5])
def test_a_cache_of_other_heads_is_refused(dev, hkv, hd, rows):
    """As many codes a position, in other heads: blocks and exponents lie elsewhere."""
    attn = eb.Attention(8, 4, 64, 0.125, None, None, None)
    kv = eb.KvCache.new_i8(dev, 1, 64, hkv, hd, 16)
    q, k = eb.Tensor.empty(dev, (rows, 512)), eb.Tensor.empty(dev, (rows, 256))
    for t in (q, k):
        t.write(np.zeros(t.shape, np.float32))
    with pytest.raises(eb.ShapeMismatch, match="block-scaled"):
        attn.forward_qkv(eb.Recorder(dev), q, k, k, eb.Rope.build(dev, 64, 64, THETA), kv, 0, rows, 0)
