"""Block-scaled 8-bit KV caches on the GPU against their definition in 64 bits: codes and exponents
bit for bit, attention within a bound derived from the kernels' arithmetic (tests/_quant.py)."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import CacheModel, attention_bound
from tests._textbook import rel_l2_f64

pytestmark = pytest.mark.gpu


def rows(rng, n, hkv, hd, spread=0.5):
    return (rng.standard_normal((n, hkv, hd)) * np.exp(spread * rng.standard_normal((n, hkv, 1)))).astype(np.float32)


class Layer:
    """A one-layer cache on the device beside its model."""

    def __init__(self, dev, max_seq, hkv, hd, block, seed=0):
        rng = np.random.default_rng(seed)
        self.dev, self.hkv, self.hd, self.max_seq = dev, hkv, hd, max_seq
        self.kv = eb.KvCache.new_i8(dev, 1, max_seq, hkv, hd, block)
        self.model = [CacheModel(max_seq, hkv, hd, block, rng) for _ in range(2)]
        for t, m in zip((self.kv.k[0], self.kv.v[0]), self.model):
            t.write(m.codes)

    def write(self, k, v, dst, model=True):
        rec = eb.Recorder(self.dev)
        eb.kv_write_i8(rec, self.kv, 0, eb.Tensor.from_array(self.dev, k), eb.Tensor.from_array(self.dev, v), len(k), dst)
        rec.submit()
        if model:
            self.model[0].write(k, dst)
            self.model[1].write(v, dst)

    def check(self, what=""):
        got = ((self.kv.k[0], self.kv.k_scale[0]), (self.kv.v[0], self.kv.v_scale[0]))
        for name, (codes, exps), m in zip("kv", got, self.model):
            assert exps.read_bytes() == m.exps.tobytes(), f"{what}: {name} exponents"
            assert codes.read_bytes() == m.codes.tobytes(), f"{what}: {name} codes"

    def values(self, n):
        return self.model[0].values(0, n), self.model[1].values(0, n)


def close(got, want, bound, what):
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    err = np.abs(got - want)
    worst = float((err / np.maximum(bound, 1e-300)).max())
    assert (err <= bound).all(), f"{what}: {worst:.3f} of the bound"
    rel = rel_l2_f64(got, want)
    assert rel <= 2e-5, f"{what}: rel-L2 {rel:.3e}"


SHAPES = [(16, 8, 128), (32, 8, 128), (16, 8, 256), (14, 2, 64), (6, 2, 96), (3, 3, 32), (5, 1, 48), (10, 2, 208)]


@pytest.mark.parametrize("h,hkv,hd", SHAPES)
@pytest.mark.parametrize("block", [16, 64, 256])
def test_write_and_read(dev, h, hkv, hd, block):
    note(f"i8 write {hkv}x{hd} block {block}")
    rng = np.random.default_rng(hd + block)
    la = Layer(dev, 600, hkv, hd, block, 1)
    dst = 0
    # appends of every kind: inside a block, to its end, over several; sizes that make the exponent
    # grow, stay, and (at a block's first row) shrink; one row of zeros; a rewind.
    for n, scale in ((1, 1.0), (1, 0.01), (3, 8.0), (40, 1.0), (1, 0.0), (70, 1e-3), (200, 300.0), (1, 1e-30), (30, 1e20)):
        k, v = rows(rng, n, hkv, hd) * np.float32(scale), rows(rng, n, hkv, hd)
        la.write(k, v, dst)
        la.check(f"{n} rows at {dst}")
        dst += n
    la.write(rows(rng, 20, hkv, hd), rows(rng, 20, hkv, hd), 100)
    la.check("rewind")
    count, start = 333, 7
    kt, vt = (eb.Tensor.empty(dev, (count, hkv, hd)) for _ in range(2))
    rec = eb.Recorder(dev)
    eb.kv_read_i8(rec, la.kv, 0, kt, vt, count, start)
    rec.submit()
    for t, m in zip((kt, vt), la.model):
        want = m.values(start, start + count).astype(np.float32)
        assert t.to_f32().reshape(want.shape).tobytes() == want.tobytes()


def test_write_takes_the_last_row_and_no_row(dev):
    la = Layer(dev, 100, 2, 64, 64)
    rng = np.random.default_rng(3)
    la.write(rows(rng, 100, 2, 64), rows(rng, 100, 2, 64), 0)
    la.write(rows(rng, 1, 2, 64) * 50, rows(rng, 1, 2, 64), 99)
    la.check()
    empty = eb.Tensor.empty(dev, (0, 2, 64))
    rec = eb.Recorder(dev)
    eb.kv_write_i8(rec, la.kv, 0, empty, empty, 0, 100)
    eb.kv_read_i8(rec, la.kv, 0, empty, empty, 0, 100)
    rec.submit()
    la.check()


def test_code_borders(dev):
    """Values at halves of a step round to even codes; the largest at and just past 127 steps."""
    hd = 32
    x = np.zeros((4, 1, hd), np.float32)
    x[0, 0] = (np.arange(hd) - 15.5) * 0.5  # halves and wholes
    x[0, 0, 0] = 127.0
    for i, top in enumerate((127.0, np.nextafter(np.float32(127), np.float32(200)), np.float32(2.0 ** -140))):
        la = Layer(dev, 64, 1, hd, 16)
        y = x.copy()
        y[0, 0, 0] = top
        if i == 2:
            y[:] = 0
            y[1, 0, 3] = top
        la.write(y, -y, 0)
        la.check(f"border {i}")


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_non_finite_value_makes_its_block_nan(dev, bad):
    la = Layer(dev, 128, 2, 64, 32)
    rng = np.random.default_rng(5)
    k, v = rows(rng, 70, 2, 64), rows(rng, 70, 2, 64)
    k[40, 1, 9] = bad
    la.write(k, v, 0)
    la.check("written")
    la.write(rows(rng, 1, 2, 64), rows(rng, 1, 2, 64), 50)  # (still NaN: row 40 stays)
    la.check("appended")
    h, q = 4, rng.standard_normal((1, 4, 64)).astype(np.float32)
    got = attend(dev, la, q, 49, 64 ** -0.5)
    assert np.isnan(got[0, 2:]).all() and np.isfinite(got[0, :2]).all()
    # a window that ends before the block, and one that starts behind it
    assert np.isfinite(attend(dev, la, q, 31, 64 ** -0.5)).all()
    assert np.isfinite(attend(dev, la, q, 69, 64 ** -0.5, window=6)).all()
    # rows of one call that see the block, beside one that does not
    q2 = rng.standard_normal((2, h, 64)).astype(np.float32)
    got = attend(dev, la, q2, 31, 64 ** -0.5)
    assert np.isfinite(got[0]).all() and np.isnan(got[1, 2:]).all()
    # written anew from its first row on
    la.write(rows(rng, 38, 2, 64), rows(rng, 38, 2, 64), 32)
    assert np.isfinite(attend(dev, la, q, 69, 64 ** -0.5)).all()


def attend(dev, la, q, pos, scale, window=0):
    n, h, hd = q.shape
    qt, ot = eb.Tensor.from_array(dev, q), eb.Tensor.empty(dev, q.shape)
    rec = eb.Recorder(dev)
    if n == 1:
        eb.attn_decode_i8(rec, qt, la.kv, 0, ot, h, pos, scale, window)
    else:
        eb.attn_prefill_chunk_i8(rec, qt, la.kv, 0, ot, h, pos, n, scale, window)
    rec.submit()
    return ot.to_f32().reshape(q.shape)


@pytest.mark.parametrize("h,hkv,hd", SHAPES)
@pytest.mark.parametrize("pos", [0, 1, 15, 16, 63, 64, 127, 200, 1537])
def test_decode(dev, h, hkv, hd, pos):
    note(f"i8 decode {h}/{hkv}x{hd} pos {pos}")
    rng = np.random.default_rng(pos + hd)
    la = Layer(dev, pos + 1 + pos % 3, hkv, hd, 64, 2)
    la.write(rows(rng, pos + 1, hkv, hd), rows(rng, pos + 1, hkv, hd, 2.0), 0)
    q = rng.standard_normal((1, h, hd)).astype(np.float32)
    for window in (0, 1, 40):
        k, v = la.values(pos + 1)
        want, bound = attention_bound(q, k, v, hd ** -0.5, pos, window)
        close(attend(dev, la, q, pos, hd ** -0.5, window), want, bound, f"window {window}")


@pytest.mark.parametrize("h,hkv,hd", [(16, 8, 128), (32, 8, 128), (16, 8, 256), (14, 2, 64), (6, 2, 96), (34, 2, 64), (80, 1, 32)])
@pytest.mark.parametrize("pos", [0, 1, 63, 64, 100, 640, 2050])
@pytest.mark.parametrize("block", [16, 64, 256])
def test_step(dev, h, hkv, hd, pos, block):
    """The fused step: cache bit for bit, attention over the cache as it then is; a second step on
    the next row, whose larger values round the block's codes again."""
    note(f"i8 step {h}/{hkv}x{hd} pos {pos} block {block}")
    rng = np.random.default_rng(pos + block)
    la = Layer(dev, pos + 2, hkv, hd, block, 3)
    if pos:
        la.write(rows(rng, pos, hkv, hd), rows(rng, pos, hkv, hd), 0)
    for i, size in enumerate((1.0, 9.0)):
        q = rng.standard_normal((1, h, hd)).astype(np.float32)
        k, v = rows(rng, 1, hkv, hd) * np.float32(size), rows(rng, 1, hkv, hd) * np.float32(size)
        ot = eb.Tensor.empty(dev, (h, hd))
        window = (0, 70)[i]
        rec = eb.Recorder(dev)
        eb.attn_decode_step_i8(rec, eb.Tensor.from_array(dev, q[0]), eb.Tensor.from_array(dev, k[0]),
                               eb.Tensor.from_array(dev, v[0]), la.kv, 0, ot, h, pos + i, hd ** -0.5, window)
        rec.submit()
        la.model[0].write(k, pos + i)
        la.model[1].write(v, pos + i)
        la.check(f"step {i}")
        kk, vv = la.values(pos + i + 1)
        want, bound = attention_bound(q, kk, vv, hd ** -0.5, pos + i, window)
        close(ot.to_f32().reshape(1, h, hd), want, bound, f"step {i}")


@pytest.mark.parametrize("h,hkv,hd", [(16, 8, 128), (8, 2, 128), (4, 2, 256), (14, 2, 64), (6, 2, 96), (3, 3, 32)])
@pytest.mark.parametrize("pos,n", [(0, 2), (0, 33), (5, 3), (30, 17), (100, 40), (700, 9), (513, 130)])
@pytest.mark.parametrize("window", [0, 50])
def test_chunk(dev, h, hkv, hd, pos, n, window):
    note(f"i8 chunk {h}/{hkv}x{hd} pos {pos} rows {n} window {window}")
    rng = np.random.default_rng(pos + n)
    la = Layer(dev, pos + n + 5, hkv, hd, 32, 4)
    la.write(rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd), 0)
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    k, v = la.values(pos + n)
    want, bound = attention_bound(q, k, v, hd ** -0.5, pos, window)
    close(attend(dev, la, q, pos, hd ** -0.5, window), want, bound, "chunk")


def test_blocks_of_unlike_size(dev):
    """V blocks 2^40 apart: the small ones keep their precision where the large one has no weight,
    and the large one is right where it has."""
    hkv, hd, n = 1, 64, 512
    rng = np.random.default_rng(11)
    for big_weight in (False, True):
        la = Layer(dev, n, hkv, hd, 64, 5)
        k, v = rng.standard_normal((n, hkv, hd)).astype(np.float32), rows(rng, n, hkv, hd)
        q = rng.standard_normal((1, 4, hd)).astype(np.float32)
        v[128:192] *= np.float32(2.0 ** 40)
        if not big_weight:
            k[128:192, 0] = -20.0 * q[0].mean(0)  # scores far below the others'
            q[:] = q[0].mean(0)
        la.write(k, v, 0)
        kk, vv = la.values(n)
        want, bound = attention_bound(q, kk, vv, 1.0, n - 1)
        close(attend(dev, la, q, n - 1, 1.0), want, bound, f"big weight {big_weight}")


def test_large_and_small_scores(dev):
    """q and K far from 1 in both directions, and scores that single out one key."""
    rng = np.random.default_rng(13)
    la = Layer(dev, 300, 2, 64, 64, 6)
    k, v = rows(rng, 300, 2, 64), rows(rng, 300, 2, 64)
    for fq, fk, scale in ((1e-20, 1e20, 0.125), (1e15, 1e-15, 0.125), (1.0, 1.0, 3.0), (1e-30, 1.0, 1.0)):
        la.write((k * np.float32(fk)).astype(np.float32), v, 0)
        q = (rng.standard_normal((1, 4, 64)) * fq).astype(np.float32)
        kk, vv = la.values(300)
        want, bound = attention_bound(q, kk, vv, scale, 299)
        close(attend(dev, la, q, 299, scale), want, bound, f"{fq} {fk} {scale}")


def test_graph_replays(dev):
    """A captured step, replayed with new inputs between the program's own calls."""
    rng = np.random.default_rng(17)
    h, hkv, hd, pos = 8, 2, 64, 150
    la = Layer(dev, 256, hkv, hd, 64, 7)
    la.write(rows(rng, pos, hkv, hd), rows(rng, pos, hkv, hd), 0)
    qt, kt, vt = eb.Tensor.empty(dev, (h, hd)), eb.Tensor.empty(dev, (hkv, hd)), eb.Tensor.empty(dev, (hkv, hd))
    ot = eb.Tensor.empty(dev, (h, hd))

    def step():
        rec = eb.Recorder(dev)
        eb.attn_decode_step_i8(rec, qt, kt, vt, la.kv, 0, ot, h, pos, hd ** -0.5)
        rec.submit()

    for t in (qt, kt, vt):
        t.write(np.zeros(t.shape, np.float32))
    step()  # (the workspace)
    la.model[0].write(np.zeros((1, hkv, hd), np.float32), pos)
    la.model[1].write(np.zeros((1, hkv, hd), np.float32), pos)
    dev.begin_capture()
    step()
    graph = dev.end_capture()
    for i in range(4):
        q, k, v = rng.standard_normal((1, h, hd)).astype(np.float32), rows(rng, 1, hkv, hd) * (i + 1), rows(rng, 1, hkv, hd)
        qt.write(q[0])
        kt.write(np.float32(k[0]))
        vt.write(v[0])
        graph.launch()
        dev.synchronize()
        la.model[0].write(np.float32(k), pos)
        la.model[1].write(v, pos)
        la.check(f"replay {i}")
        kk, vv = la.values(pos + 1)
        want, bound = attention_bound(q, kk, vv, hd ** -0.5, pos)
        close(ot.to_f32().reshape(1, h, hd), want, bound, f"replay {i}")
        other = eb.Tensor.from_f32(dev, (5,), np.arange(5))
        assert other.to_f32()[4] == 4.0


def test_two_calls_give_the_same_bits(dev):
    rng = np.random.default_rng(19)
    la = Layer(dev, 3000, 8, 128, 64, 8)
    la.write(rows(rng, 3000, 8, 128), rows(rng, 3000, 8, 128), 0)
    q = rng.standard_normal((1, 32, 128)).astype(np.float32)
    first = attend(dev, la, q, 2999, 128 ** -0.5)
    assert attend(dev, la, q, 2999, 128 ** -0.5).tobytes() == first.tobytes()


def test_raw_launches(dev):
    """The raw entry points on the same memory give the handle calls' bits."""
    rng = np.random.default_rng(23)
    h, hkv, hd, block, n = 16, 8, 128, 64, 700
    la, lb = (Layer(dev, 1024, hkv, hd, block, 9) for _ in range(2))
    k, v = rows(rng, n, hkv, hd), rows(rng, n, hkv, hd)
    la.write(k, v, 0)
    kt, vt = eb.Tensor.from_array(dev, k), eb.Tensor.from_array(dev, v)
    kv = lb.kv
    cache = eb.CacheI8(kv.k[0].data_ptr, kv.k_scale[0].data_ptr, kv.v[0].data_ptr, kv.v_scale[0].data_ptr,
                       kv.k[0].numel(), kv.k_scale[0].numel(), 1024, hkv, hd, block)
    eb.launch_kv_write_i8(dev.stream, cache, kt.data_ptr, vt.data_ptr, k.size, n, 0)
    dev.synchronize()
    lb.model = la.model
    lb.check("raw write")
    for m in (1, 90):
        q = rng.standard_normal((m, h, hd)).astype(np.float32)
        qt, ot = eb.Tensor.from_array(dev, q), eb.Tensor.empty(dev, q.shape)
        floats = eb.attn_i8_workspace_floats(h, hkv, hd, n - m, m, block, 0, dev.cu_count)
        ws = eb.Tensor.empty(dev, (max(floats, 1),))
        if m == 1:
            eb.launch_attn_decode_i8(dev.stream, qt.data_ptr, q.size, 0, 0, 0, cache, ot.data_ptr, q.size, h, n - 1,
                                     0.1, 0, ws.data_ptr, floats, dev.cu_count)
        else:
            eb.launch_attn_prefill_chunk_i8(dev.stream, qt.data_ptr, q.size, cache, ot.data_ptr, q.size, h, n - m, m,
                                            0.1, 0, ws.data_ptr, floats, dev.cu_count)
        dev.synchronize()
        assert ot.to_f32().tobytes() == attend(dev, la, q, n - m, 0.1).tobytes()
        with pytest.raises(eb.ShapeMismatch):
            eb.launch_attn_prefill_chunk_i8(dev.stream, qt.data_ptr, q.size, cache, ot.data_ptr, q.size, h, n - m, m,
                                            0.1, 0, ws.data_ptr, floats - 1, dev.cu_count)
