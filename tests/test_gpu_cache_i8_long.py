"""Block-scaled 8-bit KV caches: chunks on both sides of the few-row kernel's limit, positions whose
codes lie past 2^31 bytes, the raw token step with its append, and two graphs on one workspace."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import CacheModel, attention_bound
from tests.test_gpu_cache_i8 import Layer, attend, close, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h,hkv,hd", [(4, 4, 64), (16, 8, 128), (16, 8, 256), (14, 2, 64), (6, 2, 96), (3, 3, 32)])
@pytest.mark.parametrize("pos,n", [(0, 193), (0, 257), (63, 200), (1100, 224), (640, 97), (641, 96)])
@pytest.mark.parametrize("window", [0, 90])
def test_longer_chunks(dev, h, hkv, hd, pos, n, window):
    note(f"i8 chunk {h}/{hkv}x{hd} pos {pos} rows {n} window {window}")
    rng = np.random.default_rng(pos + n)
    la = Layer(dev, pos + n, hkv, hd, 64, 4)
    la.write(rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd), 0)
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    k, v = la.values(pos + n)
    want, bound = attention_bound(q, k, v, hd ** -0.5, pos, window)
    close(attend(dev, la, q, pos, hd ** -0.5, window), want, bound, "chunk")
    la.check("after the chunk")


@pytest.mark.parametrize("n", [1, 5, 200])
def test_past_2_31_codes(dev, n):
    """The last rows of a cache of 2.25 GB of codes on each side: write, read back, step, chunk."""
    h, hkv, hd, block, max_seq, window = 16, 8, 256, 64, 1_100_000, 300
    note(f"i8 cache of {max_seq} rows, {n} rows at its end")
    rng = np.random.default_rng(29 + n)
    kv = eb.KvCache.new_i8(dev, 1, max_seq, hkv, hd, block)
    size = 704
    start = (max_seq - size) // block * block  # (a block's start)
    size = max_seq - start
    assert start * hkv * hd > 2 ** 31
    model = [CacheModel(size, hkv, hd, block, rng) for _ in range(2)]
    k, v = rows(rng, size, hkv, hd), rows(rng, size, hkv, hd)
    filled = size - n
    rec = eb.Recorder(dev)
    eb.kv_write_i8(rec, kv, 0, eb.Tensor.from_array(dev, k[:filled]), eb.Tensor.from_array(dev, v[:filled]), filled, start)
    rec.submit()
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    qt, ot = eb.Tensor.from_array(dev, q), eb.Tensor.empty(dev, q.shape)
    kt, vt = eb.Tensor.from_array(dev, k[filled:]), eb.Tensor.from_array(dev, v[filled:])
    rec = eb.Recorder(dev)
    if n == 1:
        eb.attn_decode_step_i8(rec, qt, kt, vt, kv, 0, ot, h, max_seq - 1, hd ** -0.5, window)
    else:
        eb.kv_write_i8(rec, kv, 0, kt, vt, n, max_seq - n)
        eb.attn_prefill_chunk_i8(rec, qt, kv, 0, ot, h, max_seq - n, n, hd ** -0.5, window)
    rec.submit()
    for m, x in zip(model, (k, v)):
        m.write(x[:filled], 0)
        m.write(x[filled:], filled)
    kk, vv = model[0].values(0, size), model[1].values(0, size)
    got_k, got_v = eb.Tensor.empty(dev, k.shape), eb.Tensor.empty(dev, v.shape)
    rec = eb.Recorder(dev)
    eb.kv_read_i8(rec, kv, 0, got_k, got_v, size, start)
    rec.submit()
    assert got_k.to_f32().tobytes() == kk.astype(np.float32).tobytes()
    assert got_v.to_f32().tobytes() == vv.astype(np.float32).tobytes()
    want, bound = attention_bound(q, kk, vv, hd ** -0.5, filled, window)
    close(ot.to_f32().reshape(q.shape), want, bound, f"{n} rows")


@pytest.mark.parametrize("h,hkv,hd,pos", [(16, 8, 128, 500), (16, 8, 128, 64), (40, 2, 64, 300)])
def test_raw_step(dev, h, hkv, hd, pos):
    """The raw token step leaves the handle step's cache and output, bit for bit."""
    rng = np.random.default_rng(pos)
    block = 64
    la, lb = (Layer(dev, pos + 1, hkv, hd, block, 9) for _ in range(2))
    k, v = rows(rng, pos + 1, hkv, hd), rows(rng, pos + 1, hkv, hd)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    for x in (la, lb):
        x.write(k[:pos], v[:pos], 0)
    qt, kt, vt = (eb.Tensor.from_array(dev, x) for x in (q, k[pos], v[pos]))
    oa, ob = eb.Tensor.empty(dev, q.shape), eb.Tensor.empty(dev, q.shape)
    rec = eb.Recorder(dev)
    eb.attn_decode_step_i8(rec, qt, kt, vt, la.kv, 0, oa, h, pos, hd ** -0.5)
    rec.submit()
    kv = lb.kv
    cache = eb.CacheI8(kv.k[0].data_ptr, kv.k_scale[0].data_ptr, kv.v[0].data_ptr, kv.v_scale[0].data_ptr,
                       kv.k[0].numel(), kv.k_scale[0].numel(), pos + 1, hkv, hd, block)
    floats = eb.attn_i8_workspace_floats(h, hkv, hd, pos, 1, block, 0, dev.cu_count)
    ws = eb.Tensor.empty(dev, (max(floats, 1),))
    eb.launch_attn_decode_i8(dev.stream, qt.data_ptr, q.size, kt.data_ptr, vt.data_ptr, hkv * hd, cache, ob.data_ptr,
                             q.size, h, pos, hd ** -0.5, 0, ws.data_ptr, floats, dev.cu_count)
    dev.synchronize()
    la.model[0].write(k[pos:], pos)
    la.model[1].write(v[pos:], pos)
    lb.model = la.model
    la.check("handle")
    lb.check("raw")
    assert oa.to_f32().tobytes() == ob.to_f32().tobytes()


def test_two_graphs_share_the_workspace(dev):
    """Two captured steps over two caches, replayed in turn between eager calls that use the same
    workspace for a longer context."""
    rng = np.random.default_rng(31)
    h, hkv, hd, pos = 32, 8, 128, 900
    caches, steps = [], []
    big = Layer(dev, 3000, hkv, hd, 64, 3)
    big.write(rows(rng, 3000, hkv, hd), rows(rng, 3000, hkv, hd), 0)
    qb = rng.standard_normal((1, h, hd)).astype(np.float32)
    first = attend(dev, big, qb, 2999, hd ** -0.5)  # (the workspace, at its largest)
    for i in range(2):
        la = Layer(dev, pos + 1, hkv, hd, 64, i)
        la.write(rows(rng, pos, hkv, hd), rows(rng, pos, hkv, hd), 0)
        new = rows(rng, 2, hkv, hd)
        q = rng.standard_normal((h, hd)).astype(np.float32)
        ts = [eb.Tensor.from_array(dev, x) for x in (q, new[0], new[1])] + [eb.Tensor.empty(dev, (h, hd))]

        def step(la=la, ts=ts):
            rec = eb.Recorder(dev)
            eb.attn_decode_step_i8(rec, ts[0], ts[1], ts[2], la.kv, 0, ts[3], h, pos, hd ** -0.5)
            rec.submit()

        step()
        caches.append(ts[3].to_f32().tobytes())
        steps.append((step, ts, la))
    graphs = []
    for step, _, _ in steps:
        dev.begin_capture()
        step()
        graphs.append(dev.end_capture())
    for _ in range(3):
        for i in (0, 1):
            steps[i][1][3].write(np.zeros((h, hd), np.float32))
            graphs[i].launch()
        assert attend(dev, big, qb, 2999, hd ** -0.5).tobytes() == first.tobytes()
        for i in (0, 1):
            assert steps[i][1][3].to_f32().tobytes() == caches[i]


def test_a_cache_is_made_outside_a_capture(dev):
    dev.begin_capture()
    try:
        with pytest.raises(eb.EyebrowseError, match="captured"):
            eb.KvCache.new_i8(dev, 1, 64, 2, 64, 16)
    finally:
        dev.end_capture()
    assert set(eb.KvCache.new_i8(dev, 1, 64, 2, 64, 16).k_scale[0].read_bytes()) == {1}
