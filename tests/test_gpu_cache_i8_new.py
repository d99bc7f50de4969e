"""Making a block-scaled cache: complete when the call returns."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._quant import CacheModel, pack_q4

pytestmark = pytest.mark.gpu


def test_a_new_cache_takes_another_streams_rows_at_once(dev):
    """The device's stream is busy while a cache is made; rows that the null stream writes right
    after the call stay as written."""
    rng = np.random.default_rng(1)
    n, hkv, hd, block = 130, 2, 64, 32
    w, s = eb.Tensor.from_array(dev, pack_q4(rng.integers(0, 16, (16, 128)))), eb.Tensor.from_array(dev, np.ones((16, 1), np.float16))
    long = 16384
    big = eb.KvCache.new_i8(dev, 1, long, 8, 128, 64)
    load = eb.Tensor.empty(dev, (long, 8, 128))
    load.write(np.ones((long, 8, 128), np.float32))
    k, v = (rng.standard_normal((n, hkv, hd)).astype(np.float32) for _ in range(2))
    kt, vt = eb.Tensor.from_array(dev, k), eb.Tensor.from_array(dev, v)
    rec = eb.Recorder(dev)
    for _ in range(300):
        eb.kv_write_i8(rec, big, 0, load, load, long, 0)
    rec.submit()
    kv = eb.KvCache.new_i8(dev, 1, n, hkv, hd, block)
    cache = eb.CacheI8(kv.k[0].data_ptr, kv.k_scale[0].data_ptr, kv.v[0].data_ptr, kv.v_scale[0].data_ptr, kv.k[0].numel(),
                       kv.k_scale[0].numel(), n, hkv, hd, block)
    eb.launch_kv_write_i8(0, cache, kt.data_ptr, vt.data_ptr, k.size, n, 0)
    eb.LinearQ4(w, s, None, 128, 16, 128)  # (waits for both streams)
    for x, codes, exps in ((k, kv.k[0], kv.k_scale[0]), (v, kv.v[0], kv.v_scale[0])):
        m = CacheModel(n, hkv, hd, block)
        m.write(x, 0)
        assert codes.read_bytes() == m.codes.tobytes()
        assert exps.read_bytes() == m.exps.tobytes()


def test_a_cache_is_made_beside_another_capture(dev):
    """Another device's stream (of the same GPU) is being captured meanwhile; its graph is whole."""
    rng = np.random.default_rng(2)
    other = eb.Device.new(0)
    x = rng.standard_normal((5, 2, 64)).astype(np.float32)
    kv = eb.KvCache.new_i8(other, 1, 40, 2, 64, 16)
    xt = eb.Tensor.from_array(other, x)
    other.begin_capture()
    try:
        mine = eb.KvCache.new_i8(dev, 2, 100, 2, 64, 16)
        rec = eb.Recorder(other)
        eb.kv_write_i8(rec, kv, 0, xt, xt, 5, 3)
        rec.submit()
    finally:
        graph = other.end_capture()
    assert all(set(e.read_bytes()) == {1} for e in mine.k_scale + mine.v_scale)
    for scale in (1.0, 3.0, 0.5):
        y = x * np.float32(scale)
        xt.write(y)
        kv.k_scale[0].write(np.ones((3, 2), np.uint8))
        graph.launch()
        other.synchronize()
        m = CacheModel(40, 2, 64, 16)
        m.write(y, 3)
        assert kv.k_scale[0].read_bytes() == m.exps.tobytes()
        got = np.frombuffer(kv.k[0].read_bytes(), np.int8).reshape(m.codes.shape)
        np.testing.assert_array_equal(got[3:8], m.codes[3:8])
