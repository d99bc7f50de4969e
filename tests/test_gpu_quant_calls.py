"""The quantised operators where other tests do not go: calls from several threads at once, more heads
per KV head than the few-row kernel takes, layers of unlike head dims."""
import threading

import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import attention_bound, pack_q4
from tests.test_gpu_cache_i8 import Layer, attend, close, rows

pytestmark = pytest.mark.gpu


def test_threads_share_the_workspace(dev):
    """Three threads whose calls use the device's workspace give the bits of calls one by one."""
    note("quantised calls from three threads")
    rng = np.random.default_rng(1)
    h, hkv, hd, n = 32, 8, 128, 3000
    la = Layer(dev, n, hkv, hd, 64, 1)
    la.write(rows(rng, n, hkv, hd), rows(rng, n, hkv, hd), 0)
    q1, q2 = (eb.Tensor.from_array(dev, rng.standard_normal((m, h, hd)).astype(np.float32)) for m in (1, 60))
    w = eb.LinearQ4(eb.Tensor.from_array(dev, pack_q4(rng.integers(0, 16, (512, 2048)))),
                    eb.Tensor.from_array(dev, (rng.random((512, 16)) * 0.1).astype(np.float16)), None, 2048, 512, 128)
    xs = [eb.Tensor.from_array(dev, rng.standard_normal((m, 2048)).astype(np.float32)) for m in (20, 100)]
    logits = eb.Tensor.from_array(dev, (3 * rng.standard_normal((5, 50000))).astype(np.float32))
    u, p = (eb.Tensor.from_array(dev, rng.random(5).astype(np.float32)) for _ in range(2))

    def attention(rec):
        o1, o2 = eb.Tensor.empty(dev, (h, hd)), eb.Tensor.empty(dev, (60, h, hd))
        eb.attn_decode_i8(rec, q1, la.kv, 0, o1, h, n - 1, 0.1)
        eb.attn_prefill_chunk_i8(rec, q2, la.kv, 0, o2, h, n - 60, 60, 0.1)
        return o1, o2

    def linear(rec):
        return [w.forward(rec, x, m) for x, m in zip(xs, (20, 100))]

    def sample(rec):
        out = eb.Tensor.empty(dev, (5,), eb.DType.U32)
        eb.sample(rec, logits, u, out, 5, 50000, top_p=p)
        return (out,)

    def run(call):
        rec = eb.Recorder(dev)
        outs = call(rec)
        rec.submit()
        return [o.read_bytes() for o in outs]

    calls = (attention, linear, sample)
    want = [run(c) for c in calls]
    wrong = []

    def loop(i):
        for _ in range(40):
            if run(calls[i]) != want[i]:
                wrong.append(calls[i].__name__)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("h,hkv,hd,pos", [(208, 1, 32, 300), (512, 2, 64, 70), (194, 1, 48, 0)])
def test_many_heads_per_kv_head(dev, h, hkv, hd, pos):
    """A token of more columns than the few-row kernel takes: the step's cache and both its forms."""
    note(f"i8 step {h}/{hkv}x{hd} pos {pos}")
    rng = np.random.default_rng(h)
    la = Layer(dev, pos + 1, hkv, hd, 32, 2)
    if pos:
        la.write(rows(rng, pos, hkv, hd), rows(rng, pos, hkv, hd), 0)
    k, v = rows(rng, 1, hkv, hd) * np.float32(5), rows(rng, 1, hkv, hd)
    q = rng.standard_normal((1, h, hd)).astype(np.float32)
    for window in (0, 9):
        ot = eb.Tensor.empty(dev, (h, hd))
        rec = eb.Recorder(dev)
        eb.attn_decode_step_i8(rec, *(eb.Tensor.from_array(dev, x[0]) for x in (q, k, v)), la.kv, 0, ot, h, pos, 0.2, window)
        rec.submit()
        la.model[0].write(k, pos)
        la.model[1].write(v, pos)
        la.check("step")
        kk, vv = la.values(pos + 1)
        want, bound = attention_bound(q, kk, vv, 0.2, pos, window)
        close(ot.to_f32().reshape(q.shape), want, bound, f"step, window {window}")
        close(attend(dev, la, q, pos, 0.2, window), want, bound, f"attention, window {window}")


def test_layers_of_unlike_head_dims(dev):
    """A cache of several layers: each call touches its own."""
    rng = np.random.default_rng(3)
    dims, hkv, n = (64, 32, 128), 2, 70
    kv = eb.KvCache.new_i8_per_layer(dev, dims, 100, hkv, 16)
    data = [(rows(rng, n, hkv, d), rows(rng, n, hkv, d)) for d in dims]
    rec = eb.Recorder(dev)
    for l, (k, v) in enumerate(data):
        eb.kv_write_i8(rec, kv, l, eb.Tensor.from_array(dev, k), eb.Tensor.from_array(dev, v), n, 0)
    rec.submit()
    for l, d in enumerate(dims):
        la = Layer(dev, 100, hkv, d, 16, 4)
        la.write(*data[l], 0)
        la.kv, alone = kv, la.kv
        assert kv.k_scale[l].read_bytes() == alone.k_scale[0].read_bytes()
        q = rng.standard_normal((1, 6, d)).astype(np.float32)
        kk, vv = la.values(n)
        want, bound = attention_bound(q, kk, vv, 0.1, n - 1)
        ot = eb.Tensor.empty(dev, (6, d))
        rec = eb.Recorder(dev)
        eb.attn_decode_i8(rec, eb.Tensor.from_array(dev, q), kv, l, ot, 6, n - 1, 0.1)
        rec.submit()
        close(ot.to_f32().reshape(q.shape), want, bound, f"layer {l}")
