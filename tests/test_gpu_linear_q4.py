"""4-bit projections on the GPU against their definition in 64 bits, within the bound of the
kernels' arithmetic (tests/_quant.py)."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import linear_q4_bound, pack_q4, unpack_q4

pytestmark = pytest.mark.gpu


def weight(rng, out_f, in_f, group, zeros):
    codes = rng.integers(0, 16, (out_f, in_f))
    scales = (np.exp(rng.standard_normal((out_f, in_f // group))) * 0.02).astype(np.float16)
    scales *= rng.choice(np.array([-1, 1], np.float16), scales.shape)
    z = rng.integers(0, 16, scales.shape).astype(np.uint8) if zeros else None
    return codes, scales, z


def device_weight(dev, codes, scales, z, group):
    return eb.LinearQ4(eb.Tensor.from_array(dev, pack_q4(codes)), eb.Tensor.from_array(dev, scales),
                       None if z is None else eb.Tensor.from_array(dev, z), codes.shape[1], codes.shape[0], group)


def run(dev, a, w):
    out = eb.Tensor.empty(dev, (len(a), w.out_f))
    out.write(np.full((len(a), w.out_f), np.nan, np.float32))
    rec = eb.Recorder(dev)
    eb.linear_q4(rec, eb.Tensor.from_array(dev, a), w, out, len(a))
    rec.submit()
    return out.to_f32().reshape(len(a), w.out_f)


def close(got, want, bound, what):
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    err = np.abs(got - want)
    worst = float((err / np.maximum(bound, 1e-300)).max())
    assert (err <= bound).all(), f"{what}: {worst:.3f} of the bound"


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 31, 33, 64, 65, 130])
def test_rows(dev, m, group, zeros):
    note(f"q4 {m} rows group {group} zeros {zeros}")
    rng = np.random.default_rng(m)
    for in_f, out_f in ((128, 1), (384, 129), (640, 48), (group, 7), (3 * group, 130), (2048, 300)):
        codes, scales, z = weight(rng, out_f, in_f, group, zeros)
        a = (rng.standard_normal((m, in_f)) * np.exp(2 * rng.standard_normal((m, 1)))).astype(np.float32)
        want, bound = linear_q4_bound(a, codes, scales, z, group)
        close(run(dev, a, device_weight(dev, codes, scales, z, group)), want, bound, f"{in_f} to {out_f}")


@pytest.mark.parametrize("m,in_f,out_f", [(1, 1024, 20000), (4, 4096, 5000), (8, 4736, 257), (8, 6144, 100), (1, 16384, 64),
                                          (300, 1152, 777), (1, 40960, 33), (2, 1024, 9000), (700, 1024, 3000), (129, 640, 16500)])
def test_large(dev, m, in_f, out_f):
    note(f"q4 {m} rows {in_f} to {out_f}")
    rng = np.random.default_rng(in_f)
    codes, scales, z = weight(rng, out_f, in_f, 64, True)
    a = rng.standard_normal((m, in_f)).astype(np.float32)
    want, bound = linear_q4_bound(a, codes, scales, z, 64)
    close(run(dev, a, device_weight(dev, codes, scales, z, 64)), want, bound, "large")


@pytest.mark.parametrize("m,in_f,out_f,group", [(33, 8320, 130, 32), (40, 512, 128, 128), (128, 4128, 64, 32),
                                                (129, 4096, 1000, 64), (257, 384, 5, 128), (200, 2112, 4096, 64)])
def test_shared_contraction(dev, m, in_f, out_f, group):
    """Few tiles of a long contraction: workgroups share it; the same bits every time."""
    note(f"q4 {m} rows {in_f} to {out_f} group {group}")
    rng = np.random.default_rng(in_f + m)
    codes, scales, z = weight(rng, out_f, in_f, group, m % 2 == 0)
    a = rng.standard_normal((m, in_f)).astype(np.float32)
    want, bound = linear_q4_bound(a, codes, scales, z, group)
    w = device_weight(dev, codes, scales, z, group)
    got = run(dev, a, w)
    close(got, want, bound, "shared")
    assert run(dev, a, w).tobytes() == got.tobytes()


@pytest.mark.parametrize("m", [1, 20, 100])
def test_extreme_rows(dev, m):
    """Rows of zeros, of tiny and of huge values beside ordinary ones; a zero point above 15."""
    rng = np.random.default_rng(7)
    codes, scales, z = weight(rng, 40, 256, 64, True)
    z[:] = rng.integers(0, 256, z.shape)
    a = rng.standard_normal((m, 256)).astype(np.float32)
    for i, f in enumerate((1e-38, 1e30, 0.0)):
        a[i * m // 3] *= np.float32(f)
    want, bound = linear_q4_bound(a, codes, scales, z, 64)
    # (below f32's normal range a result may lose bits: one step of 2^-149, with its sums')
    close(run(dev, a, device_weight(dev, codes, scales, z, 64)), want, bound + 1e-42, "extreme")


@pytest.mark.parametrize("m", [2, 70])
def test_a_row_that_is_not_finite_stays_alone(dev, m):
    rng = np.random.default_rng(9)
    codes, scales, z = weight(rng, 50, 256, 32, False)
    a = rng.standard_normal((m, 256)).astype(np.float32)
    a[1, 17] = np.inf
    got = run(dev, a, device_weight(dev, codes, scales, z, 32))
    assert not np.isfinite(got[1]).any()
    a[1] = 0
    want, bound = linear_q4_bound(a, codes, scales, z, 32)
    got[1] = 0
    close(got, want, bound, "the other rows")


@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_multi_is_the_single_calls(dev, m):
    rng = np.random.default_rng(m)
    a = rng.standard_normal((m, 512)).astype(np.float32)
    ws = [device_weight(dev, *weight(rng, n, 512, 64, True), 64) for n in (256, 100, 33)]
    at = eb.Tensor.from_array(dev, a)
    outs = [eb.Tensor.empty(dev, (m, w.out_f)) for w in ws]
    rec = eb.Recorder(dev)
    eb.linear_q4_multi(rec, at, ws, outs, m)
    rec.submit()
    for w, o in zip(ws, outs):
        want = run(dev, a, w)
        # (the grid, and with it how waves share a contraction, may differ: f32 sums, not bits)
        np.testing.assert_allclose(o.to_f32().reshape(m, -1), want, rtol=0, atol=1e-4 * np.abs(want).max())


def test_from_f32_and_forward(dev):
    rng = np.random.default_rng(1)
    w = rng.standard_normal((96, 256)).astype(np.float32)
    w[3, :64] = 0
    x = rng.standard_normal((3, 256)).astype(np.float32)
    for group in (32, 64, 128):
        for symmetric in (True, False):
            p = eb.LinearQ4.from_f32(dev, w, group, symmetric)
            rec = eb.Recorder(dev)
            y = p.forward(rec, eb.Tensor.from_array(dev, x), 3)
            rec.submit()
            got = y.to_f32().reshape(3, 96)
            # a code is off by half a step (and a clipped end by one): the group's range / 14 or / 15
            span = np.ptp(np.concatenate((w, np.zeros((96, 1), np.float32)), 1), axis=1).max() if not symmetric else 2 * np.abs(w).max()
            assert np.abs(got - x @ w.T).max() <= span / 14 * np.abs(x).sum(1).max()


def test_graph_replays(dev):
    rng = np.random.default_rng(2)
    codes, scales, z = weight(rng, 70, 512, 128, True)
    w = device_weight(dev, codes, scales, z, 128)
    for m in (1, 50):
        at, out = eb.Tensor.empty(dev, (m, 512)), eb.Tensor.empty(dev, (m, 70))
        at.write(np.zeros((m, 512), np.float32))

        def step():
            rec = eb.Recorder(dev)
            eb.linear_q4(rec, at, w, out, m)
            rec.submit()

        step()
        dev.begin_capture()
        step()
        graph = dev.end_capture()
        for _ in range(3):
            a = rng.standard_normal((m, 512)).astype(np.float32)
            at.write(a)
            graph.launch()
            dev.synchronize()
            want, bound = linear_q4_bound(a, codes, scales, z, 128)
            close(out.to_f32().reshape(m, 70), want, bound, "replay")
            assert run(dev, a, w).tobytes() == out.to_f32().tobytes()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_pack(dev, group):
    """The packed layout holds the weight, and zeros besides."""
    rng = np.random.default_rng(group)
    for out_f, in_f in ((1, group), (16, 128), (50, 3 * group), (129, 1152)):
        for zeros in (False, True):
            codes, scales, z = weight(rng, out_f, in_f, group, zeros)
            w = device_weight(dev, codes, scales, z, group)
            assert w.packed.numel() == eb.q4_packed_bytes(in_f, out_f, group, zeros)
            c, s, zz, clean = unpack_q4(w.packed.read_bytes(), in_f, out_f, group, zeros)
            np.testing.assert_array_equal(c, codes)
            assert s.tobytes() == scales.tobytes() and clean
            if zeros:
                np.testing.assert_array_equal(zz, z)


def test_infinite_scales_stay_with_their_feature(dev):
    rng = np.random.default_rng(12)
    for m in (1, 20, 200):
        codes, scales, z = weight(rng, 40, 160, 32, True)
        scales[7, 4], scales[20, 0] = np.inf, np.nan
        a = rng.standard_normal((m, 160)).astype(np.float32)
        got = run(dev, a, device_weight(dev, codes, scales, z, 32))
        assert not np.isfinite(got[:, [7, 20]]).any()
        keep = [i for i in range(40) if i not in (7, 20)]
        want, bound = linear_q4_bound(a, codes[keep], scales[keep], z[keep], 32)
        close(got[:, keep], want, bound, "the other features")


def test_raw_launch(dev):
    rng = np.random.default_rng(3)
    codes, scales, z = weight(rng, 65, 256, 64, True)
    w = device_weight(dev, codes, scales, z, 64)
    wt, st, zt = (eb.Tensor.from_array(dev, x) for x in (pack_q4(codes), scales, z))
    packed = eb.Tensor.empty(dev, (w.packed.numel(),), eb.DType.U8)
    eb.launch_q4_pack(dev.stream, wt.data_ptr, wt.numel(), st.data_ptr, st.numel(), zt.data_ptr, zt.numel(), 256, 65, 64,
                      packed.data_ptr, packed.numel())
    dev.synchronize()
    assert packed.read_bytes() == w.packed.read_bytes()
    for m in (1, 17, 300):
        a = rng.standard_normal((m, 256)).astype(np.float32)
        at, out = eb.Tensor.from_array(dev, a), eb.Tensor.empty(dev, (m, 65))
        floats = eb.linear_q4_workspace_floats(m, 256)
        ws = eb.Tensor.empty(dev, (max(floats, 1),))
        eb.launch_linear_q4(dev.stream, at.data_ptr, a.size, packed.data_ptr, packed.numel(), out.data_ptr, m * 65, m, 256, 65,
                            64, True, ws.data_ptr, floats)
        dev.synchronize()
        assert out.to_f32().tobytes() == run(dev, a, w).tobytes()


def test_pack_waits_for_the_null_stream(dev):
    """A weight that the null stream is still filling is packed whole, and may be overwritten at once.
    (It writes the words as the codes of a block-scaled cache laid over them.)"""
    rng = np.random.default_rng(21)
    out_f, in_f, hkv, hd, block = 600, 2048, 4, 256, 16
    b = rng.integers(-127, 128, (out_f, in_f // 2))
    b[::block, ::hd] = 127  # (every block's exponent leaves whole numbers as they are)
    words = b.astype(np.int8).view(np.uint32)
    codes = (words[..., None] >> (4 * np.arange(8, dtype=np.uint32)) & 15).reshape(out_f, in_f)
    _, scales, _ = weight(rng, out_f, in_f, 128, False)
    wt, st = eb.Tensor.empty(dev, words.shape, eb.DType.U32), eb.Tensor.from_array(dev, scales)
    wt.write(np.zeros_like(words))
    spare = eb.Tensor.empty(dev, (out_f, hkv, hd), eb.DType.I8)
    exps = [eb.Tensor.empty(dev, ((out_f + block - 1) // block, hkv), eb.DType.U8) for _ in range(2)]
    cache = eb.CacheI8(wt.data_ptr, exps[0].data_ptr, spare.data_ptr, exps[1].data_ptr, spare.numel(), exps[0].numel(),
                       out_f, hkv, hd, block)
    n = 16384
    big = eb.KvCache.new_i8(dev, 1, n, 8, 128, 64)
    long = eb.CacheI8(big.k[0].data_ptr, big.k_scale[0].data_ptr, big.v[0].data_ptr, big.v_scale[0].data_ptr,
                      big.k[0].numel(), big.k_scale[0].numel(), n, 8, 128, 64)
    load = eb.Tensor.empty(dev, (n, 8, 128))
    load.write(np.ones((n, 8, 128), np.float32))
    x, none = eb.Tensor.from_array(dev, b.astype(np.float32)), eb.Tensor.from_array(dev, np.zeros(b.shape, np.float32))
    dev.synchronize()
    for _ in range(20):
        eb.launch_kv_write_i8(0, long, load.data_ptr, load.data_ptr, load.numel(), n, 0)
    eb.launch_kv_write_i8(0, cache, x.data_ptr, x.data_ptr, b.size, out_f, 0)
    w = eb.LinearQ4(wt, st, None, in_f, out_f, 128)
    eb.launch_kv_write_i8(0, cache, none.data_ptr, none.data_ptr, b.size, out_f, 0)
    a = rng.standard_normal((2, in_f)).astype(np.float32)
    want, bound = linear_q4_bound(a, codes, scales, None, 128)
    close(run(dev, a, w), want, bound, "packed behind the null stream")
    eb.LinearQ4(wt, st, None, in_f, out_f, 128)  # (waits for the writes above, before their tensors go)


def test_pack_during_a_capture_is_refused(dev):
    rng = np.random.default_rng(22)
    codes, scales, z = weight(rng, 16, 128, 64, False)
    ts = eb.Tensor.from_array(dev, pack_q4(codes)), eb.Tensor.from_array(dev, scales)
    dev.begin_capture()
    try:
        with pytest.raises(eb.EyebrowseError, match="captured"):
            eb.LinearQ4(*ts, None, 128, 16, 64)
    finally:
        dev.end_capture()


def test_pack_leaves_another_capture_alone(dev):
    """Weights are loaded while another device's stream (of the same GPU) is being captured."""
    rng = np.random.default_rng(23)
    codes, scales, z = weight(rng, 48, 256, 64, True)
    other = eb.Device.new(0)
    w = device_weight(other, codes, scales, z, 64)
    a = rng.standard_normal((2, 256)).astype(np.float32)
    want, bound = linear_q4_bound(a, codes, scales, z, 64)
    at, out = eb.Tensor.from_array(other, a), eb.Tensor.empty(other, (2, 48))

    def step():
        rec = eb.Recorder(other)
        eb.linear_q4(rec, at, w, out, 2)
        rec.submit()

    step()
    out.write(np.zeros((2, 48), np.float32))
    other.begin_capture()
    try:
        mine = device_weight(dev, codes, scales, z, 64)
        step()
    finally:
        graph = other.end_capture()
    close(run(dev, a, mine), want, bound, "packed during the capture")
    for _ in range(3):
        graph.launch()
        other.synchronize()
        close(out.to_f32().reshape(2, 48), want, bound, "the captured call")
