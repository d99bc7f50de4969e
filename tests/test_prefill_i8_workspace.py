"""The workspace of a long chunk over a block-scaled cache: its records are f16 rows, no more."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import attention_bound


@pytest.mark.parametrize("h,hkv,hd", [(32, 8, 128), (16, 8, 256), (14, 2, 64), (16, 16, 32)])
def test_records_are_halves(hkv, h, hd):
    """49 rows and more behind 32000 keys: two bytes for every element of K and V (33 for 32 key
    slots of K), exponents, the rounding to whole KiB, and at most 64 shares' partial sums."""
    for rows in (200, 513):
        tiles = -(-(32000 + rows) // 32)
        records = hkv * tiles * ((32 * hd + 33 * hd) * 2 + 256 + 1024)
        partials = 64 * rows * h * (hd + 4) * 4
        assert 4 * eb.attn_i8_workspace_floats(h, hkv, hd, 32000, rows, 64) <= records + partials
    full = 4 * (eb.attn_i8_workspace_floats(h, hkv, hd, 64000, 4096, 64) - eb.attn_i8_workspace_floats(h, hkv, hd, 32000, 4096, 64))
    assert full <= hkv * 1000 * ((32 * hd + 33 * hd) * 2 + 256 + 1024)  # (a long chunk has no shares)


@pytest.mark.gpu
@pytest.mark.parametrize("h,hkv,hd", [(4, 2, 32), (6, 3, 48), (16, 8, 128), (4, 1, 256), (3, 3, 208)])
@pytest.mark.parametrize("pos,n", [(0, 200), (77, 230), (3000, 193)])
def test_the_workspace_is_enough(dev, h, hkv, hd, pos, n):
    """A chunk in the room that the call asks for; the memory behind it stays as it was."""
    note(f"i8 chunk {h}/{hkv}x{hd} pos {pos} rows {n} in its smallest workspace")
    rng = np.random.default_rng(pos + hd)
    s, block = pos + n, 32
    codes = [rng.integers(-127, 128, (s, hkv, hd)).astype(np.int8) for _ in range(2)]
    exps = [rng.integers(118, 122, (-(-s // block), hkv)).astype(np.uint8) for _ in range(2)]
    k, v = (c * 2.0 ** (e[np.arange(s) // block].astype(float)[..., None] - 127) for c, e in zip(codes, exps))
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    ts = [eb.Tensor.from_array(dev, x) for x in (codes[0], exps[0], codes[1], exps[1])]
    cache = eb.CacheI8(*(t.data_ptr for t in ts), codes[0].size, exps[0].size, s, hkv, hd, block)
    qt, ot = eb.Tensor.from_array(dev, q), eb.Tensor.empty(dev, q.shape)
    for window in (0, 150):
        floats = eb.attn_i8_workspace_floats(h, hkv, hd, pos, n, block, window, dev.cu_count)
        ws, guard = eb.Tensor.empty(dev, (floats + 4096,)), np.arange(4096, dtype=np.float32)
        ws.write(np.concatenate((np.full(floats, np.nan, np.float32), guard)))
        eb.launch_attn_prefill_chunk_i8(dev.stream, qt.data_ptr, q.size, cache, ot.data_ptr, q.size, h, pos, n, hd ** -0.5, window,
                                        ws.data_ptr, floats, dev.cu_count)
        dev.synchronize()
        want, bound = attention_bound(q, k, v, hd ** -0.5, pos, window)
        got = ot.to_f32().reshape(q.shape)
        assert (np.abs(got - want) <= bound).all()
        assert (ws.to_f32()[floats:] == guard).all()
