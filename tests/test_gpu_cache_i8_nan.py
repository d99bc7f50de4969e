"""Blocks of a block-scaled cache that hold a value that is not finite: exactly the query rows that
see one of their keys are NaN, whichever kernels a call's size picks; every other row is its
definition's."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import assert_close, note
from tests._quant import attention_bound
from tests._textbook import attention_f64
from tests.test_gpu_cache_i8 import Layer, attend, close, rows

pytestmark = pytest.mark.gpu


def check(dev, h, hkv, hd, block, pos, n, window, bad):
    """bad: (side, row, head) of the values that are not finite."""
    rng = np.random.default_rng(pos + n + hd)
    la = Layer(dev, pos + n, hkv, hd, block, 4)
    kv = [rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd)]
    nan_block = np.zeros((pos + n, hkv), bool)
    for i, (side, row, head) in enumerate(bad):
        kv[side][row, head, 7 * i % hd] = (np.inf, np.nan, -np.inf)[i % 3]
        nan_block[row // block * block:(row // block + 1) * block, head] = True
    la.write(*kv, 0)
    la.check("written")
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    at, key = pos + np.arange(n)[:, None], np.arange(pos + n)[None]
    seen = (key <= at) & ((key > at - window) if window else True)
    nan = np.repeat(seen.astype(int) @ nan_block.astype(int) > 0, h // hkv, axis=1)  # [n, h]
    got = attend(dev, la, q, pos, hd ** -0.5, window)
    assert np.isnan(got[nan]).all(), f"{np.isfinite(got[nan]).all(-1).sum()} of {nan.sum()} rows that see the block are finite"
    k, v = (np.nan_to_num(x, nan=0.0) for x in la.values(pos + n))  # (the other rows do not see these)
    want, bound = attention_bound(q, k, v, hd ** -0.5, pos, window)
    if not nan.all():
        close(got[~nan], want[~nan], bound[~nan], f"the {(~nan).sum()} rows that do not see the block")


@pytest.mark.parametrize("h,hkv,hd,block", [(4, 2, 256, 64), (4, 2, 64, 256), (8, 2, 128, 256), (3, 3, 32, 256)])
def test_k_blocks_that_fill_a_share_of_the_keys(dev, h, hkv, hd, block):
    """Workgroups share a short chunk's keys; every score of one share is NaN, the others' are not."""
    note(f"i8 nan share {h}/{hkv}x{hd} block {block}")
    check(dev, h, hkv, hd, block, 640, 200, 0, [(0, block + 5, 0)])
    check(dev, h, hkv, hd, block, 640, 200, 300, [(0, block + 5, 0)])


@pytest.mark.parametrize("h,hkv,hd,bad", [(4, 2, 256, (64, 128)), (4, 2, 64, (128, 384)), (3, 3, 32, (128, 384))])
def test_k_rows_of_an_f32_cache_that_fill_a_share(dev, h, hkv, hd, bad):
    """The same over an f32 cache, whose chunks the same merge ends."""
    note(f"f32 nan share {h}/{hkv}x{hd}")
    rng = np.random.default_rng(hd)
    pos, n = 640, 200
    k, v = rows(rng, pos + n, hkv, hd), rows(rng, pos + n, hkv, hd)
    k[bad[0]:bad[1], 0] = np.nan
    q = rng.standard_normal((n, h, hd)).astype(np.float32)
    qt, kt, vt, ot = (eb.Tensor.from_array(dev, x) for x in (q, k, v, np.zeros_like(q)))
    rec = eb.Recorder(dev)
    eb.attn_prefill_chunk(rec, qt, kt, vt, ot, h, hkv, pos, n, hd, pos + n, hd ** -0.5)
    rec.submit()
    got = ot.to_f32().reshape(q.shape)
    assert np.isnan(got[:, :h // hkv]).all()
    want = attention_f64(q, np.nan_to_num(k, nan=0.0), v, hd ** -0.5, q_offset=pos)
    assert_close(got[:, h // hkv:], want[:, h // hkv:], what="the other heads")


@pytest.mark.parametrize("h,hkv,hd,block", [(4, 2, 256, 64), (4, 2, 64, 256), (8, 2, 128, 256), (3, 3, 32, 256)])
def test_v_blocks_that_fill_a_share_of_the_keys(dev, h, hkv, hd, block):
    note(f"i8 nan V share {h}/{hkv}x{hd} block {block}")
    check(dev, h, hkv, hd, block, 640, 200, 0, [(1, block + 5, 0)])
    check(dev, h, hkv, hd, block, 640, 200, 300, [(1, block + 5, 0)])


@pytest.mark.parametrize("h,hkv,hd", [(4, 2, 64), (16, 8, 128), (4, 2, 256), (3, 3, 48)])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("pos,n", [(0, 200), (0, 33), (45, 210), (301, 200), (1000, 6)])
@pytest.mark.parametrize("window", [0, 40])
def test_rows_that_do_not_see_the_block(dev, h, hkv, hd, block, pos, n, window):
    """A block among the chunk's own rows, one behind a window's start, and one in another head."""
    note(f"i8 nan {h}/{hkv}x{hd} block {block} pos {pos} rows {n} window {window}")
    last = pos + n - 1
    for side in (0, 1):
        bad = [(side, pos + n // 2, 0), (1 - side, last, hkv - 1)]
        if window and pos > window:
            bad.append((side, pos - window + 3, 1))
        check(dev, h, hkv, hd, block, pos, n, window, bad)
