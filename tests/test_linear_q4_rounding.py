"""LinearQ4.from_f32: the weight it packs is the given one within its steps, and its products are that
weight's; what its half scales cannot hold is refused."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._quant import linear_q4_bound, unpack_q4


def weights(seed):
    """Groups of each kind: ordinary, all above or below zero, of zeros, with one large value, and
    far from 1 in size."""
    rng = np.random.default_rng(seed)
    w = rng.standard_normal((75, 384)).astype(np.float32)
    w[3, :128] = 0
    w[5] = np.abs(w[5])
    w[6] = -np.abs(w[6])
    w[7, ::50] *= 40
    w[8] *= 1e4
    w[9] *= np.float32(1e-2)
    w[10] += 3
    w[11, :] = -0.25
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [True, False])
def test_from_f32_keeps_the_weight(dev, group, symmetric):
    """A code is the nearest whole number of steps s, s a half next to the range's 1/14 or 1/15 (off by
    2^-11 of it), so a weight is off by s/2; where the zero point's own rounding moves the largest
    past code 15, by what 15 steps of the wrong size miss besides: (1/2 + 15 2^-11) s. The quotient
    in f32 adds 15 2^-24."""
    w = weights(group)
    p = eb.LinearQ4.from_f32(dev, w, group, symmetric)
    codes, s, z, clean = unpack_q4(p.packed.read_bytes(), 384, 75, group, p.zeros)
    assert clean and p.zeros == (not symmetric)
    steps = np.repeat(s.astype(np.float64), group, 1)
    zero = np.repeat(np.full(s.shape, 8.0) if z is None else z.astype(np.float64), group, 1)
    off = np.abs((codes - zero) * steps - w)
    assert (off <= (0.5 + 15 * 2.0 ** -11 + 16 * 2.0 ** -24) * steps).all(), (off / np.maximum(steps, 1e-30)).max()
    lo, hi = (f(w.reshape(75, -1, group), axis=-1) for f in (np.min, np.max))
    width = 2 * np.maximum(-lo, hi) / 14 if symmetric else (np.maximum(hi, 0) - np.minimum(lo, 0)) / 15
    assert (np.abs(s - width) <= width * 1.01 * 2.0 ** -11).all()
    x = np.random.default_rng(1).standard_normal((3, 384)).astype(np.float32)
    rec = eb.Recorder(dev)
    y = p.forward(rec, eb.Tensor.from_array(dev, x), 3)
    rec.submit()
    want, bound = linear_q4_bound(x, codes, s, z, group)
    assert (np.abs(y.to_f32().reshape(3, 75) - want) <= bound).all()


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 1e6, -3e38])
def test_from_f32_refuses_what_a_half_scale_cannot_hold(symmetric, bad):
    """(refused before a device is needed)"""
    w = np.ones((4, 128), np.float32)
    w[2, 70] = bad
    with pytest.raises(eb.UnsupportedConfig, match="scale"):
        eb.LinearQ4.from_f32(None, w, 64, symmetric)
