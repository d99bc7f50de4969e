"""Sampling on the GPU against its definition in 64 bits: the tokens are equal."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests._quant import sample_f64

pytestmark = pytest.mark.gpu


def run(dev, x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows, vocab = x.shape
    f = lambda a, t=np.float32: None if a is None else eb.Tensor.from_array(dev, np.broadcast_to(np.asarray(a, t), (rows,)))  # noqa: E731
    out = eb.Tensor.empty(dev, (rows,), eb.DType.U32)
    out.write(np.full(rows, 0xFFFFFFFF, np.uint32))
    rec = eb.Recorder(dev)
    eb.sample(rec, eb.Tensor.from_array(dev, x.astype(np.float32)), f(u), out, rows, vocab, temperature=f(temperature),
              top_k=f(top_k, np.uint32), top_p=f(top_p), min_p=f(min_p))
    rec.submit()
    return np.frombuffer(out.read_bytes(), np.uint32).astype(np.int64)


def want(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = len(x)
    b = [np.broadcast_to(np.asarray(a, np.float32), (rows,)) for a in (u, temperature, top_k, top_p, min_p)]
    return np.array([sample_f64(x[r].astype(np.float32), *(float(c[r]) for c in b)) for r in range(rows)])


CHOICES = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(top_p=0.05), dict(min_p=0.1),
           dict(temperature=1.3, top_k=50, top_p=0.8), dict(temperature=0.8, top_k=100, top_p=0.95, min_p=0.02),
           dict(temperature=2.0, top_p=0.99, min_p=0.001), dict(temperature=0.0), dict(top_k=5, min_p=0.5)]


@pytest.mark.parametrize("choice", CHOICES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 63), (5, 1000), (4, 4096), (7, 4097), (33, 8191), (2, 50257)])
def test_choices(dev, rows, vocab, choice):
    note(f"sample {rows}x{vocab} {choice}")
    rng = np.random.default_rng(vocab + rows)
    x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    np.testing.assert_array_equal(run(dev, x, u, **choice), want(x, u, **choice))


def test_largest_vocabulary_and_many_rows(dev):
    rng = np.random.default_rng(1)
    x = (2 * rng.standard_normal((3, 151936))).astype(np.float32)
    u = rng.random(3).astype(np.float32)
    for c in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.97), dict(temperature=5.0, top_p=0.999), dict(top_k=100000, top_p=0.7)):
        np.testing.assert_array_equal(run(dev, x, u, **c), want(x, u, **c))
    x = rng.standard_normal((700, 500)).astype(np.float32)
    u = rng.random(700).astype(np.float32)
    np.testing.assert_array_equal(run(dev, x, u, top_k=20, top_p=0.8), want(x, u, top_k=20, top_p=0.8))


def test_a_very_long_row(dev):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((1, 4300007)).astype(np.float32)
    for u in (0.1, 0.93):
        for c in (dict(top_k=30), dict(top_p=0.4)):
            np.testing.assert_array_equal(run(dev, x, np.float32([u]), **c), want(x, np.float32([u]), **c))


def test_each_row_has_its_own_parameters(dev):
    rng = np.random.default_rng(2)
    rows = 64
    x = (4 * rng.standard_normal((rows, 3001))).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    c = dict(temperature=rng.choice([0.0, 0.5, 1.0, 3.0], rows), top_k=rng.choice([0, 1, 7, 500, 3001, 5000], rows),
             top_p=rng.choice([0.1, 0.6, 0.95, 1.0, 2.0], rows), min_p=rng.choice([0.0, 0.01, 0.3, 1.0], rows))
    np.testing.assert_array_equal(run(dev, x, u, **c), want(x, u, **c))


def test_ties_rank_by_index(dev):
    """Few distinct logits: cuts fall among equal ones."""
    rng = np.random.default_rng(3)
    x = rng.integers(0, 4, (40, 5000)).astype(np.float32)
    u = rng.random(40).astype(np.float32)
    for c in (dict(top_k=7), dict(top_k=1300), dict(top_p=0.5), dict(top_p=0.001), dict(top_k=3000, top_p=0.5), dict(top_k=2000, top_p=0.999),
              dict(min_p=1.0), dict(temperature=0.0)):
        np.testing.assert_array_equal(run(dev, x, u, **c), want(x, u, **c))
    flat = np.zeros((6, 20000), np.float32)
    flat[1::2] = -0.0
    flat[:, ::3] *= -1
    u = np.linspace(0, 0.999, 6).astype(np.float32)
    for c in (dict(), dict(top_k=999), dict(top_p=0.25), dict(top_k=9999, top_p=0.5), dict(temperature=0.0)):
        np.testing.assert_array_equal(run(dev, flat, u, **c), want(flat, u, **c))


def test_unusual_logits(dev):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((12, 700)).astype(np.float32)
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, ::2] = np.nan
    x[3, 5:] = -np.inf
    x[4, 77] = np.inf
    x[5, [3, 600]] = np.inf
    x[6] *= 1e30
    x[7] *= 1e-30
    x[8] = -np.inf
    x[8, 699] = -1e38
    x[9, :] = np.finfo(np.float32).min
    x[10, 0] = np.finfo(np.float32).max
    x[11, :350] = -np.inf
    u = rng.random(12).astype(np.float32)
    for c in CHOICES:
        np.testing.assert_array_equal(run(dev, x, u, **c), want(x, u, **c))


def test_ends_of_the_random_number(dev):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 400)).astype(np.float32)
    x[:, 0] = -np.inf  # (a token of no weight is not taken, at u = 0 either)
    u = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, 2.0, -1.0, np.nan], np.float32)
    for c in (dict(), dict(top_k=3), dict(top_p=0.5)):
        np.testing.assert_array_equal(run(dev, x, u, **c), want(x, u, **c))


def test_out_of_range_parameters(dev):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((3, 900)).astype(np.float32)
    u = rng.random(3).astype(np.float32)
    best = x.argmax(1)
    for c in (dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=1.5), dict(temperature=-1.0), dict(temperature=np.nan)):
        np.testing.assert_array_equal(run(dev, x, u, **c), best)
    plain = want(x, u)
    for c in (dict(top_p=np.nan), dict(min_p=-1.0), dict(min_p=np.nan), dict(top_k=900), dict(top_k=2 ** 32 - 1), dict(top_p=np.inf)):
        np.testing.assert_array_equal(run(dev, x, u, **c), plain)
    np.testing.assert_array_equal(run(dev, x, u, temperature=1e-30), best)
    np.testing.assert_array_equal(run(dev, x, u, temperature=1e-42), best)
    np.testing.assert_array_equal(run(dev, x, u, temperature=np.inf), want(np.where(np.isfinite(x), 0, x), u))


def test_graph_replays_read_the_current_parameters(dev):
    rng = np.random.default_rng(8)
    rows, vocab = 3, 20000
    lt, ut = eb.Tensor.empty(dev, (rows, vocab)), eb.Tensor.empty(dev, (rows,))
    tt, kt, pt = eb.Tensor.empty(dev, (rows,)), eb.Tensor.empty(dev, (rows,), eb.DType.U32), eb.Tensor.empty(dev, (rows,))
    out = eb.Tensor.empty(dev, (rows,), eb.DType.U32)

    def fill(i):
        x = (3 * np.random.default_rng(i).standard_normal((rows, vocab))).astype(np.float32)
        u = np.random.default_rng(i + 50).random(rows).astype(np.float32)
        c = dict(temperature=np.float32([0.5, 1.0, 2.0]), top_k=np.array([5 * i, 0, 100 + i]), top_p=np.float32([0.9, 0.5 + 0.1 * (i % 4), 1.0]))
        for t, a in ((lt, x), (ut, u), (tt, c["temperature"]), (kt, c["top_k"].astype(np.uint32)), (pt, c["top_p"])):
            t.write(a)
        return x, u, c

    def step():
        rec = eb.Recorder(dev)
        eb.sample(rec, lt, ut, out, rows, vocab, temperature=tt, top_k=kt, top_p=pt)
        rec.submit()

    fill(0)
    step()
    dev.begin_capture()
    step()
    graph = dev.end_capture()
    for i in range(1, 5):
        x, u, c = fill(i)
        graph.launch()
        dev.synchronize()
        np.testing.assert_array_equal(np.frombuffer(out.read_bytes(), np.uint32), want(x, u, **c))
        assert run(dev, x[:1, :100], u[:1]).shape == (1,)  # (the program's own call between)


def test_raw_launch(dev):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((2, 5000)).astype(np.float32)
    u = rng.random(2).astype(np.float32)
    xt, ut, out = eb.Tensor.from_array(dev, x), eb.Tensor.from_array(dev, u), eb.Tensor.empty(dev, (2,), eb.DType.U32)
    floats = eb.sample_workspace_floats(2, 5000)
    ws = eb.Tensor.empty(dev, (max(floats, 1),))
    eb.launch_sample(dev.stream, xt.data_ptr, x.size, ut.data_ptr, out.data_ptr, 2, 5000, ws_ptr=ws.data_ptr, ws_floats=floats)
    dev.synchronize()
    np.testing.assert_array_equal(np.frombuffer(out.read_bytes(), np.uint32), want(x, u))


@pytest.mark.parametrize("choice", [dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.95, min_p=0.02), dict(temperature=0.0)])
@pytest.mark.parametrize("rows,vocab", [(900, 12289), (1900, 4100), (450, 20480)])
def test_many_rows(dev, rows, vocab, choice):
    """More slices than the card holds workgroups: a workgroup takes several of a row."""
    note(f"sample {rows}x{vocab} {choice}")
    rng = np.random.default_rng(vocab + rows)
    x = (3 * rng.standard_normal((rows, vocab), dtype=np.float32))
    x[:, vocab - 1] += np.float32(9)  # (kept tokens at the far end of a row too)
    u = rng.random(rows).astype(np.float32)
    np.testing.assert_array_equal(run(dev, x, u, **choice), want(x, u, **choice))
