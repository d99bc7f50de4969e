"""Sampling's workspace: bounded whatever the rows."""
import numpy as np
import pytest

import eyebrowse_amd as eb
from tests._gpu import note
from tests.test_gpu_sample import want


def test_many_rows_take_a_bounded_workspace():
    """The most rows there may be, of a small vocabulary (their logits: 26 MB) and of a large one."""
    assert 4 * eb.sample_workspace_floats(65535, 100) <= 192 << 20
    assert 4 * eb.sample_workspace_floats(65535, 151936) <= 192 << 20
    for vocab in (1, 5000, 1 << 24):
        sizes = [eb.sample_workspace_floats(rows, vocab) for rows in (1, 2, 63, 1023, 1024, 1025, 4096, 65535)]
        assert sizes == sorted(sizes) and sizes[0] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(4097, 77), (8192, 30), (9001, 50)])
def test_rows_past_a_batch(dev, rows, vocab):
    """Every row has its own logits, number and parameters; the memory behind the workspace stays."""
    note(f"sample {rows}x{vocab} in its smallest workspace")
    rng = np.random.default_rng(rows)
    x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    c = dict(temperature=rng.choice([0.0, 0.7, 2.0], rows).astype(np.float32), top_k=rng.choice([0, 1, 9, 40], rows).astype(np.uint32),
             top_p=rng.choice([0.3, 0.9, 1.0], rows).astype(np.float32), min_p=rng.choice([0.0, 0.05], rows).astype(np.float32))
    u = rng.random(rows).astype(np.float32)
    xt, ut = eb.Tensor.from_array(dev, x), eb.Tensor.from_array(dev, u)
    ts = {n + "_ptr": eb.Tensor.from_array(dev, a) for n, a in c.items()}
    out = eb.Tensor.from_array(dev, np.full(rows + 8, 0xFFFFFFFF, np.uint32))
    floats, guard = eb.sample_workspace_floats(rows, vocab), np.arange(256, dtype=np.float32)
    ws = eb.Tensor.empty(dev, (floats + 256,))
    ws.write(np.concatenate((np.full(floats, np.nan, np.float32), guard)))
    eb.launch_sample(dev.stream, xt.data_ptr, x.size, ut.data_ptr, out.data_ptr, rows, vocab, ws_ptr=ws.data_ptr, ws_floats=floats,
                     **{n: t.data_ptr for n, t in ts.items()})
    dev.synchronize()
    got = np.frombuffer(out.read_bytes(), np.uint32).astype(np.int64)
    np.testing.assert_array_equal(got[:rows], want(x, u, **c))
    assert (got[rows:] == 0xFFFFFFFF).all() and (ws.to_f32()[floats:] == guard).all()
