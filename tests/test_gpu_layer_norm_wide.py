"""The gradients of a layer norm's gain and offset over rows wider than any that are held in registers: sums over thousands
of rows whose error does not grow with their number."""
import numpy as np
import pytest

from test_gpu_tokens import U, Owner
from vernondsl_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.fixture
def own(dev, q):
    o = Owner(dev, q)
    yield o
    q.sync()
    for t in o.all:
        t.free()


@pytest.mark.parametrize("rows,cols", [(3500, 65537), (130, 20003)])
def test_sums_over_many_rows(q, own, rows, cols):
    """All rows alike, with mean 0 and rstd 1, so dbeta is rows * dy and dgamma rows * dy^2, all terms positive: in one f32 sum
    every addition would be rounded the same way and the error grow with its length.  At most 64 terms are added in f32
    (64 u of the sum, with a term's own rounding), then in f64, and rounded to f32 twice."""
    row = (1.0 + np.random.default_rng(rows).random(cols)).astype(np.float32)
    both = own.put(np.broadcast_to(row, (rows, cols)), "f32")
    mean, rstd = own.put(np.zeros(rows), "f32"), own.put(np.ones(rows), "f32")
    dx, dg, db = own.empty((rows, cols), "bf16"), own.empty((cols,), "f32"), own.empty((cols,), "f32")
    kernels.layer_norm_bwd(q, both, both, None, mean, rstd, dx, dgamma=dg, dbeta=db,
                           workspace=own.scratch(kernels.layer_norm_bwd_workspace_bytes(rows, cols)))
    row = row.astype(np.float64)
    for got, want in ((dg, rows * row * row), (db, rows * row)):
        assert np.abs(got.numpy(q) / want - 1.0).max() <= 66 * U
