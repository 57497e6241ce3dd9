"""The token operators refuse outputs and workspaces that share a buffer with another operand: blocks of one launch write
them while others still read, or two results would take one place.  What may share one still runs."""
import numpy as np
import pytest

from test_gpu_tokens import Owner
from vernondsl_amd import _lib, kernels

pytestmark = pytest.mark.gpu
INVALID = -1


@pytest.fixture
def own(dev, q):
    o = Owner(dev, q)
    yield o
    q.sync()
    for t in o.all:
        t.free()


def refused(fn, *a, **kw):
    with pytest.raises(_lib.VdslError) as e:
        fn(*a, **kw)
    assert e.value.status == INVALID, str(e.value)


def test_layer_norm(q, own):
    n = 16  # rows and columns alike, so that one buffer fits every place
    sq = {k: own.put(np.random.default_rng(1).standard_normal((n, n)), "f32") for k in ("x", "dy", "dx", "y")}
    v = {k: own.put(np.ones(n), "f32") for k in ("gamma", "beta", "mean", "rstd", "dg", "db")}
    ws = own.scratch(kernels.layer_norm_bwd_workspace_bytes(n, n))

    def fwd(x=sq["x"], gamma=v["gamma"], beta=v["beta"], y=sq["y"], mean=v["mean"], rstd=v["rstd"]):
        kernels.layer_norm_fwd(q, x, gamma, beta, y, mean=mean, rstd=rstd)

    def bwd(dx=sq["dx"], dg=v["dg"], db=v["db"], ws=ws, dy=sq["dy"]):
        kernels.layer_norm_bwd(q, dy, sq["x"], v["gamma"], v["mean"], v["rstd"], dx, dgamma=dg, dbeta=db, workspace=ws)

    for kw in ({"mean": v["rstd"]}, {"mean": v["gamma"]}, {"rstd": v["beta"]}):
        refused(fwd, **kw)
    for kw in ({"dg": v["db"]}, {"dg": v["gamma"]}, {"db": v["mean"]}, {"db": v["rstd"]}, {"dx": sq["x"]}, {"ws": sq["dy"]}, {"ws": sq["x"]},
               {"ws": sq["dx"]}):
        refused(bwd, **kw)
    fwd()
    fwd(y=sq["x"])            # in place
    fwd(beta=v["gamma"])      # inputs may share
    bwd()
    bwd(dx=sq["dy"])          # in place
    bwd(dg=None, db=None, ws=sq["dy"])  # not used, not looked at
    q.sync()


def test_embedding(q, own):
    ids = own.put(np.zeros(1100), "i32")
    table, out, dy = own.put(np.ones((1100, 8)), "f32"), own.empty((1100, 8), "f32"), own.put(np.ones((1100, 8)), "f32")
    need = kernels.embedding_bwd_workspace_bytes(1100, 1100, 8)
    ws = own.scratch(need)
    assert need <= out.buffer.nbytes
    refused(kernels.embedding_fwd, q, table, ids, table)
    refused(kernels.embedding_bwd, q, ids, dy, dy, workspace=ws)
    refused(kernels.embedding_bwd, q, ids, dy, out, workspace=out)
    refused(kernels.embedding_bwd, q, ids, dy, out, workspace=dy)
    kernels.embedding_fwd(q, table, ids, out)
    kernels.embedding_bwd(q, ids, dy, out, workspace=ws)
    q.sync()


def test_linear_xent(q, own):
    n = 16
    x, w, labels = own.put(np.ones((n, n)), "bf16"), own.put(np.ones((n, n)), "bf16"), own.put(np.arange(n), "i32")
    loss, each, lse = own.empty((1,), "f32"), own.empty((n,), "f32"), own.empty((n,), "f32")
    dx, dw = own.empty((n, n), "bf16"), own.empty((n, n), "bf16")
    ws = own.scratch(kernels.linear_xent_workspace_bytes(n, n, n))

    def run(x=x, w=w, dx=dx, dw=dw, each=each, lse=lse, ws=ws):
        kernels.linear_xent_fwd_bwd(q, x, w, labels, loss, dx, dw, row_loss=each, lse=lse, workspace=ws)

    for kw in ({"dx": x}, {"dx": w}, {"dw": x}, {"dw": w}, {"dx": dw}, {"each": lse}):
        refused(run, **kw)
    refused(kernels.linear_xent_fwd, q, x, w, labels, loss, row_loss=lse, lse=lse, workspace=ws)
    run()
    run(w=x)  # inputs may share
    q.sync()
