"""Token embedding, layer norm and the cross-entropy output layer on the device, against plain numpy
implementations in 64 bits, at the sizes and masks where they can go wrong; gradients also against
differences of the 64-bit forward pass.

Tolerances are rounding bounds.  u = 2^-24 is f32's unit roundoff, 2^-9 half of bf16's spacing below a
power of two relative to the value (RNE).  A sum of L terms in any order is off by at most L u times the
sum of the terms' magnitudes; where a kernel's longest chain of additions is shorter than the row, that
chain's length takes the place of L."""
import numpy as np
import pytest

from vernondsl_amd import _lib, kernels, rng
from vernondsl_amd.rhi import Queue, Tensor

pytestmark = pytest.mark.gpu
U, B = 2.0 ** -24, 2.0 ** -8  # B: bf16's largest relative rounding, 2^-9, twice (it is relative to the rounded value)


def bf16(x):
    """x (f32) rounded to bf16, as f32."""
    return rng.bf16_to_f32(rng.f32_to_bf16(np.asarray(x, np.float32)))


def put(dev, q, x, dtype):
    x = np.ascontiguousarray(x)
    if dtype == "bf16":
        return Tensor.from_numpy(dev, q, rng.f32_to_bf16(x.astype(np.float32)), "bf16")
    return Tensor.from_numpy(dev, q, x.astype({"f32": np.float32, "i32": np.int32}[dtype]), dtype)


def empty(dev, q, shape, dtype):
    """A tensor whose bytes are NaNs in every type: a kernel that leaves an element shows."""
    t = Tensor(dev, shape, dtype)
    if t.buffer.nbytes:
        t.buffer.write(q, np.full(t.buffer.nbytes, 0xFF, np.uint8))
    return t


def get(q, t):
    v = t.numpy(q)
    return (rng.bf16_to_f32(v) if t.dtype == _lib.BF16 else v).astype(np.float64)


def rounding(dtype, y):
    return (B if dtype == "bf16" else U) * np.abs(y)


def scratch(dev, q, nbytes):
    return empty(dev, q, (max(4, nbytes),), "i8") if nbytes else None


class Owner:
    """Frees the tensors of a test at its end."""

    def __init__(self, dev, q):
        self.dev, self.q, self.all = dev, q, []

    def put(self, x, dtype):
        return self.keep(put(self.dev, self.q, x, dtype))

    def empty(self, shape, dtype):
        return self.keep(empty(self.dev, self.q, shape, dtype))

    def scratch(self, nbytes):
        return self.keep(scratch(self.dev, self.q, nbytes))

    def keep(self, t):
        if t is not None:
            self.all.append(t)
        return t


@pytest.fixture
def own(dev, q):
    o = Owner(dev, q)
    yield o
    q.sync()
    for t in o.all:
        t.free()


# ---- embedding -----------------------------------------------------------------------------------
@pytest.mark.parametrize("n,dim,vocab", [(1, 1, 1), (1, 4096, 7), (3, 5, 11), (64, 1001, 50), (300, 64, 5003), (8, 4099, 9),
                                         (1000, 17, 3), (2, 40000, 4)])
@pytest.mark.parametrize("tt,ot", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16"), ("f32", "f32")])
def test_embedding_fwd(q, own, n, dim, vocab, tt, ot):
    r = np.random.default_rng(n + dim)
    table = r.standard_normal((vocab, dim)).astype(np.float32)
    ids = r.integers(-1, vocab + 1, n).astype(np.int32)
    ids[0] = vocab - 1
    if n > 2:
        ids[1], ids[2] = np.iinfo(np.int32).max, np.iinfo(np.int32).min
    scale = np.float32(np.sqrt(dim))
    out = own.empty((n, dim), ot)
    kernels.embedding_fwd(q, own.put(table, tt), own.put(ids, "i32"), out, scale=float(scale))
    held = bf16(table) if tt == "bf16" else table
    valid = (ids >= 0) & (ids < vocab)
    want = np.where(valid[:, None], held[np.where(valid, ids, 0)] * scale, np.float32(0))
    assert np.array_equal(get(q, out), (bf16(want) if ot == "bf16" else want).astype(np.float64))


def table_grad(ids, dy, vocab, scale):
    want, mag, terms = np.zeros((vocab, dy.shape[1])), np.zeros((vocab, dy.shape[1])), np.zeros(vocab)
    valid = (ids >= 0) & (ids < vocab)
    np.add.at(want, ids[valid], dy[valid])
    np.add.at(mag, ids[valid], np.abs(dy[valid]))
    np.add.at(terms, ids[valid], 1)
    return want * scale, mag * abs(scale), terms


def skewed(r, n, vocab):
    ids = (r.random(n) ** 3 * vocab).astype(np.int32)
    ids[r.random(n) < 0.05] = -1
    return ids


@pytest.mark.parametrize("n,dim,vocab,ids_of", [
    (1, 1, 1, "skewed"), (1, 8, 300, "skewed"), (5, 3, 2, "skewed"), (300, 1001, 503, "skewed"), (1000, 64, 5003, "skewed"),
    (4099, 20, 65, "skewed"), (257, 40, 4, "one"), (2500, 5, 1, "one"), (2500, 72, 700, "one"), (64, 16, 40, "none"),
    (0, 24, 33, "skewed"), (20000, 33, 3001, "skewed"), (20000, 12, 100000, "skewed"), (17000, 8, 30, "one"), (130, 4100, 10, "skewed"),
    (1024, 7, 300, "skewed"), (1025, 7, 300, "skewed"), (1024, 64, 3, "one"), (40000, 12, 3001, "skewed"), (33000, 5, 100000, "skewed"),
    (33000, 4, 200, "skewed"), (33000, 1, 17000000, "skewed"), (270000, 4, 50, "one"),
])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_embedding_bwd(q, own, n, dim, vocab, ids_of, dt):
    r = np.random.default_rng(n + dim + vocab)
    ids = {"skewed": lambda: skewed(r, n, vocab), "one": lambda: np.full(n, vocab // 2, np.int32),
           "none": lambda: np.where(np.arange(n) % 2, -1, vocab).astype(np.int32)}[ids_of]()
    dy = r.standard_normal((n, dim)).astype(np.float32)
    scale = 1.75
    ws = own.scratch(kernels.embedding_bwd_workspace_bytes(n, vocab, dim))
    tids, tdy = own.put(ids, "i32"), own.put(dy, dt)
    first = None
    for _ in range(2):
        out = own.empty((vocab, dim), "f32")
        kernels.embedding_bwd(q, tids, tdy, out, scale=scale, workspace=ws)
        got = out.numpy(q)
        assert first is None or np.array_equal(got, first), "another call gave other bits"
        first = got
    held = (bf16(dy) if dt == "bf16" else dy).astype(np.float64)
    want, mag, terms = table_grad(ids, held, vocab, scale)
    assert np.all(np.abs(first - want) <= (terms[:, None] + 1) * U * mag)


def test_embedding_grad_is_the_difference_of_the_lookup(q, own):
    """<dy, lookup(table + d) - lookup(table)> = <dtable, d>, the lookup being linear."""
    r = np.random.default_rng(5)
    n, dim, vocab, scale = 200, 33, 70, 3.0
    ids, dy, d = skewed(r, n, vocab), r.standard_normal((n, dim)), r.standard_normal((vocab, dim))
    valid = ids >= 0
    out = own.empty((vocab, dim), "f32")
    kernels.embedding_bwd(q, own.put(ids, "i32"), own.put(dy, "f32"), out, scale=scale,
                          workspace=own.scratch(kernels.embedding_bwd_workspace_bytes(n, vocab, dim)))
    dy = dy.astype(np.float32).astype(np.float64)
    moved = np.where(valid[:, None], d[np.where(valid, ids, 0)], 0.0) * scale
    _, mag, terms = table_grad(ids, dy, vocab, scale)
    tol = float(np.sum((terms[:, None] + 1) * U * mag * np.abs(d)))
    assert abs(float(np.sum(dy * moved)) - float(np.sum(get(q, out) * d))) <= tol


# ---- layer norm ----------------------------------------------------------------------------------
def depth(cols):
    """No kernel's chain of additions over a row is longer."""
    return 64 + cols / 1024


def norm(x, gamma, beta, eps):
    mean = x.mean(1, keepdims=True)
    d = x - mean
    var = (d * d).mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(var + eps)
    return d * rstd * gamma + beta, mean, d, var, rstd


def norm_tolerances(x, gamma, beta, eps):
    """Bounds of the errors of y (before its rounding), mean and rstd, the latter relative."""
    cols = x.shape[1]
    _, mean, d, var, rstd = norm(x, gamma, beta, eps)
    em = (depth(cols) + 2) * U * np.abs(x).mean(1, keepdims=True) + U * np.abs(mean)
    ed = em + 2 * U * np.abs(d)
    evar = (2 * np.abs(d) * ed + ed * ed).mean(1, keepdims=True) + (depth(cols) + 4) * U * var
    erstd = 0.5 * evar / (var + eps) + 4 * U
    ey = np.abs(gamma) * rstd * (ed + np.abs(d) * (erstd + 3 * U)) + 2 * U * np.abs(beta)
    return ey, em, erstd


def norm_input(r, rows, cols, dt, offset=0.5):
    x = (r.standard_normal((rows, cols)) * (0.5 + r.random(cols)) + offset + r.standard_normal(cols)).astype(np.float32)
    return bf16(x) if dt == "bf16" else x


SHAPES = [(1, 1), (1, 2), (5, 3), (3, 63), (7, 257), (300, 512), (2, 513), (9, 1001), (4, 1024), (3, 1025), (130, 2047), (2, 4096),
          (3, 4097), (5, 8192), (2, 8193), (3, 16384), (2, 16385), (3, 20003)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16"), ("f32", "f32")])
def test_layer_norm_fwd(q, own, rows, cols, xt, yt):
    r = np.random.default_rng(rows * 7 + cols)
    x = norm_input(r, rows, cols, xt)
    pt = "bf16" if (rows + cols) % 2 else "f32"
    gamma, beta = (r.standard_normal(cols).astype(np.float32) for _ in range(2))
    if pt == "bf16":
        gamma, beta = bf16(gamma), bf16(beta)
    eps = 1e-5
    y, mean, rstd = own.empty((rows, cols), yt), own.empty((rows,), "f32"), own.empty((rows,), "f32")
    kernels.layer_norm_fwd(q, own.put(x, xt), own.put(gamma, pt), own.put(beta, pt), y, mean=mean, rstd=rstd, eps=eps)
    x64, g64, b64 = (a.astype(np.float64) for a in (x, gamma, beta))
    want, wmean, _, _, wrstd = norm(x64, g64, b64, np.float64(np.float32(eps)))
    ey, em, er = norm_tolerances(x64, g64, b64, eps)
    assert np.all(np.abs(get(q, y) - want) <= ey + rounding(yt, np.abs(want) + ey))
    assert np.all(np.abs(get(q, mean) - wmean[:, 0]) <= em[:, 0])
    assert np.all(np.abs(get(q, rstd) - wrstd[:, 0]) <= (er * wrstd)[:, 0])


def test_layer_norm_fwd_without_parameters_and_in_place(q, own):
    r = np.random.default_rng(1)
    for cols in (100, 3000, 20000):
        x = norm_input(r, 6, cols, "f32")
        one, zero = np.ones(cols), np.zeros(cols)
        want = norm(x.astype(np.float64), one, zero, 1e-5)[0]
        ey, _, _ = norm_tolerances(x.astype(np.float64), one, zero, 1e-5)
        t = own.put(x, "f32")
        kernels.layer_norm_fwd(q, t, None, None, t)
        assert np.all(np.abs(get(q, t) - want) <= ey + rounding("f32", want))


def test_layer_norm_fwd_large_mean_constant_rows_and_nan(q, own):
    """A mean a thousand times the spread loses only what x itself does; a constant row gives beta; a NaN
    or infinity stays in its row."""
    r = np.random.default_rng(2)
    cols = 700
    x = r.standard_normal((6, cols)).astype(np.float32)
    x[0] += 1000.0
    x[1] = 2.5
    x[3, 17] = np.nan
    x[4, 5] = np.inf
    gamma, beta = (r.standard_normal(cols).astype(np.float32) for _ in range(2))
    y = own.empty(x.shape, "f32")
    kernels.layer_norm_fwd(q, own.put(x, "f32"), own.put(gamma, "f32"), own.put(beta, "f32"), y)
    got = get(q, y)
    ok = [0, 1, 2, 5]
    x64, g64, b64 = x[ok].astype(np.float64), gamma.astype(np.float64), beta.astype(np.float64)
    want = norm(x64, g64, b64, 1e-5)[0]
    ey, _, _ = norm_tolerances(x64, g64, b64, 1e-5)
    assert np.all(np.abs(got[ok] - want) <= ey + rounding("f32", want))
    assert np.array_equal(got[1], beta.astype(np.float64))
    assert np.isnan(got[3]).all() and np.isnan(got[4]).all()


def norm_grads(dy, x, gamma, mean, rstd):
    h = (x - mean) * rstd
    g = dy * gamma
    m1, m2 = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    return rstd * (g - m1 - h * m2), (dy * h).sum(0), dy.sum(0), h, g


@pytest.mark.parametrize("rows,cols", SHAPES + [(0, 40), (1500, 96), (1100, 4), (700, 5000)])
@pytest.mark.parametrize("xt,dyt,dxt", [("bf16", "bf16", "bf16"), ("f32", "f32", "f32"), ("bf16", "f32", "bf16"), ("f32", "bf16", "f32"),
                                        ("bf16", "bf16", "f32")])
def test_layer_norm_bwd(q, own, rows, cols, xt, dyt, dxt):
    r = np.random.default_rng(rows * 3 + cols)
    x, dy = norm_input(r, rows, cols, xt), r.standard_normal((rows, cols)).astype(np.float32)
    dy = bf16(dy) if dyt == "bf16" else dy
    gamma = r.standard_normal(cols).astype(np.float32)
    mean = x.astype(np.float64).mean(1).astype(np.float32)
    rstd = (1.0 / np.sqrt(x.astype(np.float64).var(1) + 1e-5)).astype(np.float32)
    dx, dg, db = own.empty((rows, cols), dxt), own.empty((cols,), "f32"), own.empty((cols,), "f32")
    ws = own.scratch(kernels.layer_norm_bwd_workspace_bytes(rows, cols))
    args = [own.put(dy, dyt), own.put(x, xt), own.put(gamma, "f32"), own.put(mean, "f32"), own.put(rstd, "f32")]
    kernels.layer_norm_bwd(q, *args, dx, dgamma=dg, dbeta=db, workspace=ws)
    x, dy, gamma, mean, rstd = (a.astype(np.float64) for a in (x, dy, gamma, mean, rstd))
    mean, rstd = mean[:, None], rstd[:, None]
    wdx, wdg, wdb, h, g = norm_grads(dy, x, gamma, mean, rstd)
    eh = 3 * U * np.abs(h)
    e1 = (depth(cols) + 2) * U * np.abs(g).mean(1, keepdims=True)
    e2 = (depth(cols) + 6) * U * np.abs(g * h).mean(1, keepdims=True)
    m1, m2 = np.abs(g).mean(1, keepdims=True), np.abs(g * h).mean(1, keepdims=True)
    e = rstd * (6 * U * (np.abs(g) + m1 + np.abs(h) * m2) + e1 + np.abs(h) * e2 + eh * m2)
    assert np.all(np.abs(get(q, dx) - wdx) <= e + rounding(dxt, np.abs(wdx) + e))
    # rows of a block in order, blocks and waves in order: chains of at most rows + 4 additions
    assert np.all(np.abs(get(q, dg) - wdg) <= ((rows + 8) * U * np.abs(dy * h)).sum(0))
    assert np.all(np.abs(get(q, db) - wdb) <= ((rows + 4) * U * np.abs(dy)).sum(0))
    again = own.empty((cols,), "f32")
    alone = own.empty((rows, cols), dxt)
    kernels.layer_norm_bwd(q, *args, alone, dgamma=again, workspace=ws)  # dbeta not wanted
    assert np.array_equal(again.numpy(q), dg.numpy(q)) and np.array_equal(alone.numpy(q), dx.numpy(q))
    kernels.layer_norm_bwd(q, *args, alone)  # neither: no workspace
    assert np.array_equal(alone.numpy(q), dx.numpy(q))


@pytest.mark.parametrize("rows,cols", [(1024, 9), (1025, 3), (1040, 700), (1030, 1500), (1030, 3001), (420, 5001), (240, 9000), (130, 16384),
                                       (1000, 2097), (2000, 513)])
@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_layer_norm_bwd_around_partial_rows(q, own, rows, cols, t):
    """Sizes on both sides of the one that takes partial rows, for each shape of a row."""
    test_layer_norm_bwd(q, own, rows, cols, t, t, t)


def test_layer_norm_bwd_in_place_equals_apart(q, own):
    """dx over dy's buffer takes partial rows where dx apart does not: the same dx, and sums within their bounds."""
    r = np.random.default_rng(21)
    rows, cols = 300, 1001
    x, dy = norm_input(r, rows, cols, "f32"), r.standard_normal((rows, cols)).astype(np.float32)
    mean = x.astype(np.float64).mean(1).astype(np.float32)
    rstd = (1.0 / np.sqrt(x.astype(np.float64).var(1) + 1e-5)).astype(np.float32)
    args = [own.put(x, "f32"), None, own.put(mean, "f32"), own.put(rstd, "f32")]
    ws = own.scratch(kernels.layer_norm_bwd_workspace_bytes(rows, cols))
    tdy, dx = own.put(dy, "f32"), own.empty((rows, cols), "f32")
    dg, db = ([own.empty((cols,), "f32") for _ in range(2)] for _ in range(2))
    kernels.layer_norm_bwd(q, tdy, *args, dx, dgamma=dg[0], dbeta=db[0], workspace=ws)
    kernels.layer_norm_bwd(q, tdy, *args, tdy, dgamma=dg[1], dbeta=db[1], workspace=ws)
    assert np.array_equal(dx.numpy(q), tdy.numpy(q))
    h = (x.astype(np.float64) - mean[:, None]) * rstd[:, None]
    assert np.all(np.abs(get(q, dg[0]) - get(q, dg[1])) <= 2 * ((rows + 8) * U * np.abs(dy * h)).sum(0))
    assert np.all(np.abs(get(q, db[0]) - get(q, db[1])) <= 2 * ((rows + 4) * U * np.abs(dy)).sum(0))


@pytest.mark.parametrize("cols", [90, 3000, 20000])
def test_layer_norm_bwd_in_place_and_against_differences(q, own, cols):
    """dx over dy's own buffer; dx, dgamma and dbeta against central differences of the 64-bit forward pass
    along a direction.  With a step t the differences are off by t^2 / 6 times a third derivative, which is
    measured by halving the step: what remains is below the change."""
    r = np.random.default_rng(cols)
    rows, eps = 5, 1e-5
    x = norm_input(r, rows, cols, "f32")
    dy, gamma, beta = (r.standard_normal(s).astype(np.float32) for s in ((rows, cols), cols, cols))
    mean = x.astype(np.float64).mean(1).astype(np.float32)
    rstd = (1.0 / np.sqrt(x.astype(np.float64).var(1) + eps)).astype(np.float32)
    tdy, dg, db = own.put(dy, "f32"), own.empty((cols,), "f32"), own.empty((cols,), "f32")
    kernels.layer_norm_bwd(q, tdy, own.put(x, "f32"), own.put(gamma, "f32"), own.put(mean, "f32"), own.put(rstd, "f32"), tdy, dgamma=dg,
                           dbeta=db, workspace=own.scratch(kernels.layer_norm_bwd_workspace_bytes(rows, cols)))
    x, dy, gamma, beta = (a.astype(np.float64) for a in (x, dy, gamma, beta))
    ux, ug, ub = r.standard_normal(x.shape), r.standard_normal(cols), r.standard_normal(cols)

    def loss(t):
        return float(np.sum(dy * norm(x + t * ux, gamma + t * ug, beta + t * ub, eps)[0]))

    d1, d2 = ((loss(t) - loss(-t)) / (2 * t) for t in (1e-4, 5e-5))
    dx = get(q, tdy)
    got = float(np.sum(dx * ux) + np.sum(get(q, dg) * ug) + np.sum(get(q, db) * ub))
    terms = np.sum(np.abs(dx * ux)) + np.sum(np.abs(dy) @ np.abs(ub)) + np.sum(np.abs(dy * norm(x, 1.0, 0.0, eps)[0]) @ np.abs(ug))
    # 64-bit differences at a step of 5e-5 cancel to 2^-52 / 5e-5 of the loss's terms
    noise = 2.0 ** -52 / 5e-5 * np.sum(np.abs(dy * norm(x, gamma, beta, eps)[0]))
    assert abs(got - d2) <= abs(d1 - d2) + (2 * depth(cols) + 16) * U * terms + noise


# ---- cross entropy -------------------------------------------------------------------------------
def xent(x, w, labels):
    """(loss, row losses, lse, G, rows that count) in 64 bits."""
    z = x @ w.T
    top = z.max(1, keepdims=True)
    lse = top[:, 0] + np.log(np.exp(z - top).sum(1))
    counts = (labels >= 0) & (labels < w.shape[0])
    at = np.where(counts, labels, 0)
    rows = np.arange(len(labels))
    each = np.where(counts, lse - z[rows, at], 0.0)
    g = np.exp(z - lse[:, None])
    g[rows, at] -= 1.0
    return each.sum() / max(1, counts.sum()), each, lse, g * counts[:, None], counts


def xent_input(r, n, dim, vocab, spread=2.0):
    w = bf16(r.standard_normal((vocab, dim)) * (spread / np.sqrt(dim)))
    labels = r.integers(0, vocab, n).astype(np.int32)
    x = r.standard_normal((n, dim))
    x += w[labels] / np.maximum(1e-20, np.linalg.norm(w[labels], axis=1, keepdims=True)) * (6 * r.random((n, 1)))
    if n > 1:
        labels[r.random(n) < 0.1] = -1
    if n > 4:
        labels[1], labels[2] = vocab, np.iinfo(np.int32).min
    return bf16(x), w, labels


def xent_tolerances(x, w, labels):
    """Bounds of the errors of lse, the rows' losses, and G's entries before and after their rounding."""
    dim, vocab = x.shape[1], w.shape[0]
    z = x @ w.T
    ez = (dim + 4) * U * (np.abs(x) @ np.abs(w).T) + 2 * U * np.abs(z)  # products in f32, then times log2 e
    # a row's sum: chains of vocab terms at most, each exp to 2 ulp and its f32 argument (to 2 u of z's size)
    el = ez.max(1) + 4 * U * np.abs(z).max(1) + (vocab + 16) * U + 4 * U * np.log(vocab + 1.0)
    _, each, lse, g, counts = xent(x, w, labels)
    el = el + 4 * U * np.abs(lse)
    p = np.exp(z - lse[:, None])
    eg = p * (ez + el[:, None] + 8 * U * (np.abs(z) + np.abs(lse)[:, None]) + 2.0 ** -12) + 2.0 ** -31 + 4 * U
    return el, np.where(counts, el + ez.max(1), 0.0), (eg + 2.0 ** -9 * 2 * (np.abs(g) + eg)) * counts[:, None]


def check_xent(q, own, x, w, labels, piece=0, gt="f32", grad_scale=1.0):
    n, dim = x.shape
    vocab = w.shape[0]
    tx, tw, tl = own.put(x, "bf16"), own.put(w, "bf16"), own.put(labels, "i32")
    loss, each, lse = own.empty((1,), "f32"), own.empty((n,), "f32"), own.empty((n,), "f32")
    dx, dw = own.empty((n, dim), gt), own.empty((vocab, dim), gt)
    ws = own.scratch(kernels.linear_xent_workspace_bytes(n, vocab, dim, piece=piece))
    kernels.linear_xent_fwd_bwd(q, tx, tw, tl, loss, dx, dw, row_loss=each, lse=lse, piece=piece, grad_scale=grad_scale, workspace=ws)
    x, w = x.astype(np.float64), w.astype(np.float64)
    wloss, weach, wlse, g, counts = xent(x, w, labels)
    el, ee, eg = xent_tolerances(x, w, labels)
    inv = grad_scale / max(1, counts.sum())
    assert np.all(np.abs(get(q, lse) - wlse) <= el)
    assert np.all(np.abs(get(q, each) - weach) <= ee)
    assert abs(get(q, loss)[0] - wloss) <= ee.sum() / max(1, counts.sum()) + 2 * U * abs(wloss)
    for got, want, tol in ((dx, g @ w, eg @ np.abs(w) + (vocab + 8) * U * (np.abs(g) @ np.abs(w))),
                           (dw, g.T @ x, eg.T @ np.abs(x) + (n + 8) * U * (np.abs(g).T @ np.abs(x)))):
        want, tol = want * inv, tol * abs(inv)
        assert np.all(np.abs(get(q, got) - want) <= tol + rounding(gt, np.abs(want) + tol) + 1e-45)
    return [t.numpy(q) for t in (loss, each, lse, dx, dw)]


@pytest.mark.parametrize("n,dim,vocab,piece", [
    (1, 8, 1, 0), (1, 8, 2, 0), (1, 9, 300, 0), (3, 40, 33, 0), (16, 512, 1003, 0), (65, 100, 700, 256), (130, 64, 2048, 512),
    (300, 250, 1500, 300), (64, 256, 1024, 0), (257, 264, 515, 256), (2, 1000, 3001, 1000), (128, 128, 4096, 1024), (33, 33, 65, 0),
    (256, 256, 512, 0), (512, 512, 768, 256),
])
@pytest.mark.parametrize("gt", ["f32", "bf16"])
def test_linear_xent(q, own, n, dim, vocab, piece, gt):
    r = np.random.default_rng(n + dim + vocab)
    check_xent(q, own, *xent_input(r, n, dim, vocab), piece=piece, gt=gt)


def test_linear_xent_large_tiles(q, own):
    """Sizes that take the large tiles, ragged and whole."""
    r = np.random.default_rng(8)
    check_xent(q, own, *xent_input(r, 700, 72, 6150), gt="bf16")
    check_xent(q, own, *xent_input(r, 512, 256, 8192), piece=4096)
    check_xent(q, own, *xent_input(r, 1000, 512, 5003), piece=2048)


@pytest.mark.parametrize("n,dim,vocab,piece,gt", [(2100, 64, 5501, 0, "bf16"), (2048, 128, 6144, 0, "f32"), (2305, 192, 11000, 5632, "f32"),
                                                  (520, 320, 16500, 0, "bf16"), (2081, 64, 11264, 5632, "bf16")])
def test_linear_xent_256_tiles(q, own, n, dim, vocab, piece, gt):
    """Sizes that take the tiles of 256 x 256: ragged rows, vocabularies and last pieces, one stage of dim and
    several, rows that are and are not a multiple of a stage."""
    check_xent(q, own, *xent_input(np.random.default_rng(n), n, dim, vocab), piece=piece, gt=gt)


def test_linear_xent_grad_scale_and_calls_agree(q, own):
    r = np.random.default_rng(9)
    x, w, labels = xent_input(r, 70, 96, 900)
    a = check_xent(q, own, x, w, labels, grad_scale=256.0)
    b = check_xent(q, own, x, w, labels, grad_scale=256.0)
    assert all(np.array_equal(s, t) for s, t in zip(a, b)), "another call gave other bits"
    loss, each, lse = (own.empty(s, "f32") for s in ((1,), (70,), (70,)))
    kernels.linear_xent_fwd(q, own.put(x, "bf16"), own.put(w, "bf16"), own.put(labels, "i32"), loss, row_loss=each, lse=lse,
                            workspace=own.scratch(kernels.linear_xent_workspace_bytes(70, 900, 96, backward=False)))
    for t, v in zip((loss, each, lse), a):
        assert np.array_equal(t.numpy(q), v), "the loss alone differs from the loss with its gradients"


def test_linear_xent_no_row_counts(q, own):
    r = np.random.default_rng(10)
    x, w, _ = xent_input(r, 20, 64, 300)
    out = check_xent(q, own, x, w, np.where(np.arange(20) % 2, -1, 300).astype(np.int32))
    assert out[0][0] == 0 and not out[1].any() and not out[3].any() and not out[4].any()


def test_linear_xent_no_rows(q, own):
    w = own.put(np.ones((40, 9)), "bf16")
    for gt in ("f32", "bf16"):
        dw, loss = own.empty((40, 9), gt), own.empty((1,), "f32")
        kernels.linear_xent_fwd_bwd(q, own.empty((0, 9), "bf16"), w, own.empty((0,), "i32"), loss, own.empty((0, 9), gt), dw,
                                    workspace=own.scratch(kernels.linear_xent_workspace_bytes(0, 40, 9)))
        assert not dw.numpy(q).any() and loss.numpy(q)[0] == 0


def test_linear_xent_extreme_logits(q, own):
    """Logits of thousands: certain rows whose other probabilities underflow, and certain wrong ones."""
    r = np.random.default_rng(11)
    x, w, labels = xent_input(r, 40, 64, 500)
    x = bf16(x * 600.0)
    check_xent(q, own, x, w, labels, piece=256)


def test_linear_xent_nan_and_inf_stay_in_their_rows(q, own):
    r = np.random.default_rng(12)
    x, w, labels = xent_input(r, 50, 64, 700)
    labels[:] = np.arange(50) % 700
    x[7, 3], x[9, 0] = np.nan, np.inf
    tx, tw, tl = own.put(x, "bf16"), own.put(w, "bf16"), own.put(labels, "i32")
    loss, lse, dx, dw = (own.empty(s, "f32") for s in ((1,), (50,), (50, 64), (700, 64)))
    kernels.linear_xent_fwd_bwd(q, tx, tw, tl, loss, dx, dw, lse=lse, piece=256,
                                workspace=own.scratch(kernels.linear_xent_workspace_bytes(50, 700, 64, piece=256)))
    bad = np.isin(np.arange(50), (7, 9))
    assert np.array_equal(np.isnan(lse.numpy(q)), bad) and np.isnan(loss.numpy(q)[0])
    assert np.array_equal(np.isnan(dx.numpy(q)).all(1), bad) and np.array_equal(np.isnan(dx.numpy(q)).any(1), bad)


def test_linear_xent_row_of_minus_infinity(q, own):
    """A row whose logits all are -inf has no softmax: NaN in its loss and its gradient, whole or in pieces, and no
    other row's."""
    r = np.random.default_rng(14)
    x, w, labels = xent_input(r, 50, 64, 700)
    labels[:] = np.arange(50) % 700
    w[:, 5] = np.abs(w[:, 5]) + 1.0
    x[7, 5] = -np.inf
    tx, tw, tl = own.put(x, "bf16"), own.put(bf16(w), "bf16"), own.put(labels, "i32")
    bad = np.arange(50) == 7
    for piece in (0, 256):
        loss, each, dx, dw = (own.empty(s, "f32") for s in ((1,), (50,), (50, 64), (700, 64)))
        kernels.linear_xent_fwd_bwd(q, tx, tw, tl, loss, dx, dw, row_loss=each, piece=piece,
                                    workspace=own.scratch(kernels.linear_xent_workspace_bytes(50, 700, 64, piece=piece)))
        assert np.array_equal(np.isnan(each.numpy(q)), bad)
        assert np.array_equal(np.isnan(dx.numpy(q)).all(1), bad) and np.array_equal(np.isnan(dx.numpy(q)).any(1), bad)


def test_linear_xent_piece_of_any_size(q, own):
    r = np.random.default_rng(15)
    x, w, labels = xent_input(r, 20, 24, 300)
    whole = check_xent(q, own, x, w, labels)
    for piece in (300, 301, 2 ** 62, 2 ** 63 - 1):
        for a, b in zip(whole, check_xent(q, own, x, w, labels, piece=piece)):
            assert np.array_equal(a, b)


# gradients on 256 x 256 tiles, in splits: smaller tiles for the logits; f32; pieces; ragged rows and columns
@pytest.mark.parametrize("n,dim,vocab,piece,gt", [(500, 1600, 16500, 0, "bf16"), (2048, 1152, 6144, 0, "f32"), (2305, 1024, 11000, 5632, "bf16"),
                                                  (1100, 2112, 5701, 0, "bf16"), (2100, 1001, 6300, 0, "bf16"), (2100, 1003, 6300, 0, "f32"),
                                                  (2100, 1000, 6300, 3328, "bf16")])
def test_linear_xent_gradients_on_256_tiles(q, own, n, dim, vocab, piece, gt):
    check_xent(q, own, *xent_input(np.random.default_rng(n), n, dim, vocab), piece=piece, gt=gt)


# smaller tiles in pieces: enough rows that the pieces are not raised (4 MiB); ragged last pieces, dims that are copied
@pytest.mark.parametrize("n,dim,vocab,piece,gt", [(8300, 64, 700, 256, "bf16"), (4200, 71, 1300, 512, "f32"), (4200, 72, 1030, 512, "bf16"),
                                                  (9001, 16, 513, 256, "f32")])
def test_linear_xent_pieces_on_smaller_tiles(q, own, n, dim, vocab, piece, gt):
    few, whole = (kernels.linear_xent_workspace_bytes(n, vocab, dim, piece=p) for p in (piece, 0))
    assert few != whole
    check_xent(q, own, *xent_input(np.random.default_rng(n), n, dim, vocab), piece=piece, gt=gt)


def test_linear_xent_rows_without_softmax_in_pieces(q, own):
    """NaN, +inf and rows of -inf alone in a call of three pieces: their own losses and gradients are NaN, no other's."""
    n, dim, vocab = 8300, 64, 700
    r = np.random.default_rng(17)
    x, w, labels = xent_input(r, n, dim, vocab)
    labels[:] = np.arange(n) % vocab
    w[:, 5] = np.abs(w[:, 5]) + 1.0
    x[7, 5], x[8, 5], x[8000, 3] = -np.inf, np.inf, np.nan
    tx, tw, tl = own.put(x, "bf16"), own.put(bf16(w), "bf16"), own.put(labels, "i32")
    loss, each, dx, dw = (own.empty(s, "f32") for s in ((1,), (n,), (n, dim), (vocab, dim)))
    kernels.linear_xent_fwd_bwd(q, tx, tw, tl, loss, dx, dw, row_loss=each, piece=256,
                                workspace=own.scratch(kernels.linear_xent_workspace_bytes(n, vocab, dim, piece=256)))
    bad = np.isin(np.arange(n), (7, 8, 8000))
    assert np.array_equal(np.isnan(each.numpy(q)), bad)
    assert np.array_equal(np.isnan(dx.numpy(q)).all(1), bad) and np.array_equal(np.isnan(dx.numpy(q)).any(1), bad)


# long sums for the weights' gradient in few tiles
@pytest.mark.parametrize("n,dim,vocab,piece", [(2000, 72, 300, 0), (1500, 71, 130, 0), (1100, 64, 700, 256)])
def test_linear_xent_many_rows_few_logits(q, own, n, dim, vocab, piece):
    check_xent(q, own, *xent_input(np.random.default_rng(n), n, dim, vocab), piece=piece)


def test_linear_xent_rows_past_a_launch(q, own):
    """More rows than one dimension of a launch holds blocks for.  Rows repeat with a period, so 64 bits of a period give
    every row's loss and gradient."""
    r = np.random.default_rng(16)
    period, dim, vocab = 1024, 8, 24
    n = (1 << 24) + period
    x, w, labels = xent_input(r, period, dim, vocab)
    tx, tw, tl = own.put(np.tile(x, (n // period, 1)), "bf16"), own.put(w, "bf16"), own.put(np.tile(labels, n // period), "i32")
    loss, each, dx, dw = own.empty((1,), "f32"), own.empty((n,), "f32"), own.empty((n, dim), "f32"), own.empty((vocab, dim), "f32")
    kernels.linear_xent_fwd_bwd(q, tx, tw, tl, loss, dx, dw, row_loss=each,
                                workspace=own.scratch(kernels.linear_xent_workspace_bytes(n, vocab, dim)))
    x, w = x.astype(np.float64), w.astype(np.float64)
    wloss, weach, _, g, counts = xent(x, w, labels)
    _, ee, eg = xent_tolerances(x, w, labels)
    inv = 1.0 / (counts.sum() * (n // period))
    assert np.all(np.abs(each.numpy(q).reshape(-1, period) - weach) <= ee)
    assert abs(loss.numpy(q)[0] - wloss) <= ee.sum() / counts.sum() + 2 * U * abs(wloss)
    tol = (eg @ np.abs(w) + (vocab + 8) * U * (np.abs(g) @ np.abs(w))) * inv
    want = g @ w * inv
    assert np.all(np.abs(dx.numpy(q).reshape(-1, period, dim) - want) <= tol + U * (np.abs(want) + tol))


def test_linear_xent_against_differences(q, own):
    """The gradients against central differences of the 64-bit loss along a direction (see the layer norm's)."""
    r = np.random.default_rng(13)
    x, w, labels = xent_input(r, 60, 80, 400)
    _, _, _, dx, dw = check_xent(q, own, x, w, labels, piece=256)
    x, w = x.astype(np.float64), w.astype(np.float64)
    ux, uw = r.standard_normal(x.shape), r.standard_normal(w.shape) / np.sqrt(80)

    def loss(t):
        return float(xent(x + t * ux, w + t * uw, labels)[0])

    d1, d2 = ((loss(t) - loss(-t)) / (2 * t) for t in (1e-4, 5e-5))
    got = float(np.sum(dx.astype(np.float64) * ux) + np.sum(dw.astype(np.float64) * uw))
    _, _, eg = xent_tolerances(x, w, labels)
    inv = 1.0 / ((labels >= 0) & (labels < 400)).sum()
    _, _, _, g, _ = xent(x, w, labels)
    tol = inv * (np.sum((eg + 512 * U * np.abs(g)) @ np.abs(w) * np.abs(ux)) + np.sum((eg + 512 * U * np.abs(g)).T @ np.abs(x) * np.abs(uw)))
    assert abs(got - d2) <= abs(d1 - d2) + tol + 2.0 ** -52 / 5e-5 * abs(loss(0.0))


# ---- recordings, queues, refusals ----------------------------------------------------------------
def test_recorded_and_on_another_queue(dev, q, own):
    """All the operators recorded into one graph: each replay, with eager work on another queue between,
    gives the eager run's bits."""
    r = np.random.default_rng(14)
    n, dim, vocab = 90, 72, 600
    table = bf16(r.standard_normal((vocab, dim)))
    ids = skewed(r, n, vocab)
    labels = np.roll(ids, -1)
    tt, ti, tl = own.put(table, "bf16"), own.put(ids, "i32"), own.put(labels, "i32")
    gamma, beta = own.put(np.ones(dim), "f32"), own.put(np.zeros(dim), "f32")
    names = {"h": ((n, dim), "f32"), "y": ((n, dim), "bf16"), "mean": ((n,), "f32"), "rstd": ((n,), "f32"), "loss": ((1,), "f32"),
             "dy": ((n, dim), "f32"), "dw": ((vocab, dim), "f32"), "dh": ((n, dim), "f32"), "dg": ((dim,), "f32"), "db": ((dim,), "f32"),
             "dtable": ((vocab, dim), "f32")}
    o = {k: own.empty(*v) for k, v in names.items()}
    w1 = own.scratch(kernels.linear_xent_workspace_bytes(n, vocab, dim, piece=256))
    w2 = own.scratch(kernels.layer_norm_bwd_workspace_bytes(n, dim))
    w3 = own.scratch(kernels.embedding_bwd_workspace_bytes(n, vocab, dim))

    def step(queue):
        kernels.embedding_fwd(queue, tt, ti, o["h"], scale=8.0)
        kernels.layer_norm_fwd(queue, o["h"], gamma, beta, o["y"], mean=o["mean"], rstd=o["rstd"])
        kernels.linear_xent_fwd_bwd(queue, o["y"], tt, tl, o["loss"], o["dy"], o["dw"], piece=256, workspace=w1)
        kernels.layer_norm_bwd(queue, o["dy"], o["h"], gamma, o["mean"], o["rstd"], o["dh"], dgamma=o["dg"], dbeta=o["db"], workspace=w2)
        kernels.embedding_bwd(queue, ti, o["dh"], o["dtable"], scale=8.0, workspace=w3)

    step(q)
    want = {k: t.numpy(q) for k, t in o.items()}
    other = Queue(dev)
    with q.capture() as rec:
        step(q)
    for k in range(3):
        for t in o.values():
            t.buffer.fill_u32(q, 0x7FC07FC0)
        q.sync()
        if k == 1:  # an eager run on a queue of its own, then poisoned again
            step(other)
            assert all(np.array_equal(t.numpy(other), want[name]) for name, t in o.items())
            for t in o.values():
                t.buffer.fill_u32(other, 0x7FC07FC0)
            other.sync()
        rec.graph.launch(q)
        for name, t in o.items():
            assert np.array_equal(t.numpy(q), want[name]), f"replay {k} differs in {name}"
    rec.graph.destroy()
    other.destroy()


def test_refusals(dev, q, own):
    t = {k: own.empty(*v) for k, v in {"x": ((4, 16), "bf16"), "f": ((4, 16), "f32"), "w": ((9, 16), "bf16"), "ids": ((4,), "i32"),
                                       "dw": ((9, 16), "f32"), "one": ((1,), "f32"), "row": ((4,), "f32"), "col": ((16,), "f32"),
                                       "small": ((4,), "i8"), "bytes": ((4, 16), "i8"), "thin": ((4, 4), "bf16"), "thinw": ((9, 4), "bf16"),
                                       "thinf": ((4, 4), "f32"), "thindw": ((9, 4), "f32")}.items()}
    ro = own.keep(Tensor(dev, (4, 16), "f32", "uniform_constant"))
    ws = own.scratch(1 << 16)
    many = own.empty((1025,), "i32"), own.empty((1025, 16), "f32")

    def status(fn, *a, **kw):
        with pytest.raises(_lib.VdslError) as e:
            fn(q, *a, **kw)
        return e.value.status

    # shapes and types that Python sees
    for fn, a in ((kernels.embedding_fwd, (t["w"], t["ids"], t["dw"])), (kernels.embedding_fwd, (t["w"], t["row"], t["f"])),
                  (kernels.embedding_bwd, (t["ids"], t["dw"], t["dw"])), (kernels.embedding_bwd, (t["ids"], t["f"], t["w"])),
                  (kernels.layer_norm_fwd, (t["x"], t["row"], None, t["f"])), (kernels.layer_norm_fwd, (t["x"], None, None, t["dw"])),
                  (kernels.layer_norm_bwd, (t["f"], t["x"], None, t["row"], t["col"], t["f"])),
                  (kernels.linear_xent_fwd, (t["f"], t["w"], t["ids"], t["one"])),
                  (kernels.linear_xent_fwd, (t["x"], t["w"], t["row"], t["one"])),
                  (kernels.linear_xent_fwd_bwd, (t["x"], t["w"], t["ids"], t["one"], t["dw"], t["dw"]))):
        with pytest.raises(ValueError):
            fn(q, *a)
    # what the C ABI refuses
    unsupported, invalid, shape, handle = -5, -1, -7, -2
    assert status(kernels.embedding_fwd, t["w"], t["ids"], t["bytes"]) == unsupported
    assert status(kernels.embedding_fwd, t["w"], t["ids"], ro) == invalid
    assert status(kernels.embedding_bwd, t["ids"], t["bytes"], t["dw"], workspace=ws) == unsupported
    assert status(kernels.embedding_bwd, *many, t["dw"]) == handle  # (1024 positions need no workspace)
    assert status(kernels.embedding_bwd, *many, t["dw"], workspace=t["small"]) == shape
    assert status(kernels.layer_norm_fwd, t["x"], None, None, t["bytes"]) == unsupported
    assert status(kernels.layer_norm_fwd, t["x"], None, None, t["f"], eps=-1.0) == invalid
    assert status(kernels.layer_norm_fwd, t["x"], None, None, t["f"], eps=float("nan")) == invalid
    assert status(kernels.layer_norm_fwd, t["x"], None, None, ro) == invalid
    bwd = (t["f"], t["x"], None, t["row"], t["row"])
    assert status(kernels.layer_norm_bwd, *bwd, t["bytes"]) == unsupported
    assert status(kernels.layer_norm_bwd, *bwd, t["x"]) == invalid
    assert status(kernels.layer_norm_bwd, *bwd, ro) == invalid
    assert status(kernels.layer_norm_bwd, *bwd, t["f"], dgamma=t["col"]) == handle
    assert status(kernels.layer_norm_bwd, *bwd, t["f"], dgamma=t["col"], workspace=t["small"]) == shape
    assert status(kernels.linear_xent_fwd, t["x"], t["w"], t["ids"], t["one"]) == handle
    assert status(kernels.linear_xent_fwd, t["x"], t["w"], t["ids"], t["one"], workspace=t["small"]) == shape
    assert status(kernels.linear_xent_fwd, t["thin"], t["thinw"], t["ids"], t["one"], workspace=ws) == unsupported
    xb = (t["x"], t["w"], t["ids"], t["one"])
    assert status(kernels.linear_xent_fwd_bwd, *xb, t["bytes"], t["dw"], workspace=ws) == unsupported
    assert status(kernels.linear_xent_fwd_bwd, *xb, t["f"], t["w"], workspace=ws) == invalid
    assert status(kernels.linear_xent_fwd_bwd, *xb, t["f"], t["dw"], piece=-1, workspace=ws) == invalid
    q.sync()
