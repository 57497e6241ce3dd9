"""The cross entropy's gradients with the vocabulary in several pieces, each call shown to have them, against numpy in 64
bits; norm-wise, beside the element-wise bounds of test_gpu_tokens.py.

Norm-wise bound.  The products take G rounded to bf16, which moves every entry by at most 2^-8 of itself (half of the
spacing of 8 significant bits), so G by 2^-8 |G| in Frobenius norm.  Before that p = exp(z - lse) is off by less than
2^-12 p: 1.7e-4 through its code, and the f32 error of these inputs' logits (|z| < 40: 2^-18 octaves a rounding) far
below that; a label's entry p - 1 by 2^-12 in all.  The products accumulate in f32: L terms, at most L u of the sum
of their magnitudes.  A matrix E moves E w by at most |E| times w's largest singular value; the result's own
rounding moves it by 2^-8 (bf16) or u (f32) of its norm."""
import numpy as np
import pytest

from test_gpu_tokens import U, Owner, bf16, check_xent, get, xent, xent_input
from test_linear_xent_plan import WIDE, plan
from vernondsl_amd import graph, kernels, rng
from vernondsl_amd.rhi import Queue

pytestmark = pytest.mark.gpu


@pytest.fixture
def own(dev, q):
    o = Owner(dev, q)
    yield o
    q.sync()
    for t in o.all:
        t.free()


def largest_singular_value(a):
    """Power iteration; 128 steps from a random start come within 0.87 ln(dim) / 127 of its square whatever the spectrum
    (Kuczynski and Wozniakowski, 1992), which the factor covers."""
    v = np.random.default_rng(0).standard_normal(a.shape[1])
    for _ in range(128):
        v = a.T @ (a @ (v / np.linalg.norm(v)))
    return 1.1 * np.sqrt(np.linalg.norm(v))


class Reference:
    """Loss and gradients in 64 bits, and how far a call's may be off in norm."""

    def __init__(self, x, w, labels):
        x, w = x.astype(np.float64), w.astype(np.float64)
        self.loss, _, _, g, counts = xent(x, w, labels)
        inv = 1.0 / max(1, counts.sum())
        self.dx, self.dw = inv * (g @ w), inv * (g.T @ x)
        off = 2.0 ** -8 * np.linalg.norm(g) + 2.0 ** -12 * (np.linalg.norm(np.maximum(g, 0.0)) + np.sqrt(counts.sum()))
        self.tol_dx, self.tol_dw = (inv * (off * largest_singular_value(f) + f.shape[0] * U * np.linalg.norm(g) * np.linalg.norm(f))
                                    for f in (w, x))

    def check(self, q, loss, dx, dw, gt):
        assert abs(float(loss.numpy(q)[0]) - self.loss) <= 1e-4 * max(1.0, abs(self.loss))
        for t, want, tol in ((dx, self.dx, self.tol_dx), (dw, self.dw, self.tol_dw)):
            tol += (2.0 ** -8 if gt == "bf16" else U) * np.linalg.norm(want)
            assert np.linalg.norm(get(q, t) - want) <= tol


def run(q, own, x, w, labels, piece, gt, workspace=None):
    """One call's loss, dx and dw."""
    n, dim = x.shape
    vocab = w.shape[0]
    out = own.empty((1,), "f32"), own.empty((n, dim), gt), own.empty((vocab, dim), gt)
    ws = workspace or own.scratch(kernels.linear_xent_workspace_bytes(n, vocab, dim, piece=piece))
    kernels.linear_xent_fwd_bwd(q, own.put(x, "bf16"), own.put(w, "bf16"), own.put(labels, "i32"), *out, piece=piece, workspace=ws)
    return out


def test_short_last_piece_with_splits(q, own):
    """The last piece, worked on first, is 8 columns: it fills one of the two splits of dx's sum."""
    n, dim, vocab, piece = 1024, 5504, 18440, 2304
    p = plan(n, vocab, dim, piece)
    assert p["grads"] == WIDE and p["pieces"] == 9 and p["last"] == 8 and (p["splits"], p["last_splits"]) == (2, 1)
    data = xent_input(np.random.default_rng(n), n, dim, vocab)
    ref = Reference(*data)
    for gt in ("f32", "bf16"):
        ref.check(q, *run(q, own, *data, piece, gt), gt)


# every tile; whole, and in pieces of it: ragged last pieces, dims that are copied, rows that fill no stage
@pytest.mark.parametrize("n,dim,vocab,piece,pieces,gt", [
    (16, 512, 1003, 0, 1, "bf16"), (300, 1000, 5003, 0, 1, "bf16"), (700, 72, 6150, 0, 1, "f32"), (2305, 1024, 11000, 0, 1, "bf16"),
    (8300, 64, 700, 256, 3, "f32"), (8300, 72, 513, 256, 3, "bf16"), (4200, 71, 2600, 512, 6, "bf16"), (2305, 1024, 11000, 5632, 2, "f32"),
    (2305, 1024, 11000, 1024, 11, "bf16"), (3001, 1001, 6300, 1024, 7, "f32"), (8193, 520, 3000, 1024, 3, "bf16")])
def test_gradients_in_norm(q, own, n, dim, vocab, piece, pieces, gt):
    assert plan(n, vocab, dim, piece)["pieces"] == pieces
    data = xent_input(np.random.default_rng(n + vocab), n, dim, vocab)
    Reference(*data).check(q, *run(q, own, *data, piece, gt), gt)


def test_extreme_logits_in_pieces(q, own):
    """Logits of thousands: certain rows whose other probabilities underflow, and certain wrong ones."""
    n, dim, vocab, piece = 8300, 64, 700, 256
    assert plan(n, vocab, dim, piece)["pieces"] == 3
    x, w, labels = xent_input(np.random.default_rng(11), n, dim, vocab)
    check_xent(q, own, bf16(x * 600.0), w, labels, piece=piece)


def test_grad_scale_in_pieces(q, own):
    """A power of two scales the gradients exactly, and a second call gives the same bits."""
    n, dim, vocab, piece = 8300, 40, 520, 256
    assert plan(n, vocab, dim, piece)["pieces"] == 3
    data = xent_input(np.random.default_rng(12), n, dim, vocab)
    one, many, again = (check_xent(q, own, *data, piece=piece, grad_scale=s) for s in (1.0, 256.0, 256.0))
    for a, b, c, factor in zip(one, many, again, (1, 1, 1, 256, 256)):
        assert np.array_equal(a * np.float32(factor), b) and np.array_equal(b, c)


def test_differences_in_pieces(q, own):
    """The gradients against central differences of the 64-bit loss along a direction: with steps t and t / 2 those are off by
    t^2 / 6 and t^2 / 24 times a third derivative, so what the halved step leaves is below the change."""
    n, dim, vocab, piece = 8300, 24, 600, 256
    assert plan(n, vocab, dim, piece)["pieces"] == 3
    r = np.random.default_rng(13)
    x, w, labels = xent_input(r, n, dim, vocab)
    _, _, _, dx, dw = check_xent(q, own, x, w, labels, piece=piece)
    x, w = x.astype(np.float64), w.astype(np.float64)
    ux, uw = r.standard_normal(x.shape), r.standard_normal(w.shape) / np.sqrt(dim)

    def loss(t):
        return float(xent(x + t * ux, w + t * uw, labels)[0])

    d1, d2 = ((loss(t) - loss(-t)) / (2 * t) for t in (1e-4, 5e-5))
    got = float(np.sum(dx.astype(np.float64) * ux) + np.sum(dw.astype(np.float64) * uw))
    ref = Reference(x, w, labels)
    tol = ref.tol_dx * np.linalg.norm(ux) + ref.tol_dw * np.linalg.norm(uw) + U * (np.sum(np.abs(dx * ux)) + np.sum(np.abs(dw * uw)))
    assert abs(got - d2) <= abs(d1 - d2) + tol + 2.0 ** -52 / 5e-5 * abs(loss(0.0))


def test_recorded_in_pieces(dev, q, own):
    """A recorded call in pieces, replayed with eager work on another queue between, gives the eager call's bits."""
    n, dim, vocab, piece = 8300, 72, 600, 256
    assert plan(n, vocab, dim, piece)["pieces"] == 3
    x, w, labels = xent_input(np.random.default_rng(14), n, dim, vocab)
    t = own.put(x, "bf16"), own.put(w, "bf16"), own.put(labels, "i32")
    out = own.empty((1,), "f32"), own.empty((n, dim), "f32"), own.empty((vocab, dim), "bf16")
    ws = own.scratch(kernels.linear_xent_workspace_bytes(n, vocab, dim, piece=piece))

    def call(queue):
        kernels.linear_xent_fwd_bwd(queue, *t, *out, piece=piece, workspace=ws)

    def poison(queue):
        for o in out:
            o.buffer.fill_u32(queue, 0x7FC07FC0)
        queue.sync()

    call(q)
    want = [o.numpy(q) for o in out]
    other = Queue(dev)
    with q.capture() as rec:
        call(q)
    for k in range(3):
        poison(q)
        if k == 1:
            call(other)
            assert all(np.array_equal(o.numpy(other), v) for o, v in zip(out, want))
            poison(other)
        rec.graph.launch(q)
        assert all(np.array_equal(o.numpy(q), v) for o, v in zip(out, want)), f"replay {k}"
    rec.graph.destroy()
    other.destroy()


def test_training_step_in_pieces(dev, q):
    """The token model's step with the output layer in three pieces against the same step whole.  A piece's logits that are
    formed again give p from f32 logits where the whole call takes codes, so G moves by 2^-12 of p besides its rounding
    to bf16, at most 2^-7 of itself between the two; every gradient is linear in it and passes the same roundings after it (12
    tensors at most, 2^-8 of their norm each)."""
    tokens, vocab, dim, hidden = 8300, 700, 64, 128
    assert plan(tokens, vocab, dim, 256)["pieces"] == 3 and plan(tokens, vocab, dim, 0)["pieces"] == 1
    r = np.random.default_rng(15)
    ids, labels = (r.integers(-1, vocab + 1, tokens).astype(np.int32) for _ in range(2))
    feeds, results = {}, []
    for piece in (0, 256):
        g, grads = graph.token_mlp_train_graph(tokens, vocab, dim, hidden, 1, piece=piece)
        exe = g.compile(dev)
        for name in grads:
            v = g.values[name]
            if name not in feeds:
                scale = v.shape[-1] ** -0.5 if len(v.shape) == 2 else 0.2
                feeds[name] = (r.standard_normal(v.shape) * scale + name.endswith("gamma")).astype(np.float32)
            exe.write(q, name, rng.f32_to_bf16(feeds[name]) if v.dtype == "bf16" else feeds[name])
        exe.write(q, "ids", ids)
        exe.write(q, "labels", labels)
        exe.run(q)
        results.append({n: exe.read(q, v.name).astype(np.float64) for n, v in [("loss", g.values["loss"]), *grads.items()]})
        exe.free()
    whole, pieces = results
    assert whole["loss"][0] == pieces["loss"][0]
    for n, a in whole.items():
        assert np.linalg.norm(a - pieces[n]) <= 12 * 2.0 ** -8 * np.linalg.norm(a), n
