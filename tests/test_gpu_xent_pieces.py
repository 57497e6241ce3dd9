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

from test_gpu_tokens import U, Owner, get, xent, xent_input
from test_linear_xent_plan import WIDE, plan
from vernondsl_amd import kernels

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
