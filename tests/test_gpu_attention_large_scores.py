"""Attention at scores up to 2^30, the largest that the forward passes are made for: the largest of a row wins, equal ones share.

Scores are exact in f32: q is a power of two in one column, k a whole number below 2^8 in that column.  Their distances are 2^22 and
more, so weights are 1 / (equal largest scores) or 0, and out is an average of few values: f32 sums of bf16 products with one
weight, which bf16 may round (common to all of a row's weights), over their sum."""
import numpy as np
import pytest

from test_gpu_attention import own, starts_of  # noqa: F401
from test_gpu_tokens import B, U, bf16, get
from vernondsl_amd import kernels

pytestmark = pytest.mark.gpu


def expected(scores, seen, v):
    """Of one head: the average of the values of the largest scores, and lse."""
    s = np.where(seen, scores, -np.inf)
    top = s.max(1)
    win = (s == top[:, None]).astype(np.float64)
    return win @ v / win.sum(1)[:, None], top + np.log(win.sum(1))


def check(got, got_lse, want, want_lse):
    assert np.all(np.abs(got - want) <= (2 * B + 64 * U) * np.abs(want).max() + 1e-30)
    assert np.all(np.abs(got_lse - want_lse) <= 4 * U * np.abs(want_lse))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("n,heads,kv,dim", [(90, 2, 1, 64), (700, 4, 2, 16), (1100, 32, 32, 64)])
def test_packed(q, own, n, heads, kv, dim, sign):
    r = np.random.default_rng(n)
    a, b = np.zeros((n, heads, dim), np.float32), np.zeros((n, kv, dim), np.float32)
    a[..., 3] = 2.0 ** 22
    b[..., 3] = sign * r.integers(1, 257, (n, kv))
    c = bf16(1.0 + r.random((n, kv, dim)))
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    kernels.attention_fwd(q, *[own.put(x, "bf16") for x in (a, b, c)], own.put(starts_of([n]), "i32"), out, lse=lse, scale=1.0)
    got, got_lse = get(q, out).reshape(n, heads, dim), get(q, lse)
    for h in range(heads):
        g = h * kv // heads
        s = a[:, h].astype(np.float64) @ b[:, g].astype(np.float64).T
        assert np.abs(s).max() <= 2.0 ** 30
        check(got[:, h], got_lse[h], *expected(s, np.tril(np.ones((n, n), bool)), c[:, g].astype(np.float64)))


@pytest.mark.parametrize("sign", [1, -1])
# few rows and many, whole and split
@pytest.mark.parametrize("rows,length,cols", [(3, 30, 2), (3, 1900, 120), (100, 200, 13), (100, 1900, 120)])
def test_paged(q, own, rows, length, cols, sign):
    heads, kv, dim, page = 4, 2, 64, 16
    r = np.random.default_rng(rows + length)
    a, kc = np.zeros((rows, heads, dim), np.float32), np.zeros((cols, kv, page, dim), np.float32)
    a[..., 3] = 2.0 ** 22
    kc[..., 3] = sign * r.integers(1, 257, (cols, kv, page))
    vc = bf16(1.0 + r.random((cols, kv, page, dim)))
    out, lse = own.empty((rows, heads * dim), "f32"), own.empty((heads, rows), "f32")
    need = kernels.paged_attention_workspace_bytes(rows, 1, heads, kv, dim, cols * page)
    assert (need > 0) == (length == 1900)
    kernels.paged_attention(q, own.put(a, "bf16"), own.put(kc, "bf16"), own.put(vc, "bf16"), own.put(starts_of([rows]), "i32"),
                            own.put(np.array([length]), "i32"), own.put(np.arange(cols)[None], "i32"), out, lse=lse, scale=1.0,
                            workspace=own.scratch(need) if need else None)
    got, got_lse = get(q, out).reshape(rows, heads, dim), get(q, lse)
    seen = np.arange(length)[None] <= (length - rows + np.arange(rows))[:, None]
    for h in range(heads):
        k, v = (x[:, h // 2].reshape(-1, dim)[:length].astype(np.float64) for x in (kc, vc))
        check(got[:, h], got_lse[h], *expected(a[:, h].astype(np.float64) @ k.T, seen, v))
