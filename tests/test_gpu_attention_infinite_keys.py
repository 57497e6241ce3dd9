"""Attention over keys that hold infinities, as masks of them do: rows that give no key a weight, a key that no row gives one."""
import numpy as np
import pytest

import attention64 as ref
from test_gpu_attention import check, make_cache, own, projection, rounding, starts_of  # noqa: F401
from test_gpu_tokens import bf16, get
from vernondsl_amd import kernels

pytestmark = pytest.mark.gpu


# four parts of the keys a block, and one; causal and not
@pytest.mark.parametrize("n,heads,kv,dim,causal", [(96, 2, 1, 64, True), (300, 4, 2, 128, False), (1100, 32, 32, 64, True), (1100, 32, 32, 80, False)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_scores_of_minus_infinity_all_of_them(q, own, n, heads, kv, dim, causal, bad):
    """Every score is -inf: out 0 and lse -inf, whatever the values hold."""
    a, b = np.ones((n, heads, dim), np.float32), np.full((n, kv, dim), -np.inf, np.float32)
    c = bf16(np.random.default_rng(n).standard_normal((n, kv, dim)))
    c[::3], c[1::3, :, ::2] = bad, bad
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    kernels.attention_fwd(q, *[own.put(x, "bf16") for x in (a, b, c)], own.put(starts_of([n]), "i32"), out, lse=lse, causal=causal)
    assert not get(q, out).any() and np.isneginf(get(q, lse)).all()


# few rows and many, whole and split
@pytest.mark.parametrize("rows,length,cols", [(3, 30, 2), (3, 1900, 120), (100, 200, 13), (100, 1900, 120)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_paged_scores_of_minus_infinity_all_of_them(q, own, rows, length, cols, bad):
    heads, kv, dim, page = 4, 2, 64, 16
    _, vc = make_cache(np.random.default_rng(rows), cols, kv, page, dim)
    vc[:, :, ::3], vc[:, :, 1::3, ::2] = bad, bad
    kc = np.full_like(vc, -np.inf)
    out, lse = own.empty((rows, heads * dim), "f32"), own.empty((heads, rows), "f32")
    need = kernels.paged_attention_workspace_bytes(rows, 1, heads, kv, dim, cols * page)
    assert (need > 0) == (length == 1900)
    kernels.paged_attention(q, own.put(np.ones((rows, heads, dim)), "bf16"), own.put(kc, "bf16"), own.put(vc, "bf16"), own.put(starts_of([rows]), "i32"),
                            own.put(np.array([length]), "i32"), own.put(np.arange(cols)[None], "i32"), out, lse=lse,
                            workspace=own.scratch(need) if need else None)
    assert not get(q, out).any() and np.isneginf(get(q, lse)).all()

# 64 keys a block, with splits of the rows and without, and 128; rows that are no whole tiles
@pytest.mark.parametrize("n,heads,kv,dim,causal", [(100, 1, 1, 64, True), (333, 4, 2, 128, True), (400, 16, 1, 128, True), (201, 2, 2, 40, False),
                                                   (900, 40, 40, 64, True), (500, 40, 40, 96, False)])
def test_a_key_that_no_row_gives_a_weight(q, own, n, heads, kv, dim, causal):
    """Key 5 is -inf in a column where every q is 1, and so has score -inf with all rows: its dk and dv are 0, and the other keys' and
    rows' gradients those without it (but for dq's column that is 0 times infinity)."""
    r = np.random.default_rng(n)
    a, b, c = projection(r, n, heads, kv, dim)
    d = bf16(r.standard_normal((n, heads, dim)))
    a[..., 0], b[..., 0] = 1.0, 0.0
    b[5, :, 0] = -np.inf
    starts, scale = own.put(starts_of([n]), "i32"), dim ** -0.5
    x = [own.put(y, "bf16") for y in (a, b, c)]
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    kernels.attention_fwd(q, *x, starts, out, lse=lse, causal=causal)
    b[5, :, 0] = -1e4  # the same weights in 64 bits: exp(-1e4 / sqrt(128)) is 0
    b64 = b.astype(np.float64)
    want, want_lse, eo, el = ref.packed(a.astype(np.float64), b64, c.astype(np.float64), starts_of([n]), scale, causal)
    got = get(q, out).reshape(n, heads, dim)
    check(get(q, lse), want_lse, el, "lse")
    check(got, want, eo + rounding("f32", np.abs(want) + eo), "out")
    g = [own.empty((n, h, dim), "f32") for h in (heads, kv, kv)]
    kernels.attention_bwd(q, own.put(d.reshape(n, -1), "bf16"), *x, starts, out, lse, *g, causal=causal,
                          workspace=own.scratch(kernels.attention_bwd_workspace_bytes(n, 1, heads, kv, dim)))
    want, bound = ref.packed_grad(a.astype(np.float64), b64, c.astype(np.float64), got, get(q, lse), d.astype(np.float64), starts_of([n]), scale, causal)
    dq, dk, dv = (get(q, y) for y in g)
    assert not dk[5].any() and not dv[5].any()
    for name, y, w, e in (("dq", dq[..., 1:], want[0][..., 1:], bound[0][..., 1:]), ("dk", dk, want[1], bound[1]), ("dv", dv, want[2], bound[2])):
        check(y, w, e + rounding("f32", np.abs(w) + e), name)
