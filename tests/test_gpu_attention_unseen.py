"""Attention where values that are no finite numbers meet rows that have no use for them: positions of a paged cache that only
some new rows see, gradients in bf16 columns of one tensor beside rows that are left out of their products."""
import numpy as np
import pytest

import attention64 as ref
from attention64 import B, U
from test_gpu_attention import check, fused, make_cache, own, projection, rounding, starts_of  # noqa: F401
from test_gpu_tokens import bf16, get
from vernondsl_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (128, 8, 1), (80, 2, 2)])
# few rows in one split and in several, many rows likewise; the rows from `at` on are bad; a page of each sequence is none
@pytest.mark.parametrize("rows,at,length,cols,split", [(3, 1, 30, 2, False), (3, 2, 1000, 64, True), (100, 37, 200, 15, False), (100, 71, 1100, 80, True)])
def test_paged_positions_that_some_rows_see(q, own, rows, at, length, cols, split, dim, heads, kv, bad):
    """The chunk's rows from `at` on append keys and values that are no finite numbers: the rows before do not see them."""
    r = np.random.default_rng(rows + dim)
    page, seqs, n = 16, 2, 2 * rows
    pages = seqs * cols
    kc, vc = make_cache(r, pages, kv, page, dim)
    table = r.permutation(pages).reshape(seqs, cols).astype(np.int32)
    if cols > 2:
        table[:, 1] = (-1, pages)  # a page that is none
    lengths = np.array([length, length - 7], np.int32)
    a, b, c = projection(r, n, heads, kv, dim)
    clean = [x.copy() for x in (a, b, c)]
    late = np.tile(np.arange(rows) >= at, seqs)
    a[late], b[late] = bad, bad
    c[late, :, ::3] = bad
    tk, tv = own.put(kc, "bf16"), own.put(vc, "bf16")
    ts, tl, tt = own.put(starts_of([rows] * seqs), "i32"), own.put(lengths, "i32"), own.put(table, "i32")
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    need = kernels.paged_attention_workspace_bytes(n, seqs, heads, kv, dim, cols * page)
    assert (need > 0) == split
    qkv = fused(own, a, b, c)
    kernels.cache_append(q, *qkv[1:], ts, tl, tt, tk, tv)
    kernels.paged_attention(q, qkv[0], tk, tv, ts, tl, tt, out, lse=lse, workspace=own.scratch(need) if need else None)
    for s, first, m, pos in ref.cache_positions(starts_of([rows] * seqs), lengths, n):
        for i in range(m):
            p = pos + i
            if 0 <= table[s, p // page] < pages:
                kc[table[s, p // page], :, p % page], vc[table[s, p // page], :, p % page] = clean[1][first + i], clean[2][first + i]
    want, want_lse, eo, el = ref.paged(*(x.astype(np.float64) for x in (clean[0], kc, vc)), starts_of([rows] * seqs), lengths, table, dim ** -0.5)
    check(get(q, lse)[:, ~late], want_lse[:, ~late], el[:, ~late], "lse")
    check(get(q, out).reshape(n, heads, dim)[~late], want[~late], (eo + rounding("f32", want) + U * eo)[~late], "out")


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
# 64 keys a block, with splits of the rows and without, and 128
@pytest.mark.parametrize("dim,heads,kv,n,at", [(64, 2, 1, 200, 70), (128, 16, 1, 400, 130), (80, 24, 2, 300, 40), (64, 40, 40, 900, 400),
                                               (128, 72, 36, 1000, 530)])
def test_gradients_in_bf16_columns(q, own, dim, heads, kv, n, at, bad):
    """Rows before `at` whose q and dout are no finite numbers leave dk and dv of the keys from `at` on alone, in bf16 columns
    of one tensor; keys from `at` on that are none leave dq of the rows before alone."""
    r = np.random.default_rng(n + dim)
    a, b, c = projection(r, n, heads, kv, dim)
    d = bf16(r.standard_normal((n, heads, dim)))
    starts, scale = own.put(starts_of([n]), "i32"), dim ** -0.5
    out, lse = own.empty((n, heads * dim), "bf16"), own.empty((heads, n), "f32")
    kernels.attention_fwd(q, *[own.put(x, "bf16") for x in (a, b, c)], starts, out, lse=lse)
    width = (heads + 2 * kv) * dim + 24

    def backward(a, b, c, d):
        t = own.empty((n, width), "bf16")
        g = [kernels.Heads(t, h, dim, 16 + f * dim) for h, f in ((heads, 0), (kv, heads), (kv, heads + kv))]
        ws = own.scratch(kernels.attention_bwd_workspace_bytes(n, 1, heads, kv, dim))
        kernels.attention_bwd(q, own.put(d.reshape(n, -1), "bf16"), *fused(own, a, b, c), starts, out, lse, *g, workspace=ws)
        x = get(q, t)
        assert np.isnan(x[:, :16]).all() and np.isnan(x[:, -8:]).all()
        return [x[:, y.first:y.first + y.heads * dim].reshape(n, y.heads, dim) for y in g]

    want, bound = ref.packed_grad(*(x.astype(np.float64) for x in (a, b, c)), get(q, out).reshape(n, heads, dim), get(q, lse), d.astype(np.float64),
                                  starts_of([n]), scale, True)
    a2, b2, c2, d2 = a.copy(), b.copy(), c.copy(), d.copy()
    b2[at:], c2[at:, :, ::3] = bad, bad
    check(backward(a, b2, c2, d)[0][:at], want[0][:at], (bound[0] + rounding("bf16", np.abs(want[0]) + bound[0]))[:at], "dq")
    a2[:at], d2[:at] = bad, bad
    # A key whose block leaves rows out is stored, read and stored again: two roundings, the first of a partial sum.  That one is no
    # larger than the sum of the terms' magnitudes, of which `bound` holds B already (of p and ds as the products' operands).
    for g, w, e, name in list(zip(backward(a2, b, c, d2), want, bound, ("dq", "dk", "dv")))[1:]:
        once = e + B * (np.abs(w) + e)
        check(g[at:], w[at:], (once + (1 + B) * e + B * (1 + B) * e)[at:], name)
