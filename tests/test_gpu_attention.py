"""Attention over packed sequences and over a paged cache, the append to it, and rotary positions on the device against
attention64's plain forms in 64 bits, at the lengths, layouts and masks where they can go wrong."""
import ctypes as C

import numpy as np
import pytest

import attention64 as ref
from attention64 import B, U
from test_gpu_tokens import Owner, bf16, empty, get
from vernondsl_amd import _lib, kernels, rng

pytestmark = pytest.mark.gpu


@pytest.fixture
def own(dev, q):
    o = Owner(dev, q)
    yield o
    q.sync()
    for t in o.all:
        t.free()


def rounding(dtype, y):
    return (B if dtype == "bf16" else U) * np.abs(y)


def starts_of(lengths, front=0):
    return np.concatenate([[front], front + np.cumsum(lengths)]).astype(np.int32)


def projection(r, n, heads, kv, dim, spread=1.5):
    """q, k, v as f32 values that bf16 holds."""
    return [bf16(r.standard_normal((n, h, dim)) * s) for h, s in ((heads, spread), (kv, spread), (kv, 1.0))]


def fused(own, q, k, v, lead=8, tail=16):
    """The three as columns of one tensor with other columns before and behind, NaN."""
    n, heads, dim = q.shape
    kv = k.shape[1]
    width = lead + (heads + 2 * kv) * dim + tail
    x = np.full((n, width), np.nan, np.float32)
    at, out = lead, []
    for part in (q, k, v):
        x[:, at:at + part.shape[1] * dim] = part.reshape(n, -1)
        out.append(at)
        at += part.shape[1] * dim
    t = own.put(x, "bf16")
    return [kernels.Heads(t, h, dim, first) for h, first in zip((heads, kv, kv), out)]


def check(got, want, bound, what):
    assert np.all(np.isfinite(got) | np.isneginf(want)), what
    fine = np.isneginf(want) & np.isneginf(got)
    with np.errstate(invalid="ignore"):
        off = np.where(fine, 0.0, np.abs(got - want) - bound)
    assert np.all(off <= 1e-30), (what, float(np.nanmax(off)), np.unravel_index(np.nanargmax(off), off.shape))


# lengths, rows before the first sequence, rows behind the last, heads, kv heads, dim, causal
PACKED = [([1], 0, 0, 1, 1, 8, True), ([2, 0, 1], 1, 2, 2, 1, 16, True), ([33], 0, 0, 3, 1, 64, True), ([63, 64, 65], 0, 3, 4, 2, 64, True),
          ([127, 0, 130, 1], 2, 5, 6, 2, 80, True), ([300], 0, 0, 5, 1, 128, True), ([257, 31], 0, 0, 4, 4, 40, True),
          ([129, 70], 3, 0, 8, 1, 96, True), ([200, 0, 56], 0, 7, 2, 2, 128, False), ([1, 1, 1, 1, 1], 0, 0, 4, 2, 64, False),
          ([513], 0, 0, 2, 1, 104, False), ([0, 0], 0, 9, 2, 1, 64, True), ([90] * 70, 0, 0, 2, 2, 32, True),
          ([4200], 0, 0, 16, 2, 64, True), ([2300, 2000], 0, 11, 16, 4, 128, True), ([4100], 0, 0, 16, 2, 88, False),
          # as above, with so many kv heads that the gradient's blocks have 128 keys
          ([1100], 0, 0, 32, 32, 8, True), ([1000, 50], 0, 3, 40, 40, 128, True), ([500, 0, 600], 2, 0, 64, 32, 64, True), ([700], 0, 0, 32, 32, 96, False),
          # few kv heads that many share, whose rows the gradient splits
          ([700], 0, 5, 64, 1, 128, True), ([40, 900, 3], 1, 0, 12, 2, 72, False),
          # more sequences than a wave's lanes hold, at both sides of it
          ([3, 0] * 62 + [17], 2, 3, 4, 2, 16, True), ([3, 0] * 63, 0, 3, 4, 2, 16, True), ([2] * 300, 1, 0, 2, 1, 8, False)]


@pytest.mark.parametrize("lengths,front,back,heads,kv,dim,causal", PACKED)
def test_packed(q, own, lengths, front, back, heads, kv, dim, causal):
    r = np.random.default_rng(dim + sum(lengths))
    n = front + sum(lengths) + back
    a, b, c = projection(r, n, heads, kv, dim)
    for x in (a, b, c):  # rows of no sequence hold anything
        x[:front] = np.nan
        x[n - back:] = np.inf
    starts = starts_of(lengths, front)
    out_dtype = "f32" if dim % 16 else "bf16"
    out, lse = own.empty((n, heads * dim), out_dtype), own.empty((heads, n), "f32")
    ts = own.put(starts, "i32")
    qkv = fused(own, a, b, c) if heads % 2 == 0 else [own.put(x, "bf16") for x in (a, b, c)]
    kernels.attention_fwd(q, *qkv, ts, out, lse=lse, causal=causal)
    got, got_lse = get(q, out).reshape(n, heads, dim), get(q, lse)
    a, b, c = (np.where(np.isfinite(x), x, 0).astype(np.float64) for x in (a, b, c))
    want, want_lse, eo, el = ref.packed(a, b, c, starts, dim ** -0.5, causal)
    check(got_lse, want_lse, el, "lse")
    check(got, want, eo + rounding(out_dtype, np.abs(want) + eo), "out")
    inside = np.zeros(n, bool)
    inside[front:n - back] = True
    assert not got[~inside].any() and np.isneginf(got_lse[:, ~inside]).all()

    # the gradient, of dout in either type, into columns of one tensor or apart, from this out and lse
    dout = r.standard_normal((n, heads, dim)).astype(np.float32)
    dout[~inside] = np.nan
    dt = "f32" if heads % 4 == 0 else "bf16"
    grad_dtype = "f32" if dim % 32 else "bf16"
    tdo = own.put(dout.reshape(n, -1), dt)
    ws = own.scratch(kernels.attention_bwd_workspace_bytes(n, len(lengths), heads, kv, dim))
    if heads % 2 == 0:
        width = (heads + 2 * kv) * dim + 8
        t = own.empty((n, width), grad_dtype)
        grads = [kernels.Heads(t, h, dim, f * dim) for h, f in ((heads, 0), (kv, heads), (kv, heads + kv))]
    else:
        grads = [own.empty((n, h, dim), grad_dtype) for h in (heads, kv, kv)]
    kernels.attention_bwd(q, tdo, *qkv, ts, out, lse, *grads, causal=causal, workspace=ws)
    dout = np.where(np.isfinite(dout), bf16(np.nan_to_num(dout)), 0).astype(np.float64)
    lse64 = np.where(np.isfinite(got_lse), got_lse, 0.0)
    want, bound = ref.packed_grad(a, b, c, got, lse64, dout, starts, dim ** -0.5, causal)
    if heads % 2 == 0:
        all_ = get(q, t)
        assert np.isnan(all_[:, -8:]).all()  # columns of no head stay
        found = [all_[:, g.first:g.first + g.heads * dim].reshape(n, g.heads, dim) for g in grads]
    else:
        found = [get(q, g) for g in grads]
    for name, g, w, e in zip(("dq", "dk", "dv"), found, want, bound):
        check(g, w, e + rounding(grad_dtype, np.abs(w) + e), name)
        assert not g[~inside].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dim,heads,kv,n,at", [(64, 2, 1, 200, 70), (128, 4, 2, 333, 150), (80, 1, 1, 100, 99), (64, 40, 40, 900, 400), (128, 72, 36, 1000, 530), (128, 16, 1, 400, 130)])
def test_what_is_not_seen_has_no_influence(q, own, dim, heads, kv, n, at, bad):
    """Rows from `at` on hold NaN or infinities: the rows before have the outputs that they would have alone, and their dq too;
    rows before `at` whose q and dout are so leave the gradients of the keys from `at` on alone."""
    r = np.random.default_rng(n)
    a, b, c = projection(r, n, heads, kv, dim)
    d = bf16(r.standard_normal((n, heads, dim)))
    starts, scale = own.put(starts_of([n]), "i32"), dim ** -0.5
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")

    def forward(*x):
        kernels.attention_fwd(q, *[own.put(y, "bf16") for y in x], starts, out, lse=lse)

    def backward(a, b, c, d):
        ws = own.scratch(kernels.attention_bwd_workspace_bytes(n, 1, heads, kv, dim))
        g = [own.empty((n, h, dim), "f32") for h in (heads, kv, kv)]
        kernels.attention_bwd(q, own.put(d.reshape(n, -1), "bf16"), *[own.put(x, "bf16") for x in (a, b, c)], starts, out, lse, *g, workspace=ws)
        return [get(q, x) for x in g]

    clean = [x.astype(np.float64) for x in (a, b, c)]
    want, want_lse, eo, el = ref.packed(*clean, starts_of([n]), scale, True)
    a2, b2, c2, d2 = a.copy(), b.copy(), c.copy(), d.copy()
    a2[at:], b2[at:], c2[at:, :, ::3] = bad, bad, bad
    forward(a2, b2, c2)
    check(get(q, lse)[:, :at], want_lse[:, :at], el[:, :at], "lse")
    check(get(q, out).reshape(n, heads, dim)[:at], want[:at], (eo + rounding("f32", want) + U * eo)[:at], "out")
    forward(a, b, c)
    want, bound = ref.packed_grad(*clean, get(q, out).reshape(n, heads, dim), get(q, lse), d.astype(np.float64), starts_of([n]), scale, True)
    bound = [e + rounding("f32", np.abs(w) + e) for w, e in zip(want, bound)]
    check(backward(a, b2, c2, d)[0][:at], want[0][:at], bound[0][:at], "dq")
    a3 = a.copy()
    a3[:at], d2[:at] = bad, bad
    for g, w, e, name in list(zip(backward(a3, b, c, d2), want, bound, ("dq", "dk", "dv")))[1:]:
        check(g[at:], w[at:], e[at:], name)


def test_extreme_scores(q, own):
    """Scores of +-1e4 and far beyond: the largest wins, nothing overflows; scores that are -inf all of them count as not seen."""
    n, dim = 96, 64
    r = np.random.default_rng(3)
    a, b, c = projection(r, n, 2, 1, dim, spread=40.0)
    out, lse = own.empty((n, 2 * dim), "f32"), own.empty((2, n), "f32")
    starts = own.put(starts_of([n]), "i32")
    kernels.attention_fwd(q, *[own.put(x, "bf16") for x in (a, b, c)], starts, out, lse=lse, scale=8.0)
    want, want_lse, eo, el = ref.packed(*(x.astype(np.float64) for x in (a, b, c)), starts_of([n]), 8.0, True)
    check(get(q, lse), want_lse, el, "lse")
    check(get(q, out).reshape(n, 2, dim), want, eo + rounding("f32", want), "out")
    a[:], b[:] = 1.0, -np.inf
    kernels.attention_fwd(q, *[own.put(x, "bf16") for x in (a, b, c)], starts, out, lse=lse)
    assert not get(q, out).any() and np.isneginf(get(q, lse)).all()


def test_nan_is_handed_on(q, own):
    """A row whose q is NaN, in one head: NaN for that row and head alone, and for the gradients that it has a part in."""
    n, heads, kv, dim, bad = 150, 4, 2, 64, 70
    a, b, c = projection(np.random.default_rng(7), n, heads, kv, dim)
    a[bad, 1] = np.nan
    starts = own.put(starts_of([n]), "i32")
    x = [own.put(y, "bf16") for y in (a, b, c)]
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    kernels.attention_fwd(q, *x, starts, out, lse=lse)
    hit = np.zeros((n, heads), bool)
    hit[bad, 1] = True

    def of_that_row_only(n=n, hit=hit):
        found = get(q, out).reshape(n, heads, dim)
        assert np.isnan(found[hit]).all() and np.isfinite(found[~hit]).all()
        assert np.array_equal(np.isnan(get(q, lse)).T, hit) and np.isfinite(get(q, lse).T[~hit]).all()

    of_that_row_only()
    g = [own.empty((n, h, dim), "f32") for h in (heads, kv, kv)]
    kernels.attention_bwd(q, own.put(np.ones((n, heads * dim)), "bf16"), *x, starts, out, lse, *g,
                          workspace=own.scratch(kernels.attention_bwd_workspace_bytes(n, 1, heads, kv, dim)))
    dq, dk, dv = (get(q, y) for y in g)
    assert np.isnan(dq[hit]).all() and np.isfinite(dq[~hit]).all()
    for d in (dk, dv):
        assert np.isnan(d[:bad + 1, 0]).all() and np.isfinite(d[bad + 1:]).all() and np.isfinite(d[:, 1]).all()

    page = 16
    for rows, keys, cols in ((3, 30, 2), (3, 1900, 120), (100, 200, 13), (100, 1900, 120)):  # of few rows and many, whole and split
        kc, vc = (own.put(y, "bf16") for y in make_cache(np.random.default_rng(8), cols, kv, page, dim))
        out, lse = own.empty((rows, heads * dim), "f32"), own.empty((heads, rows), "f32")
        y = a[bad - 1:bad - 1 + rows]  # row 1 is the one
        need = kernels.paged_attention_workspace_bytes(rows, 1, heads, kv, dim, cols * page)
        assert (need > 0) == (keys == 1900)
        kernels.paged_attention(q, own.put(np.concatenate([y, a[:rows - len(y)]]), "bf16"), kc, vc, own.put(starts_of([rows]), "i32"),
                                own.put(np.array([keys]), "i32"), own.put(np.arange(cols)[None], "i32"), out, lse=lse, workspace=own.scratch(max(4, need)))
        hit = np.zeros((rows, heads), bool)
        hit[1, 1] = True
        of_that_row_only(rows, hit)


# page, table's columns, lengths, new rows, heads, kv heads, dim, rows behind
CACHES = [(16, 4, [20, 64, 1], [1, 1, 1], 4, 2, 64, 0), (16, 40, [40, 7, 0], [1, 1, 0], 2, 1, 128, 2), (64, 3, [130, 192, 64, 65], [1, 0, 1, 1], 8, 1, 80, 1),
          (16, 20, [300, 17], [40, 17], 4, 4, 128, 0), (256, 8, [2000, 1000, 5], [130, 1, 5], 8, 2, 128, 3), (32, 64, [2048], [1], 32, 8, 128, 0),
          (32, 30, [200, 100], [200, 3], 6, 2, 40, 0), (64, 64, [4000, 3000], [600, 2], 16, 2, 96, 0), (16, 64, [1000] * 40, [1] * 40, 8, 2, 64, 0),
          (65536, 1, [700], [9], 1, 1, 8, 0)]


def make_cache(r, pages, kv, page, dim):
    return [bf16(r.standard_normal((pages, kv, page, dim)) * s) for s in (1.5, 1.0)]


@pytest.mark.parametrize("page,cols,lengths,new,heads,kv,dim,back", CACHES)
def test_paged(q, own, page, cols, lengths, new, heads, kv, dim, back):
    r = np.random.default_rng(page + sum(lengths))
    seqs, n = len(lengths), sum(new) + back
    pages = seqs * cols + 1
    kc, vc = make_cache(r, pages, kv, page, dim)
    table = r.permutation(pages)[:seqs * cols].reshape(seqs, cols).astype(np.int32)
    lengths = np.array(lengths, np.int32)
    for s in range(seqs):  # behind a sequence's end: anything, and no pages
        used = -(-int(lengths[s]) // page)
        if lengths[s] % page:
            kc[table[s, used - 1], :, lengths[s] % page:] = np.nan
            vc[table[s, used - 1], :, lengths[s] % page:] = np.inf
        table[s, used:] = r.choice([-1, pages, 1 << 30, -(1 << 31)])
    a, b, c = projection(r, n, heads, kv, dim)
    a[n - back:] = b[n - back:] = c[n - back:] = np.nan
    starts = starts_of(new)
    tk, tv = own.put(kc, "bf16"), own.put(vc, "bf16")
    ts, tl, tt = own.put(starts, "i32"), own.put(lengths, "i32"), own.put(table, "i32")
    qkv = fused(own, a, b, c)
    out, lse = own.empty((n, heads * dim), "bf16"), own.empty((heads, n), "f32")
    ws = own.scratch(kernels.paged_attention_workspace_bytes(n, seqs, heads, kv, dim, cols * page))
    kernels.cache_append(q, *qkv[1:], ts, tl, tt, tk, tv)
    kernels.paged_attention(q, qkv[0], tk, tv, ts, tl, tt, out, lse=lse, workspace=ws)
    for s, at, m, pos in ref.cache_positions(starts, lengths, n):
        for i in range(m):
            p = pos + i
            kc[table[s, p // page], :, p % page], vc[table[s, p // page], :, p % page] = b[at + i], c[at + i]
    for t, x in ((tk, kc), (tv, vc)):
        assert np.array_equal(get(q, t), x, equal_nan=True)  # the appended rows, and nothing else
    k64, v64 = (x.astype(np.float64) for x in (kc, vc))
    a = np.where(np.isfinite(a), a, 0).astype(np.float64)
    want, want_lse, eo, el = ref.paged(a, np.nan_to_num(k64, posinf=0), np.nan_to_num(v64, posinf=0), starts, lengths, table, dim ** -0.5)
    check(get(q, lse), want_lse, el, "lse")
    check(get(q, out).reshape(n, heads, dim), want, eo + rounding("bf16", np.abs(want) + eo), "out")


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_that_are_none(q, own, rows):
    """Entries outside the cache in the middle of a sequence, positions before 0 and past the table's room: nothing there."""
    r = np.random.default_rng(rows)
    heads, kv, dim, page, cols, pages = 4, 2, 64, 16, 6, 12
    kc, vc = make_cache(r, pages, kv, page, dim)
    vc[0] = np.inf  # what a masked key might read
    kc[0] = np.nan
    table = np.array([[3, -1, 5, 900, 7, 8], [-5, 1 << 30, -1, -1, -1, -1], [1, 2, 4, 6, 9, 10], [11, -1, -1, -1, -1, -1]], np.int32)
    lengths = np.array([80, 50, 96 + 20, rows - 1], np.int32)  # the third passes its table's room; the fourth has a row before 0
    starts = starts_of([rows] * 4)
    n = 4 * rows
    a, b, c = projection(r, n, heads, kv, dim)
    t = {k: own.put(x, d) for k, x, d in (("k", kc, "bf16"), ("v", vc, "bf16"), ("s", starts, "i32"), ("l", lengths, "i32"), ("t", table, "i32"))}
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    ws = own.scratch(kernels.paged_attention_workspace_bytes(n, 4, heads, kv, dim, cols * page))
    qkv = fused(own, a, b, c)
    kernels.cache_append(q, *qkv[1:], t["s"], t["l"], t["t"], t["k"], t["v"])
    for s, at, m, pos in ref.cache_positions(starts, lengths, n):
        for i in range(m):
            p = pos + i
            if 0 <= p < cols * page and 0 <= table[s, p // page] < pages:
                kc[table[s, p // page], :, p % page], vc[table[s, p // page], :, p % page] = b[at + i], c[at + i]
    assert np.array_equal(get(q, t["k"]), kc, equal_nan=True) and np.array_equal(get(q, t["v"]), vc, equal_nan=True)
    kernels.paged_attention(q, qkv[0], t["k"], t["v"], t["s"], t["l"], t["t"], out, lse=lse, workspace=ws)
    want, want_lse, eo, el = ref.paged(a.astype(np.float64), kc.astype(np.float64), vc.astype(np.float64), starts, lengths, table, dim ** -0.5)
    check(get(q, lse), want_lse, el, "lse")
    check(get(q, out).reshape(n, heads, dim), want, eo + rounding("f32", want), "out")
    assert not get(q, out)[rows:2 * rows].any()  # a sequence without a page


def test_nothing_there(q, own):
    """No rows, no sequences, no pages, a table without columns: nothing read, every row written."""
    n, heads, kv, dim = 5, 2, 1, 16
    x, one = own.put(np.ones((n, heads, dim)), "bf16"), own.put(np.zeros(2), "i32")
    at = _lib.Heads(0, heads * dim), _lib.Heads(0, kv * dim)
    k = own.put(np.ones((n, kv, dim)), "bf16")

    def paged(rows, seqs, pages, cols):
        return _lib.PagedParams(rows, seqs, pages, cols, 16, heads, kv, dim, 0.25, 0, at[0], at[1], at[1])

    lengths, table = own.put(np.full(2, 30), "i32"), own.put(np.zeros(4), "i32")
    cache = [own.put(np.full((1, kv, 16, dim), 3.0), "bf16") for _ in range(2)]
    for rows, seqs in ((0, 0), (0, 1), (n, 0)):
        out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
        p = _lib.AttentionParams(rows, seqs, heads, kv, dim, 1, 0.25, 0, at[0], at[1], at[1], at[0], at[1], at[1])
        _lib.call("vdsl_op_attention_fwd", q.handle, C.byref(p), x.handle, k.handle, k.handle, one.handle, 0, out.handle, lse.handle)
        assert np.array_equal(get(q, out)[:rows], np.zeros((rows, heads * dim))) and np.isnan(get(q, out)[rows:]).all()
        assert np.isneginf(get(q, lse)).all() if rows else np.isnan(get(q, lse)).all()
        g = [own.empty((n, h, dim), "f32") for h in (heads, kv, kv)]
        ws = own.scratch(kernels.attention_bwd_workspace_bytes(rows, seqs, heads, kv, dim))
        _lib.call("vdsl_op_attention_bwd", q.handle, C.byref(p), 1, x.handle, x.handle, k.handle, k.handle, one.handle, 0, out.handle,
                  lse.handle, 0, g[0].handle, g[1].handle, g[2].handle, ws.handle)
        assert all(not get(q, y)[:rows].any() and np.isnan(get(q, y)[rows:]).all() for y in g)
    starts = own.put(starts_of([n]), "i32")
    for rows, seqs, pages, cols in ((0, 1, 1, 4), (n, 0, 1, 4), (n, 1, 0, 4), (n, 1, 1, 0)):
        p, out = paged(rows, seqs, pages, cols), own.empty((n, heads * dim), "f32")
        need = kernels.paged_attention_workspace_bytes(rows, seqs, heads, kv, dim, cols * 16)
        _lib.call("vdsl_op_cache_append", q.handle, C.byref(p), k.handle, k.handle, starts.handle, lengths.handle, table.handle,
                  cache[0].handle, cache[1].handle)
        assert all((get(q, y) == 3.0).all() for y in cache)
        _lib.call("vdsl_op_paged_attention", q.handle, C.byref(p), x.handle, cache[0].handle, cache[1].handle, starts.handle,
                  lengths.handle, table.handle, 0, out.handle, None, own.scratch(max(4, need)).handle)
        assert not get(q, out)[:rows].any() and np.isnan(get(q, out)[rows:]).all()


def test_cache_past_32_bits(dev, q, own):
    """Pages whose bytes lie past 2^32 in a cache of 4.5 GiB."""
    from vernondsl_amd.rhi import Tensor
    kv, page, dim, heads = 8, 256, 128, 8
    pages = (9 << 29) // (kv * page * dim * 2)
    r = np.random.default_rng(5)
    kc, vc = (own.keep(Tensor(dev, (pages, kv, page, dim), "bf16")) for _ in range(2))
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    n = 600
    a, b, c = projection(r, n, heads, kv, dim)
    ts, tl, tt = own.put(starts_of([n]), "i32"), own.put(np.array([n]), "i32"), own.put(table, "i32")
    out, lse = own.empty((n, heads * dim), "bf16"), own.empty((heads, n), "f32")
    ws = own.scratch(kernels.paged_attention_workspace_bytes(n, 1, heads, kv, dim, 3 * page))
    qkv = fused(own, a, b, c)
    kernels.cache_append(q, *qkv[1:], ts, tl, tt, kc, vc)
    kernels.paged_attention(q, qkv[0], kc, vc, ts, tl, tt, out, lse=lse, workspace=ws)
    want, want_lse, eo, el = ref.packed(*(x.astype(np.float64) for x in (a, b, c)), starts_of([n]), dim ** -0.5, True)
    check(get(q, lse), want_lse, el, "lse")
    check(get(q, out).reshape(n, heads, dim), want, eo + rounding("bf16", np.abs(want) + eo), "out")


# rows, width, first, heads, dim, rot, interleaved, inverse, magnitude, x, y
ROPES = [(1, 64, 0, 1, 64, 64, False, False, 1.0, "f32", "f32"), (5, 200, 8, 2, 80, 40, True, False, 1.0, "bf16", "bf16"),
         (7, 131, 3, 3, 41, 14, False, True, 1.3, "f32", "f32"), (7, 131, 3, 3, 41, 14, True, False, 1.3, "f32", "bf16"),
         (300, 6 * 128, 0, 4, 128, 64, False, True, 1.0, "f32", "bf16"), (64, 1024, 0, 8, 128, 128, True, True, 0.5, "bf16", "f32"),
         (3, 24, 4, 0, 8, 8, False, False, 1.0, "bf16", "f32"), (3, 24, 4, 2, 8, 0, False, False, 1.0, "bf16", "bf16"), (2, 20, 0, 2, 10, 10, True, False, 1.0, "bf16", "bf16")]


@pytest.mark.parametrize("rows,width,first,heads,dim,rot,interleaved,inverse,magnitude,xt,yt", ROPES)
def test_rope(q, own, rows, width, first, heads, dim, rot, interleaved, inverse, magnitude, xt, yt):
    r = np.random.default_rng(rows + width)
    x = r.standard_normal((rows, width)).astype(np.float32)
    x = bf16(x) if xt == "bf16" else x
    positions = r.integers(-5, 1 << 20, rows).astype(np.int32)
    positions[0] = (1 << 31) - 1
    freqs = own.put(kernels.rope_frequencies(rot), "f32")
    tx, tp, y = own.put(x, xt), own.put(positions, "i32"), own.empty((rows, width), yt)
    kw = dict(first=first, interleaved=interleaved, inverse=inverse, magnitude=magnitude)
    kernels.rope(q, tx, tp, freqs, y, heads, dim, **kw)
    want = ref.rope(x, positions, ref.frequencies(rot), heads, dim, first, interleaved, inverse, magnitude)
    # the angle: frequencies to 2^-48 of positions up to 2^31, a fraction of a turn rounded to f32; sine and cosine good to
    # 2 U; times the magnitude, two products and a sum
    mag = ref.rope(np.abs(x), 0 * positions, np.zeros(rot // 2), heads, dim, first, interleaved, False, 1.0)
    off = np.zeros_like(want)
    pairs = rot // 2
    for h in range(heads):
        i = first + h * dim + (2 * np.arange(pairs) if interleaved else np.arange(pairs))
        j = i + (1 if interleaved else pairs)
        off[:, i] = off[:, j] = (mag[:, i] + mag[:, j]) * magnitude * (np.pi * U + 2 * U + 3 * U + np.abs(positions.astype(np.float64))[:, None] * 2.0 ** -45)
    assert np.all(np.abs(get(q, y) - want) <= off + rounding(yt, np.abs(want) + off))
    untouched = off == 0
    assert np.array_equal(get(q, y)[untouched], (bf16(x) if yt == "bf16" else x).astype(np.float64)[untouched])
    if xt == yt:  # in place
        kernels.rope(q, tx, tp, freqs, tx, heads, dim, **kw)
        assert np.array_equal(get(q, tx), get(q, y))


def test_same_bits_and_replays(q, own):
    """A training step's calls and a served token's, recorded: replays give the eager calls' bits, also after the lengths
    changed, with eager work between them."""
    r = np.random.default_rng(9)
    n, heads, kv, dim, page, cols = 500, 8, 2, 128, 16, 40
    a, b, c = projection(r, n, heads, kv, dim)
    qkv = fused(own, a, b, c)
    starts = own.put(starts_of([200, 0, 290]), "i32")
    out, lse = own.empty((n, heads * dim), "bf16"), own.empty((heads, n), "f32")
    dout = own.put(r.standard_normal((n, heads * dim)), "f32")
    g = [own.empty((n, h, dim), "f32") for h in (heads, kv, kv)]
    ws = own.scratch(kernels.attention_bwd_workspace_bytes(n, 3, heads, kv, dim))
    kc, vc = (own.put(x, "bf16") for x in make_cache(r, 3 * cols, kv, page, dim))
    table = own.put(r.permutation(3 * cols).reshape(3, cols).astype(np.int32), "i32")
    one, lengths = own.put(starts_of([1, 1, 1]), "i32"), own.put(np.array([600, 3, 111]), "i32")
    x1 = [own.put(x[:3], "bf16") for x in (a, b, c)]
    out1, lse1 = own.empty((3, heads * dim), "bf16"), own.empty((heads, 3), "f32")
    ws1 = own.scratch(kernels.paged_attention_workspace_bytes(3, 3, heads, kv, dim, cols * page))

    def step():
        kernels.attention_fwd(q, *qkv, starts, out, lse=lse)
        kernels.attention_bwd(q, dout, *qkv, starts, out, lse, *g, workspace=ws)
        kernels.cache_append(q, *x1[1:], one, lengths, table, kc, vc)
        kernels.paged_attention(q, x1[0], kc, vc, one, lengths, table, out1, lse=lse1, workspace=ws1)

    results = [out, lse, *g, out1, lse1]
    with q.capture() as rec:
        step()
    for k, new in enumerate(([600, 3, 111], [640, 1, 112], [17, 16, 0])):
        lengths.buffer.write(q, np.array(new, np.int32))
        step()
        want = [t.numpy(q) for t in results]
        for _ in range(3):
            for t in results:
                t.buffer.fill_u32(q, 0x7FC07FC0)
            rec.graph.launch(q)
            q.sync()
            for t, w in zip(results, want):
                assert np.array_equal(t.numpy(q), w), k
    rec.graph.destroy()


def test_two_queues_at_once(dev, q, own):
    """The same calls on two queues with workspaces of their own."""
    from vernondsl_amd.rhi import Queue
    other = Queue(dev)
    r = np.random.default_rng(11)
    n, heads, kv, dim = 700, 4, 2, 64
    a, b, c = projection(r, n, heads, kv, dim)
    qkv = fused(own, a, b, c)
    starts = own.put(starts_of([n]), "i32")
    dout = own.put(r.standard_normal((n, heads * dim)), "bf16")
    sets = []
    q.sync()
    for _ in range(2):
        sets.append(([own.empty((n, heads * dim), "bf16"), own.empty((heads, n), "f32")], [own.empty((n, h, dim), "f32") for h in (heads, kv, kv)],
                     own.scratch(kernels.attention_bwd_workspace_bytes(n, 1, heads, kv, dim))))
    for _ in range(3):
        for queue, (o, g, ws) in zip((q, other), sets):
            kernels.attention_fwd(queue, *qkv, starts, o[0], lse=o[1])
            kernels.attention_bwd(queue, dout, *qkv, starts, *o, *g, workspace=ws)
    other.sync()
    for x, y in zip(sets[0][0] + sets[0][1], sets[1][0] + sets[1][1]):
        assert np.array_equal(x.numpy(q), y.numpy(q))
    other.destroy()


def refused(status, fn, *a, **kw):
    with pytest.raises(_lib.VdslError) as e:
        fn(*a, **kw)
    assert e.value.status == status, str(e.value)


def test_refusals(dev, q, own):
    INVALID, UNSUPPORTED, SHAPE = -1, -5, -7
    n, heads, kv, dim = 16, 4, 2, 16
    t = {k: own.put(np.ones((n, h, dim)), "bf16") for k, h in (("q", heads), ("k", kv), ("v", kv))}
    starts = own.put(starts_of([n]), "i32")
    out, lse = own.empty((n, heads * dim), "bf16"), own.empty((heads, n), "f32")
    g = [own.empty((n, h, dim), "bf16") for h in (heads, kv, kv)]
    ws = own.scratch(kernels.attention_bwd_workspace_bytes(n, 1, heads, kv, dim))
    small = own.scratch(64)
    dout = own.put(np.ones((n, heads * dim)), "bf16")

    def fwd(**kw):
        a = dict(qh=t["q"], k=t["k"], v=t["v"], starts=starts, out=out, lse=lse)
        a.update(kw)
        kernels.attention_fwd(q, **a)

    def bwd(**kw):
        a = dict(dout=dout, qh=t["q"], k=t["k"], v=t["v"], starts=starts, out=out, lse=lse, dq=g[0], dk=g[1], dv=g[2], workspace=ws)
        a.update(kw)
        kernels.attention_bwd(q, **a)

    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-40, 3e38):
        refused(INVALID, fwd, scale=scale)
        refused(INVALID, bwd, scale=scale)
    refused(INVALID, fwd, out=t["q"].view((n, heads * dim)))
    three = [own.put(np.ones((n, h, dim)), "bf16") for h in (4, 3, 3)]
    refused(INVALID, fwd, qh=three[0], k=three[1], v=three[2])  # 3 does not divide 4
    for d, status in ((12, UNSUPPORTED), (136, UNSUPPORTED)):
        x = [own.put(np.ones((n, h, d)), "bf16") for h in (2, 1, 1)]
        refused(status, fwd, qh=x[0], k=x[1], v=x[2], out=own.empty((n, 2 * d), "bf16"), lse=None)
    odd = own.put(np.ones((n, 8 * dim + 4)), "bf16")  # rows that are no whole 16 bytes; a first column that is none
    refused(UNSUPPORTED, fwd, k=kernels.Heads(odd, kv, dim), v=t["v"])
    even = own.put(np.ones((n, 8 * dim)), "bf16")
    refused(UNSUPPORTED, fwd, k=kernels.Heads(even, kv, dim, 4))
    with pytest.raises(ValueError):
        fwd(k=kernels.Heads(even, kv, dim, 7 * dim))
    with pytest.raises(ValueError):
        fwd(k=own.put(np.ones((n, kv, dim)), "f32"))
    with pytest.raises(ValueError):
        fwd(v=own.put(np.ones((n, 1, dim)), "bf16"))
    refused(SHAPE, bwd, workspace=small)
    for kw in ({"dq": t["q"]}, {"dk": t["v"]}, {"workspace": dout}, {"dk": g[2]}):
        refused(SHAPE if "workspace" in kw and dout.buffer.nbytes < ws.buffer.nbytes else INVALID, bwd, **kw)
    over = own.empty((n, (heads + 2 * kv) * dim), "bf16")  # dk's columns reach into dv's
    refused(INVALID, bwd, dq=kernels.Heads(over, heads, dim), dk=kernels.Heads(over, kv, dim, heads * dim),
            dv=kernels.Heads(over, kv, dim, heads * dim + dim))
    fwd()
    fwd(lse=None)
    fwd(k=t["v"])  # inputs may share
    bwd(dq=kernels.Heads(over, heads, dim), dk=kernels.Heads(over, kv, dim, heads * dim), dv=kernels.Heads(over, kv, dim, (heads + kv) * dim))

    kc, vc = own.put(np.ones((4, kv, 16, dim)), "bf16"), own.put(np.ones((4, kv, 16, dim)), "bf16")
    table, lengths = own.put(np.zeros((1, 4)), "i32"), own.put(np.array([n]), "i32")
    need = kernels.paged_attention_workspace_bytes(n, 1, heads, kv, dim, 64)
    pws = own.scratch(need)
    for page in (24, 8, 1):  # no power of two, less than 16
        refused(UNSUPPORTED, kernels.cache_append, q, t["k"], t["v"], starts, lengths, table, own.put(np.ones((4, kv, page, dim)), "bf16"),
                own.put(np.ones((4, kv, page, dim)), "bf16"))
    refused(INVALID, kernels.cache_append, q, t["k"], t["v"], starts, lengths, table, kc, kc)
    refused(INVALID, kernels.paged_attention, q, t["q"], kc, vc, starts, lengths, table, t["q"].view((n, heads * dim)), workspace=pws)
    with pytest.raises(ValueError):
        kernels.cache_append(q, t["k"], t["v"], starts, lengths, own.put(np.zeros((2, 4)), "i32"), kc, vc)
    with pytest.raises(ValueError):
        kernels.paged_attention(q, t["q"], kc, own.put(np.ones((4, kv, 32, dim)), "bf16"), starts, lengths, table, out, workspace=pws)

    x, y, pos = own.put(np.ones((4, 32)), "f32"), own.empty((4, 32), "bf16"), own.put(np.zeros(4), "i32")
    f = own.put(kernels.rope_frequencies(16), "f32")
    refused(SHAPE, kernels.rope, q, x, pos, f, y, 3, 16)       # 48 columns of 32
    refused(SHAPE, kernels.rope, q, x, pos, f, y, 2, 12)       # 16 columns of a head of 12
    refused(SHAPE, kernels.rope, q, x, pos, f, y, 2, 16, first=8)
    refused(INVALID, kernels.rope, q, x, pos, f, y, 2, 16, magnitude=float("nan"))
    refused(INVALID, kernels.rope, q, x, pos, f, y, 2, 16, first=-8)
    with pytest.raises(ValueError):
        kernels.rope(q, x, own.put(np.zeros(5), "i32"), f, y, 2, 16)
    kernels.rope(q, x, pos, f, y, 2, 16)
    q.sync()
