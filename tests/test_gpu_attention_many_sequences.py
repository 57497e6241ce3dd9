"""Attention of few rows among very many sequences, most of them empty: launches of as many blocks as there are places."""
import numpy as np
import pytest

import attention64 as ref
from attention64 import U
from test_gpu_attention import check, make_cache, own, projection, rounding, starts_of  # noqa: F401
from test_gpu_tokens import bf16, get
from vernondsl_amd import _lib, kernels

pytestmark = pytest.mark.gpu


def scattered(seqs, at):
    """Starts of `seqs` sequences of which sequence s has at[s] rows, and those of the others left out."""
    lengths = np.zeros(seqs, np.int64)
    lengths[list(at)] = list(at.values())
    return starts_of(lengths), starts_of(lengths[lengths > 0])


def test_forward(q, own):
    """More than 2^23 blocks: too many for a launch of 512 lanes each."""
    seqs, heads, dim = (1 << 20) + 3, 8, 8
    starts, few = scattered(seqs, {0: 3, 700001: 2, seqs - 1: 4})
    n = int(few[-1])
    a, b, c = projection(np.random.default_rng(1), n, heads, heads, dim)
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    x, ts = [own.put(y, "bf16") for y in (a, b, c)], own.put(starts, "i32")
    kernels.attention_fwd(q, *x, ts, out, lse=lse)
    want, want_lse, eo, el = ref.packed(*(y.astype(np.float64) for y in (a, b, c)), few, dim ** -0.5, True)
    check(get(q, lse), want_lse, el, "lse")
    check(get(q, out).reshape(n, heads, dim), want, eo + rounding("f32", want) + U * eo, "out")
    with pytest.raises(_lib.VdslError) as e:  # the gradient's blocks would be too many
        kernels.attention_bwd(q, out, *x, ts, out, lse, *[own.empty((n, heads, dim), "f32") for _ in range(3)],
                              workspace=own.scratch(kernels.attention_bwd_workspace_bytes(n, seqs, heads, heads, dim)))
    assert e.value.status == -5


def test_gradient(q, own):
    """Keys whose rows are split, and sixteen blocks each to add the parts up: 2^32 lanes and more."""
    seqs, heads, dim, n = 1200000, 2048, 8, 2
    starts, few = scattered(seqs, {5: 1, 999999: 1})
    r = np.random.default_rng(2)
    a, b, c = projection(r, n, heads, 1, dim)
    d = bf16(r.standard_normal((n, heads, dim)))
    x, ts = [own.put(y, "bf16") for y in (a, b, c)], own.put(starts, "i32")
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    kernels.attention_fwd(q, *x, ts, out, lse=lse)
    g = [own.empty((n, h, dim), "f32") for h in (heads, 1, 1)]
    kernels.attention_bwd(q, own.put(d.reshape(n, -1), "bf16"), *x, ts, out, lse, *g,
                          workspace=own.scratch(kernels.attention_bwd_workspace_bytes(n, seqs, heads, 1, dim)))
    want, bound = ref.packed_grad(*(y.astype(np.float64) for y in (a, b, c)), get(q, out).reshape(n, heads, dim), get(q, lse), d.astype(np.float64), few,
                                  dim ** -0.5, True)
    for y, w, e, name in zip(g, want, bound, ("dq", "dk", "dv")):
        check(get(q, y), w, e + rounding("f32", np.abs(w) + e), name)


def test_paged(q, own):
    """One row among 40000 sequences with room for 2^16 positions each: as many splits as a launch has blocks for."""
    seqs, heads, dim, page, at, length = 40000, 8, 8, 1 << 16, 30003, 1105
    r = np.random.default_rng(3)
    kc, vc = make_cache(r, 1, heads, page, dim)
    table, lengths = np.full((seqs, 1), -1, np.int32), np.zeros(seqs, np.int32)
    table[at], lengths[at] = 0, length
    starts = scattered(seqs, {at: 1})[0]
    a = projection(r, 1, heads, heads, dim)[0]
    out, lse = own.empty((1, heads * dim), "f32"), own.empty((heads, 1), "f32")
    need = kernels.paged_attention_workspace_bytes(1, seqs, heads, heads, dim, page)
    splits = need // (heads * (8 + 4 * dim))
    assert 1 < splits < kernels.paged_attention_workspace_bytes(1, 1, heads, heads, dim, page) // (heads * (8 + 4 * dim))
    kernels.paged_attention(q, own.put(a, "bf16"), own.put(kc, "bf16"), own.put(vc, "bf16"), own.put(starts, "i32"), own.put(lengths, "i32"),
                            own.put(table, "i32"), out, lse=lse, workspace=own.scratch(need))
    want, want_lse, eo, el = ref.paged(*(y.astype(np.float64) for y in (a, kc, vc)), starts_of([1]), lengths[at:at + 1], table[at:at + 1], dim ** -0.5)
    check(get(q, lse), want_lse, el, "lse")
    check(get(q, out).reshape(1, heads, dim), want, eo + rounding("f32", want) + U * eo, "out")
