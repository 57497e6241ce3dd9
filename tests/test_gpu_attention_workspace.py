"""One workspace for attention calls of all sizes, made for the largest of them."""
import numpy as np
import pytest

import attention64 as ref
from test_gpu_attention import check, make_cache, own, projection, rounding, starts_of  # noqa: F401
from test_gpu_tokens import bf16, get
from vernondsl_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (16, 1, 64)])
def test_gradients_of_all_sizes_in_one_workspace(q, own, heads, kv, dim):
    """Batches of fewer rows, whose rows are split more, in the workspace of the largest one: the bits of workspaces of their own."""
    largest = 2689
    shared = own.scratch(kernels.attention_bwd_workspace_bytes(largest, 3, heads, kv, dim))
    r = np.random.default_rng(dim)
    for lengths in ([largest], [largest - 1], [1216], [703], [300, 0, 400], [64], [1]):
        n = sum(lengths)
        x = [own.put(y, "bf16") for y in projection(r, n, heads, kv, dim)]
        dout, starts = own.put(bf16(r.standard_normal((n, heads * dim))), "bf16"), own.put(starts_of(lengths), "i32")
        out, lse = own.empty((n, heads * dim), "bf16"), own.empty((heads, n), "f32")
        kernels.attention_fwd(q, *x, starts, out, lse=lse)
        found = []
        for ws in (own.scratch(kernels.attention_bwd_workspace_bytes(n, len(lengths), heads, kv, dim)), shared):
            g = [own.empty((n, h, dim), "f32") for h in (heads, kv, kv)]
            kernels.attention_bwd(q, dout, *x, starts, out, lse, *g, workspace=ws)
            found.append([get(q, y) for y in g])
        assert all(np.isfinite(a).all() and np.array_equal(a, b) for a, b in zip(*found)), lengths


@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 64), (8, 2, 128)])
def test_paged_rows_of_all_sizes_in_one_workspace(q, own, heads, kv, dim):
    """Fewer rows have more splits and may need more than many: with the workspace of others, of any size or none, they are right."""
    seqs, page, cols = 4, 16, 128
    r = np.random.default_rng(dim)
    kc, vc = make_cache(r, seqs * cols, kv, page, dim)
    table = r.permutation(seqs * cols).reshape(seqs, cols).astype(np.int32)
    lengths = np.array([2048, 1500, 700, 40], np.int32)
    tk, tv, tl, tt = own.put(kc, "bf16"), own.put(vc, "bf16"), own.put(lengths, "i32"), own.put(table, "i32")

    def size(n):
        return kernels.paged_attention_workspace_bytes(n, seqs, heads, kv, dim, cols * page)

    assert size(16) > size(40) and size(4) > 0
    for new in ([1, 1, 1, 1], [4, 4, 4, 4], [20, 0, 19, 1], [100, 1, 1, 0]):
        n = sum(new)
        a = projection(r, n, heads, kv, dim)[0]
        x, starts = own.put(a, "bf16"), own.put(starts_of(new), "i32")
        want, want_lse, eo, el = ref.paged(*(y.astype(np.float64) for y in (a, kc, vc)), starts_of(new), lengths, table, dim ** -0.5)
        first = None
        for nbytes in (size(n), size(n) + 4, size(40), size(4), 2 * n * heads * (8 + 4 * dim), 4, 0):
            out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
            kernels.paged_attention(q, x, tk, tv, starts, tl, tt, out, lse=lse, workspace=own.scratch(nbytes) if nbytes else None)
            got = get(q, out)
            check(get(q, lse), want_lse, el, "lse")
            check(got.reshape(n, heads, dim), want, eo + rounding("f32", np.abs(want) + eo), "out")
            first = got if first is None else first
            assert nbytes < size(n) or np.array_equal(got, first)
