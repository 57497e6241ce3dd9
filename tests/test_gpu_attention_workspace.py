"""One workspace for attention calls of all sizes, made for the largest of them."""
import numpy as np
import pytest

from test_gpu_attention import own, projection, starts_of  # noqa: F401
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
