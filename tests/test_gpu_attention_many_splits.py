"""Single tokens over a paged cache in up to 256 splits, of contexts that fill their table's room and of ones that leave most of the
splits empty."""
import numpy as np
import pytest

import attention64 as ref
from attention64 import U
from test_gpu_attention import check, make_cache, own, projection, rounding, starts_of  # noqa: F401
from test_gpu_tokens import get
from vernondsl_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (64, 4, 1), (96, 6, 2)])
@pytest.mark.parametrize("lengths", [[16384], [16000, 1], [5, 1000, 0]])
def test_many_splits(q, own, lengths, dim, heads, kv):
    page, cols = 64, 256
    seqs, r = len(lengths), np.random.default_rng(dim + sum(lengths))
    used = [-(-n // page) for n in lengths]
    kc, vc = make_cache(r, sum(used), kv, page, dim)
    table, at = np.full((seqs, cols), -1, np.int32), 0
    for s, n in enumerate(used):
        table[s, :n] = at + r.permutation(n)
        at += n
    lengths = np.array(lengths, np.int32)
    new = np.minimum(lengths, 1)
    n, starts = int(new.sum()), starts_of(new)
    a = projection(r, n, heads, kv, dim)[0]
    out, lse = own.empty((n, heads * dim), "f32"), own.empty((heads, n), "f32")
    need = kernels.paged_attention_workspace_bytes(n, seqs, heads, kv, dim, cols * page)
    assert need // (n * heads * (8 + 4 * dim)) == 256
    kernels.paged_attention(q, own.put(a, "bf16"), own.put(kc, "bf16"), own.put(vc, "bf16"), own.put(starts, "i32"), own.put(lengths, "i32"),
                            own.put(table, "i32"), out, lse=lse, workspace=own.scratch(need))
    want, want_lse, eo, el = ref.paged(*(y.astype(np.float64) for y in (a, kc, vc)), starts, lengths, table, dim ** -0.5)
    check(get(q, lse), want_lse, el, "lse")
    check(get(q, out).reshape(n, heads, dim), want, eo + rounding("f32", want) + U * eo, "out")
