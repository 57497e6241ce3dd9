"""Attention over keys that hold infinities, as masks of them do."""
import numpy as np
import pytest

from test_gpu_attention import make_cache, own, starts_of  # noqa: F401
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
