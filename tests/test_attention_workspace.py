"""The sizes of the attention operators' workspaces over batches of different sizes."""
import numpy as np
import pytest

from vernondsl_amd import kernels


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (32, 8, 128), (8, 1, 64), (16, 16, 64), (64, 1, 128), (300, 150, 8), (4, 2, 80)])
def test_gradient_of_fewer_rows_needs_no_more(heads, kv, dim):
    """One workspace, made for the largest batch, serves every smaller one (rows and sequences vary from step to step)."""
    sizes = np.unique(np.concatenate([np.arange(300), np.arange(300, 3000, 7), 64 * np.arange(1, 80), 64 * np.arange(1, 80) + 1]))
    need = np.array([[kernels.attention_bwd_workspace_bytes(int(n), s, heads, kv, dim) for n in sizes] for s in (0, 1, 2, 5, 64, 1000)])
    assert (np.diff(need, axis=0) >= 0).all() and (np.diff(need, axis=1) >= 0).all()
