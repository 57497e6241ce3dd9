"""Graph.backward beside ops that have no gradient: refused where the loss depends on them, and only there."""
import pytest

from vernondsl_amd import graph


def two_paths():
    """A trained layer, and a paged attention and an int8 layer that serve beside it."""
    g = graph.Graph()
    x = g.input("x", (8, 64), "bf16")
    h = g.linear(x, g.param("w", (64, 64), "bf16"), act="gelu")
    qkv = g.linear(x, g.param("w_qkv", (64, 64), "bf16", requires_grad=False), out_dtype="bf16")
    cache = [g.input(n, (4, 1, 16, 16), "bf16") for n in ("k_cache", "v_cache")]
    served = g.paged_attention(qkv, *cache, g.input("starts", (3,), "i32"), g.input("lengths", (2,), "i32"), g.input("table", (2, 2), "i32"), heads=2)
    small = g.quant_linear(h, g.param("wq", (64, 64), "i8", requires_grad=False), g.param("scale", (64,), "f32", requires_grad=False), relu=False)
    labels = g.input("labels", (8,), "i32")
    return g, h, qkv, served, small, labels


def test_ops_that_the_loss_does_not_reach():
    g, h, _, _, _, labels = two_paths()
    grads = g.backward(g.linear_cross_entropy(h, g.param("w_out", (50, 64), "bf16"), labels))
    assert set(grads) == {"w", "w_out"}
    assert sum(op.kind in ("cache_append", "paged_attention", "w8a8", "w8a8_packed") for op in g.ops) == 3  # they stay


def test_ops_that_the_loss_depends_on():
    g, _, _, _, small, labels = two_paths()
    with pytest.raises(NotImplementedError):
        g.backward(g.linear_cross_entropy(small, g.param("w_out", (50, 64), "bf16"), labels))
    g = graph.Graph()
    qkv = g.linear(g.input("x", (8, 64), "bf16"), g.param("w_qkv", (64, 64), "bf16"), out_dtype="bf16")
    cache = [g.input(n, (4, 1, 16, 16), "bf16") for n in ("k_cache", "v_cache")]
    served = g.paged_attention(qkv, *cache, g.input("starts", (3,), "i32"), g.input("lengths", (2,), "i32"), g.input("table", (2, 2), "i32"), heads=2)
    with pytest.raises(NotImplementedError):
        g.backward(g.linear_cross_entropy(served, g.param("w_out", (50, 32), "bf16"), g.input("labels", (8,), "i32")))
