"""Graphs with embeddings, layer norms and a cross-entropy loss: their ops and gradients as built, on the host."""
import pytest

from vernondsl_amd import graph


def test_token_graph_backward_ops():
    g, grads = graph.token_mlp_train_graph(tokens=256, vocab=1000, dim=64, hidden=256, layers=1)
    kinds = [op.kind for op in g.ops]
    assert kinds == ["embedding", "layer_norm", "linear", "linear", "add", "layer_norm", "linear_xent", "layer_norm_bwd", "cast", "gemm",
                     "gemm_gelu_bwd", "gemm", "gemm", "layer_norm_bwd", "add", "embedding_bwd", "add"]
    assert set(grads) == {"E", "norm0_gamma", "norm0_beta", "norm_out_gamma", "norm_out_beta", "W0_up", "W0_down"}
    for name, d in grads.items():
        assert d.name == "grad_" + name and d.shape == g.values[name].shape and d.dtype == "f32"
    # tied weights: the table's gradient is the sum of the output layer's term and the embedding's
    last = g.ops[-1]
    assert last.outputs[0].name == "grad_E" and [v.producer.kind for v in last.inputs] == ["linear_xent", "embedding_bwd"]


def test_untied_output_layer():
    g, grads = graph.token_mlp_train_graph(tokens=64, vocab=300, dim=64, hidden=128, layers=0, tied=False)
    assert [op.kind for op in g.ops] == ["embedding", "layer_norm", "linear_xent", "layer_norm_bwd", "embedding_bwd"]
    xent = g.ops[2]
    assert grads["W_out"] is xent.outputs[2] and xent.outputs[2].name == "grad_W_out" and grads["E"] is g.ops[-1].outputs[0]
    assert graph.Executable.op_flops(None, xent) == 6 * 64 * 300 * 64


def test_params_that_take_no_gradient_and_no_beta():
    g = graph.Graph()
    x = g.input("X", (32, 64), "bf16")
    gamma = g.param("gamma", (64,), "f32", requires_grad=False)
    w = g.param("W", (40, 64), "bf16")
    h = g.layer_norm(x, gamma)
    loss = g.linear_cross_entropy(h, w, g.input("labels", (32,), "i32"))
    grads = g.backward(loss)
    assert set(grads) == {"W"}
    bwd = next(op for op in g.ops if op.kind == "layer_norm_bwd")
    assert len(bwd.outputs) == 1 and bwd.attrs["dgamma"] is None and bwd.attrs["dbeta"] is None


def test_loss_without_backward_reads_no_gradient():
    g = graph.Graph()
    loss = g.linear_cross_entropy(g.input("X", (8, 16), "bf16"), g.param("W", (20, 16), "bf16"), g.input("labels", (8,), "i32"))
    assert g.ops[0].outputs == [loss] and graph.Executable.op_flops(None, g.ops[0]) == 2 * 8 * 16 * 20


def test_construction_refusals():
    g = graph.Graph()
    x, f = g.input("X", (8, 16), "bf16"), g.input("F", (8, 16), "f32")
    ids, w = g.input("ids", (8,), "i32"), g.param("W", (20, 16), "bf16")
    with pytest.raises(TypeError):
        g.embedding(w, x)
    with pytest.raises(TypeError):
        g.embedding(w, ids, out_dtype="i8")
    with pytest.raises(TypeError):
        g.layer_norm(x, g.param("short", (15,), "f32"))
    with pytest.raises(TypeError):
        g.layer_norm(x, g.param("a", (16,), "f32"), g.param("b", (16,), "bf16"))
    with pytest.raises(TypeError):
        g.linear_cross_entropy(f, w, ids)
    with pytest.raises(ValueError):
        g.linear_cross_entropy(x, g.param("V", (20, 24), "bf16"), ids)
    with pytest.raises(ValueError):
        g.linear_cross_entropy(x, w, g.input("few", (7,), "i32"))
    with pytest.raises(ValueError):
        g.backward(g.layer_norm(x, g.param("g", (16,), "f32")))
