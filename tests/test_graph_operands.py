"""Graph.backward() gives every param that the loss depends on its whole gradient, whichever operand of an op the param
is, or is upstream of: the backward ops as built, run in 64 bits, against differences of the loss."""
import numpy as np
import pytest

import graph64


def upstream_params(loss):
    seen, stack, out = set(), list(loss.producer.inputs[:2 if loss.producer.kind == "linear_xent" else 1]), set()
    while stack:
        v = stack.pop()
        if v.name in seen:
            continue
        seen.add(v.name)
        if v.kind == "param" and v.requires_grad:
            out.add(v.name)
        if v.producer is not None:
            stack.extend(v.producer.inputs)
    return out


@pytest.mark.parametrize("flags", graph64.FLAGS)
@pytest.mark.parametrize("name", graph64.GRAPHS)
def test_gradients_match_differences(name, flags):
    """With steps t and t / 2 central differences are off by t^2 / 6 and t^2 / 24 times a third derivative, so what the halved
    step leaves is below the change; besides, 64-bit rounding of the loss over the step."""
    g, loss = graph64.GRAPHS[name](**graph64.FLAGS[flags])
    want = upstream_params(loss)
    grads = g.backward(loss)
    assert set(grads) == want and want
    feeds = graph64.inputs(g, 7)
    v = graph64.run(g, feeds)
    assert not any(v[d.name].shape != g.values[p].shape or d.dtype != "f32" for p, d in grads.items())
    for p, d in grads.items():
        u = np.random.default_rng(len(p)).standard_normal(feeds[p].shape)
        base = feeds[p].astype(np.float64)

        def at(t):
            return float(graph64.run(g, {**feeds, p: base + t * u})[loss.name][0])

        d1, d2 = ((at(t) - at(-t)) / (2 * t) for t in (1e-4, 5e-5))
        got = float(np.sum(v[d.name] * u))
        assert abs(got - d2) <= abs(d1 - d2) + 64 * 2.0 ** -52 / 5e-5 * max(1.0, at(0.0)), p


def test_gradient_names():
    """grad_<param> wherever the gradient is a value of its own."""
    for name in ("normed_output_weight", "rows_against_themselves", "norm_of_a_param", "param_rows", "factorised_table", "computed_gain"):
        g, loss = graph64.GRAPHS[name]()
        for p, d in g.backward(loss).items():
            assert d is g.values[d.name] and (d.name == "grad_" + p or (name, p) == ("computed_gain", "a")), (name, p, d.name)


def test_no_gradient_without_a_reader():
    """A frozen table gets none, and no op forms one for the embedding."""
    g, loss = graph64.GRAPHS["frozen_table"]()
    assert "E" not in g.backward(loss) and not any(op.kind == "embedding_bwd" for op in g.ops)
