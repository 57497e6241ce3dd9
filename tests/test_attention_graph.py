"""Graphs with rotary positions and attention on the host: gradients against differences, ops as built, refusals; and the plain
forms that the device is compared with against differences and each other."""
import numpy as np
import pytest

import attention64
import attention_graph64 as ag
from vernondsl_amd import graph, kernels


@pytest.mark.parametrize("flags", [{}, dict(prepare_transposes=True, k_major_grads=True)])
@pytest.mark.parametrize("layers,tied,causal", [(1, True, True), (2, False, True), (1, False, False)])
def test_gradients_match_differences(flags, layers, tied, causal):
    """As in test_graph_operands: the difference quotients of two steps bound each other's error; besides, the loss's rounding."""
    vocab, lengths = 19, [7, 0, 9, 1]
    g, loss = ag.plain_transformer(20, 4, vocab, 16, 4, 2, 8, 24, layers, tied, causal, **flags)
    grads = g.backward(loss)
    assert set(grads) == {v.name for v in g.values.values() if v.kind == "param" and v.requires_grad and not v.producer}
    feeds = {**ag.weights(g, 3), **ag.packed_inputs(np.random.default_rng(5), 20, lengths, vocab, 8, front=1)}
    v = ag.run(g, feeds)
    for p, d in grads.items():
        u = np.random.default_rng(len(p)).standard_normal(feeds[p].shape)
        base = feeds[p].astype(np.float64)

        def at(t):
            return float(ag.run(g, {**feeds, p: base + t * u})[loss.name][0])

        d1, d2 = ((at(t) - at(-t)) / (2 * t) for t in (1e-4, 5e-5))
        assert abs(float(np.sum(v[d.name] * u)) - d2) <= abs(d1 - d2) + 64 * 2.0 ** -52 / 5e-5 * max(1.0, at(0.0)), p


def test_serving_in_steps_is_the_whole_forward_pass():
    """Chunks and single tokens over the cache give what all tokens at once give, in 64 bits."""
    model = dict(vocab=23, dim=16, heads=4, kv_heads=2, head_dim=8, hidden=24, layers=2)
    r = np.random.default_rng(1)
    whole, loss = ag.plain_transformer(20, 2, **model)
    w = ag.weights(whole, 2)
    texts = [r.integers(0, 23, n).astype(np.int32) for n in (13, 7)]
    feeds = {"ids": np.concatenate(texts), "labels": np.zeros(20, np.int32), "positions": np.concatenate([np.arange(13), np.arange(7)]).astype(np.int32),
             "starts": np.array([0, 13, 20], np.int32), "freqs": kernels.rope_frequencies(8)}
    v = ag.run(whole, {**w, **feeds})
    h = v[loss.producer.inputs[0].name]
    want = h @ w["E"].astype(np.float64).T
    serve = graph.token_transformer_serve_graph(rows=8, seqs=2, pages=4, page=16, pages_per_seq=2, **model)
    caches = {n: np.zeros(x.shape) for n, x in serve.values.items() if "cache" in n}
    table, done = np.array([[2, 0], [1, 3]], np.int32), [0, 0]
    while done != [13, 7]:
        new = [min(n, 13 - done[0] if s == 0 else 7 - done[1]) for s, n in enumerate(r.integers(0, 5, 2))]
        ids, positions = np.full(8, -1, np.int32), np.zeros(8, np.int32)
        parts = [(s, done[s] + i) for s in range(2) for i in range(new[s])]
        for k, (s, i) in enumerate(parts):
            ids[k], positions[k] = texts[s][i], i
        done = [d + n for d, n in zip(done, new)]
        feeds = {"ids": ids, "positions": positions, "starts": np.array([0, new[0], sum(new)], np.int32), "lengths": np.array(done, np.int32),
                 "table": table, "freqs": kernels.rope_frequencies(8)}
        out = ag.run(serve, {**w, **feeds, **caches})["logits"]
        for k, (s, i) in enumerate(parts):
            assert np.allclose(out[k], want[13 * s + i], rtol=1e-9, atol=1e-9)


def test_ops_as_built():
    g, grads = graph.token_transformer_train_graph(tokens=256, seqs=3, vocab=1000, dim=64, heads=4, kv_heads=2, head_dim=32, hidden=256, layers=1)
    kinds = [op.kind for op in g.ops]
    assert kinds[:9] == ["embedding", "layer_norm", "linear", "rope", "attention", "linear", "add", "layer_norm", "linear"]
    assert kinds.count("attention_bwd") == 1 and kinds.count("rope") == 2
    bwd = next(op for op in g.ops if op.kind == "attention_bwd")
    assert bwd.outputs[0].shape == (256, 8 * 32) and next(op for op in g.ops if op.attrs.get("inverse")).inputs[0] is bwd.outputs[0]
    for name, d in grads.items():
        assert d.name == "grad_" + name and d.shape == g.values[name].shape
    s = graph.token_transformer_serve_graph(rows=16, seqs=2, vocab=100, dim=64, heads=4, kv_heads=2, head_dim=32, hidden=128, layers=2)
    assert [op.kind for op in s.ops].count("cache_append") == 2 and s.values["logits"].shape == (16, 100)
    assert {n for n in s.values if s.values[n].kind == "param" and not s.values[n].producer} == set(
        graph.token_transformer_train_graph(16, 2, 100, 64, 4, 2, 32, 128, 2)[1])
    with pytest.raises(NotImplementedError):  # serving has no gradient
        h = s.layer_norm(s.values["paged_attention#" + [n for n in s.values if n.startswith("paged_attention")][0].split("#")[1]], s.param("x", (128,), "f32"))
        s.backward(s.linear_cross_entropy(h, s.param("y", (10, 128), "bf16"), s.input("z", (16,), "i32")))


def test_construction_refusals():
    g = graph.Graph()
    x, f = g.input("X", (8, 96), "bf16"), g.input("F", (8, 96), "f32")
    positions, starts, freqs = g.input("p", (8,), "i32"), g.input("s", (3,), "i32"), g.input("f", (2, 8), "f32")
    for bad in (lambda: g.attention(f, starts, 4, 1), lambda: g.attention(x, freqs, 4, 1), lambda: g.attention(x, starts, 4, 1, out_dtype="i8"),
                lambda: g.rope(x, starts, freqs, 6, 16), lambda: g.rope(x, positions, g.input("f3", (3, 8), "f32"), 6, 16),
                lambda: g.rope(x, positions, freqs, 6, 14)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: g.attention(x, starts, 3, 2), lambda: g.attention(x, starts, 5, 5), lambda: g.rope(x, positions, freqs, 7, 16),
                lambda: g.rope(x, positions, freqs, 6, 16, first=16)):
        with pytest.raises(ValueError):
            bad()
    cache, lengths, table = g.input("c", (4, 1, 16, 16), "bf16"), g.input("l", (2,), "i32"), g.input("t", (2, 4), "i32")
    g.paged_attention(x, cache, cache, starts, lengths, table, 4)
    with pytest.raises(TypeError):
        g.paged_attention(x, cache, cache, starts, g.input("l3", (3,), "i32"), table, 4)
    with pytest.raises(ValueError):
        g.paged_attention(x, cache, cache, starts, lengths, table, 3)


def test_plain_gradient_against_differences():
    r = np.random.default_rng(4)
    n, starts = 14, np.array([1, 6, 6, 12], np.int32)
    for causal in (True, False):
        x = [r.standard_normal((n, h, 8)) for h in (4, 2, 2)]
        dout = r.standard_normal((n, 4, 8))
        out, lse, _, _ = attention64.packed(*x, starts, 0.4, causal)
        grads, _ = attention64.packed_grad(*x, out, np.where(np.isfinite(lse), lse, 0), dout, starts, 0.4, causal)
        for i in range(3):
            u = r.standard_normal(x[i].shape)

            def at(t):
                y = list(x)
                y[i] = x[i] + t * u
                return float(np.sum(attention64.packed(*y, starts, 0.4, causal)[0] * dout))

            d1, d2 = ((at(t) - at(-t)) / (2 * t) for t in (1e-4, 5e-5))
            assert abs(float(np.sum(grads[i] * u)) - d2) <= abs(d1 - d2) + 1e-9


def test_rope_frequencies():
    """Turns per position in two parts hold 48 bits; stretched kinds keep or divide the ends they say."""
    f = kernels.rope_frequencies(128)
    turns = 10000.0 ** (-np.arange(64) / 64) / (2 * np.pi)
    assert f.dtype == np.float32 and f.shape == (2, 64)
    assert np.all(np.abs(f.astype(np.float64).sum(0) - turns) <= 2.0 ** -48 * turns)
    whole = {k: kernels.rope_frequencies(64, factor=8.0, trained=4096, kind=k).astype(np.float64).sum(0) for k in ("linear", "base", "ramp")}
    one = kernels.rope_frequencies(64).astype(np.float64).sum(0)
    assert np.allclose(whole["linear"], one / 8) and np.allclose(whole["base"][0], one[0]) and np.allclose(whole["base"][-1], one[-1] / 8)
    assert np.allclose(whole["ramp"][one * 4096 > 40], one[one * 4096 > 40]) and np.allclose(whole["ramp"][one * 4096 < 0.8], one[one * 4096 < 0.8] / 8)
    assert np.all(np.diff(whole["ramp"]) < 0)
    for bad in (dict(rot=7), dict(rot=8, base=1.0), dict(rot=8, factor=0.5), dict(rot=8, factor=2.0), dict(rot=8, factor=2.0, trained=8, kind="x"),
                dict(rot=2, factor=2.0, kind="base")):
        with pytest.raises(ValueError):
            kernels.rope_frequencies(**bad)
