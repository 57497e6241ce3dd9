"""A training step of the token model on the device (embedding, layer norms, residual MLP, cross entropy with tied
weights; one captured graph) against the same step in 64 bits with the graph's bf16 roundings left out.

Each value passes a handful of bf16 roundings (weights are exact: bf16 on both sides): the norm's output, the MLP's
activation, and on the way back G, the gradient into each linear layer and through GELU'.  One moves a tensor by at
most 2^-8 of each element, so by 2^-8 of its norm; no gradient passes more than 12 of them: 12 * 2^-8 = 4.7e-2 in
norm if they all pointed one way."""
import numpy as np
import pytest

from vernondsl_amd import graph, rng
from vernondsl_amd.examples import token_model

pytestmark = pytest.mark.gpu
REL = 12 * 2.0 ** -8


def erf(x):
    from math import erf as e
    return np.vectorize(e)(x)


def layer_norm(x, gamma, beta):
    mean = x.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + 1e-5)
    h = (x - mean) * rstd

    def back(dy):
        g = dy * gamma
        return rstd * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True)), (dy * h).sum(0), dy.sum(0)

    return h * gamma + beta, back


def step64(p, ids, labels, layers):
    """(loss, gradients) of token_mlp_train_graph's step, tied weights."""
    dim = p["E"].shape[1]
    d = {n: np.zeros_like(v) for n, v in p.items()}
    real = (ids >= 0) & (ids < len(p["E"]))
    h = np.where(real[:, None], p["E"][np.where(real, ids, 0)], 0.0) * np.sqrt(dim)
    backs = []
    for k in range(layers):
        a, norm_back = layer_norm(h, p[f"norm{k}_gamma"], p[f"norm{k}_beta"])
        z = a @ p[f"W{k}_up"].T
        phi = 0.5 * (1.0 + erf(z / np.sqrt(2.0)))
        u = z * phi
        backs.append((a, norm_back, phi + z * np.exp(-0.5 * z * z) / np.sqrt(2.0 * np.pi), u))
        h = h + u @ p[f"W{k}_down"].T
    a, norm_back = layer_norm(h, p["norm_out_gamma"], p["norm_out_beta"])
    z = a @ p["E"].T
    lse = z.max(1) + np.log(np.exp(z - z.max(1, keepdims=True)).sum(1))
    counts = (labels >= 0) & (labels < len(p["E"]))
    at, rows, inv = np.where(counts, labels, 0), np.arange(len(labels)), 1.0 / max(1, counts.sum())
    loss = np.where(counts, lse - z[rows, at], 0.0).sum() * inv
    g = np.exp(z - lse[:, None])
    g[rows, at] -= 1.0
    g *= (counts * inv)[:, None]
    d["E"] += g.T @ a
    dh, d["norm_out_gamma"], d["norm_out_beta"] = norm_back(g @ p["E"])
    for k in reversed(range(layers)):
        a, norm_back, slope, u = backs[k]
        d[f"W{k}_down"] = dh.T @ u
        dz = (dh @ p[f"W{k}_down"]) * slope
        d[f"W{k}_up"] = dz.T @ a
        dx, d[f"norm{k}_gamma"], d[f"norm{k}_beta"] = norm_back(dz @ p[f"W{k}_up"])
        dh = dh + dx
    np.add.at(d["E"], ids[real], dh[real] * np.sqrt(dim))
    return loss, d


# whole packed tiles; a ragged batch and vocabulary in pieces; unpacked widths
@pytest.mark.parametrize("tokens,vocab,dim,hidden,layers,piece", [(256, 512, 256, 512, 1, 0), (300, 1003, 64, 128, 2, 256), (40, 77, 96, 160, 2, 0)])
def test_training_step_matches_64_bits(dev, q, tokens, vocab, dim, hidden, layers, piece):
    r = np.random.default_rng(tokens)
    g, grads = graph.token_mlp_train_graph(tokens, vocab, dim, hidden, layers, piece=piece)
    exe = g.compile(dev)
    p = {}
    for n in grads:
        v = g.values[n]
        x = r.standard_normal(v.shape) * (1.0 / np.sqrt(v.shape[-1]) if len(v.shape) == 2 else 0.2) + (1.0 if n.endswith("gamma") else 0.0)
        x = x.astype(np.float32)
        exe.write(q, n, rng.f32_to_bf16(x) if v.dtype == "bf16" else x)
        p[n] = (rng.bf16_to_f32(rng.f32_to_bf16(x)) if v.dtype == "bf16" else x).astype(np.float64)
    ids = r.integers(-1, vocab + 1, tokens).astype(np.int32)
    labels = r.integers(-1, vocab + 1, tokens).astype(np.int32)
    exe.write(q, "ids", ids)
    exe.write(q, "labels", labels)
    exe.run(q)
    names = ["loss"] + [d.name for d in grads.values()]
    eager = {n: exe.read(q, n) for n in names}
    loss, want = step64(p, ids, labels, layers)
    assert abs(float(eager["loss"][0]) - loss) <= REL * abs(loss)
    for n, d in grads.items():
        got = eager[d.name].astype(np.float64)
        assert np.linalg.norm(got - want[n]) <= REL * np.linalg.norm(want[n]), n
    step = exe.capture(q)
    for _ in range(3):
        for n in names:
            exe.t[n].buffer.fill_u32(q, 0x7FC07FC0)
        q.sync()
        step.launch(q)
        q.sync()
        for n in names:
            assert np.array_equal(exe.read(q, n), eager[n]), f"replay differs from the eager run in {n}"
    step.destroy()
    exe.free()


def test_example_learns():
    """The example's loss falls from about log(kinds) (nothing known) to well below the entropy of single characters:
    the model has learnt from the character before."""
    ids, kinds = token_model.text_tokens()
    share = np.bincount(ids) / len(ids)
    entropy = -np.sum(share * np.log(share))
    losses = token_model.train(steps=60)
    assert abs(losses[0] - np.log(kinds)) < 0.5
    assert np.mean(losses[-5:]) < entropy - 0.3
