"""An execution graph's ops in 64 bits on the host, and small graphs that reach a param through every operand that has a
gradient.  Nothing is rounded, so a graph's own backward ops can be compared with differences of its loss."""
import numpy as np
from scipy.special import erf

from vernondsl_amd import graph


def gelu_slope(z):
    return 0.5 * (1.0 + erf(z / np.sqrt(2.0))) + z * np.exp(-0.5 * z * z) / np.sqrt(2.0 * np.pi)


def run(g, feeds):
    """{value name: array} after all of g's ops."""
    v = {k: np.asarray(a) if np.asarray(a).dtype.kind == "i" else np.asarray(a, np.float64) for k, a in feeds.items()}
    for op in g.prepare_ops:
        a = v[op.inputs[0].name]
        v[op.outputs[0].name] = a.T if op.kind == "transpose" else a
    for op in g.ops:
        k, out = op.kind, [o.name for o in op.outputs]
        ins = [v[i.name] for i in op.inputs]
        if k == "linear":
            z = ins[0] @ ins[1].T
            if op.attrs["act"] != "none":
                v[op.attrs["pre"].name] = z
            v[out[0]] = {"none": lambda: z, "gelu": lambda: z * 0.5 * (1.0 + erf(z / np.sqrt(2.0))), "relu": lambda: np.maximum(z, 0)}[
                op.attrs["act"]]()
        elif k == "gemm":
            a, b = (ins[0].T if op.attrs["trans_a"] else ins[0]), (ins[1].T if op.attrs["trans_b"] else ins[1])
            v[out[0]] = a @ b
        elif k == "add":
            v[out[0]] = ins[0] + ins[1]
        elif k == "cast":
            v[out[0]] = ins[0]
        elif k == "transpose":
            v[out[0]] = ins[0].T
        elif k in ("gelu_bwd", "relu_bwd"):
            d = ins[0] * (gelu_slope(ins[1]) if k == "gelu_bwd" else ins[1] > 0)
            v[out[0]], v[out[1]] = d, d.T
        elif k == "mse":
            d = ins[0] - ins[1]
            v[out[0]] = np.array([np.mean(d * d)])
            if len(out) > 1:
                v[out[1]], v[out[2]] = 2.0 * d / d.size, 2.0 * d.T / d.size
        elif k == "embedding":
            real = (ins[1] >= 0) & (ins[1] < len(ins[0]))
            v[out[0]] = np.where(real[:, None], ins[0][np.where(real, ins[1], 0)], 0.0) * op.attrs["scale"]
        elif k == "embedding_bwd":
            d = np.zeros(op.outputs[0].shape)
            real = (ins[0] >= 0) & (ins[0] < len(d))
            np.add.at(d, ins[0][real], ins[1][real] * op.attrs["scale"])
            v[out[0]] = d
        elif k == "layer_norm":
            x = ins[0]
            mean = x.mean(1)
            rstd = 1.0 / np.sqrt(((x - mean[:, None]) ** 2).mean(1) + op.attrs["eps"])
            v[out[0]] = (x - mean[:, None]) * rstd[:, None] * ins[1] + (ins[2] if len(ins) > 2 else 0.0)
            v[out[1]], v[out[2]] = mean, rstd
        elif k == "layer_norm_bwd":
            dy, x, gamma, mean, rstd = ins
            h = (x - mean[:, None]) * rstd[:, None]
            d = dy * gamma
            v[out[0]] = rstd[:, None] * (d - d.mean(1, keepdims=True) - h * (d * h).mean(1, keepdims=True))
            for name, term in (("dgamma", dy * h), ("dbeta", dy)):
                if op.attrs[name] is not None:
                    v[op.attrs[name].name] = term.sum(0)
        elif k == "linear_xent":
            x, w, labels = ins
            z = x @ w.T
            lse = z.max(1) + np.log(np.exp(z - z.max(1, keepdims=True)).sum(1))
            counts = (labels >= 0) & (labels < len(w))
            at, rows, inv = np.where(counts, labels, 0), np.arange(len(labels)), 1.0 / max(1, counts.sum())
            v[out[0]] = np.array([np.where(counts, lse - z[rows, at], 0.0).sum() * inv])
            if len(out) > 1:
                d = np.exp(z - lse[:, None])
                d[rows, at] -= 1.0
                d *= (counts * inv)[:, None]
                v[out[1]], v[out[2]] = d @ w, d.T @ x
        else:
            raise NotImplementedError(k)
    return v


N, DIM, VOCAB = 48, 64, 130


def _start(**flags):
    g = graph.Graph(**flags)
    return g, g.input("ids", (N,), "i32"), g.input("labels", (N,), "i32")


def _norm(g, x, name, beta=True):
    return g.layer_norm(x, g.param(name + "_gamma", x.shape[1:], "f32"), g.param(name + "_beta", x.shape[1:], "f32") if beta else None)


def position_table(**flags):
    g, ids, labels = _start(**flags)
    h = g.add(g.embedding(g.param("E", (VOCAB, DIM), "bf16"), ids, 8.0), g.param("P", (N, DIM), "f32"))
    return g, g.linear_cross_entropy(_norm(g, h, "norm"), g.param("W", (VOCAB, DIM), "bf16"), labels)


def normed_output_weight(**flags):
    """The output weights are the norm of the embedding's table."""
    g, ids, labels = _start(**flags)
    e = g.param("E", (VOCAB, DIM), "bf16")
    h = _norm(g, g.embedding(e, ids, 8.0), "norm")
    return g, g.linear_cross_entropy(h, g.layer_norm(e, g.param("g", (DIM,), "f32")), labels)


def rows_against_themselves(**flags):
    g, ids, labels = _start(**flags)
    x = g.param("X", (N, DIM), "bf16")
    return g, g.linear_cross_entropy(x, x, labels)


def computed_rows_against_themselves(**flags):
    g, ids, labels = _start(**flags)
    x = _norm(g, g.param("P", (N, DIM), "f32"), "norm")
    return g, g.linear_cross_entropy(x, x, labels)


def param_rows(**flags):
    g, ids, labels = _start(**flags)
    return g, g.linear_cross_entropy(g.param("P", (N, DIM), "bf16"), g.param("W", (VOCAB, DIM), "bf16"), labels)


def norm_of_a_param(**flags):
    g, ids, labels = _start(**flags)
    return g, g.linear_cross_entropy(_norm(g, g.param("P", (N, DIM), "f32"), "norm"), g.param("W", (VOCAB, DIM), "bf16"), labels)


def factorised_table(**flags):
    g, ids, labels = _start(**flags)
    table = g.linear(g.param("A", (VOCAB, 32), "bf16"), g.param("B", (DIM, 32), "bf16"))
    h = _norm(g, g.embedding(table, ids, 2.0), "norm")
    return g, g.linear_cross_entropy(h, g.param("W", (VOCAB, DIM), "bf16"), labels)


def computed_gain(**flags):
    """The gain is a sum of two params, one of them another norm's offset too."""
    g, ids, labels = _start(**flags)
    b = g.param("b", (DIM,), "f32")
    gain = g.add(g.param("a", (DIM,), "f32"), b)
    h = g.layer_norm(g.embedding(g.param("E", (VOCAB, DIM), "f32"), ids), gain, b)
    return g, g.linear_cross_entropy(h, g.param("W", (VOCAB, DIM), "bf16"), labels)


def computed_linear_weight(**flags):
    """A linear layer on a param, and one whose weight is a norm's output."""
    g, ids, labels = _start(**flags)
    u = g.linear(g.param("P", (N, DIM), "bf16"), g.param("U", (96, DIM), "bf16"), act="gelu")
    y = g.linear(u, _norm(g, g.param("V", (40, 96), "f32"), "norm", beta=False))
    return g, g.mse_loss(y, g.input("T", (N, 40), "f32"))


def param_in_a_square_loss(**flags):
    """A param is the loss's own operand."""
    g, ids, labels = _start(**flags)
    p = g.param("P", (N, 40), "f32")
    return g, g.mse_loss(p, g.input("T", (N, 40), "f32"))


def param_added_to_itself(**flags):
    g, ids, labels = _start(**flags)
    p = g.param("P", (N, 40), "f32")
    y = g.add(g.add(p, p), g.linear(g.input("X", (N, DIM), "bf16"), g.param("W", (40, DIM), "bf16")))
    return g, g.mse_loss(y, g.input("T", (N, 40), "f32"))


def untied_without_offsets(**flags):
    g, ids, labels = _start(**flags)
    h = _norm(g, g.embedding(g.param("E", (VOCAB, DIM), "bf16"), ids, 8.0), "norm", beta=False)
    return g, g.linear_cross_entropy(h, g.param("W", (VOCAB, DIM), "bf16"), labels)


def frozen_table(**flags):
    """The table, which is the output weights too, takes no gradient."""
    g, ids, labels = _start(**flags)
    e = g.param("E", (VOCAB, DIM), "bf16", requires_grad=False)
    h = g.embedding(e, ids, 8.0)
    h = g.add(h, g.linear(_norm(g, h, "norm"), g.param("W", (DIM, DIM), "bf16"), act="relu"))
    return g, g.linear_cross_entropy(_norm(g, h, "norm_out", beta=False), e, labels)


GRAPHS = {f.__name__: f for f in (position_table, normed_output_weight, rows_against_themselves, computed_rows_against_themselves, param_rows,
                                  norm_of_a_param, factorised_table, computed_gain, computed_linear_weight, param_in_a_square_loss,
                                  param_added_to_itself, untied_without_offsets, frozen_table)}
FLAGS = {"plain": {}, "prepared": dict(prepare_transposes=True, fuse_gelu_backward=False, k_major_grads=True)}


def inputs(g, seed):
    """Values for g's inputs and params: gains about 1, matrices of unit rows."""
    r = np.random.default_rng(seed)
    feeds = {}
    made = {o.name for op in g.prepare_ops for o in op.outputs}
    for v in g.values.values():
        if v.name in made or v.kind not in ("input", "param"):
            continue
        if v.dtype == "i32":
            feeds[v.name] = r.integers(-1, VOCAB + 1, v.shape).astype(np.int32)
        else:
            gain = 1.0 if v.name in ("g", "a") or v.name.endswith("gamma") else 0.0
            x = r.standard_normal(v.shape) * (0.2 if len(v.shape) == 1 else 1.0 if v.name == "T" else v.shape[-1] ** -0.5) + gain
            feeds[v.name] = x.astype(np.float32)
    return feeds
