"""What the operators around an MLP that make it a model of tokens are measured on.

Three operators, each in the directions it is called in: token embedding (lookup, and the gradient of
the table), layer norm (forward, and backward with the reductions of the gain's and the offset's
gradients), and the output layer with its softmax cross entropy over a vocabulary (the loss alone, and
the loss with both gradients).  A case is a dict whose "kind" selects the functions below.

With `own` false, `run` computes the plain form: elementary torch operations in 32 bits, rounded once
at the end.  With `own` true it makes the framework's calls.  A program of this framework holds its
tensors in the framework's own buffers, so for `own` `prepare` copies the inputs into such buffers and
allocates the outputs and the workspace there; the inputs are the same ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}
_EPS = 1e-5


# ---- the framework's device and buffers (only where `own` is true) --------------------------------
class _Context:
    """The device and the queue every call runs on, opened at first use."""
    dev = None
    queue = None


def _open():
    from vernondsl_amd.rhi import Device, Queue
    if _Context.dev is None:
        torch.cuda.init()
        _Context.dev = Device(0)
        _Context.queue = Queue(_Context.dev)
    return _Context.dev, _Context.queue


_TYPESTR = {0: "<f4", 1: "<i2", 2: "|i1", 3: "<i4"}  # by the framework's dtype codes; bf16 as 16-bit words


class _Exported:
    """A framework tensor in the form torch takes device memory in; keeps the tensor alive."""

    def __init__(self, t):
        self.tensor = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": _TYPESTR[t.dtype], "version": 2,
                                         "data": (t.buffer.address(), False), "strides": None}


def _torch(t):
    """The same memory as a torch tensor."""
    x = torch.as_tensor(_Exported(t), device="cuda")
    return x.view(torch.bfloat16) if t.dtype == 1 else x


def _empty(shape, dtype):
    from vernondsl_amd.rhi import Tensor
    return Tensor(_open()[0], shape, dtype)


def _put(x):
    """A framework tensor holding the torch tensor x."""
    t = _empty(tuple(x.shape), {torch.float32: "f32", torch.bfloat16: "bf16", torch.int32: "i32"}[x.dtype])
    _torch(t).copy_(x)
    return t


def _workspace(nbytes):
    return _empty((max(4, nbytes),), "i8")


# ---- inputs --------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype="f32", sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * sigma).to(_TORCH[dtype])


def _tokens(g, n, vocab):
    """Token ids of a heavy-tailed distribution, id 0 the most frequent (vocab^(-1/3) of all); 3 in 100
    are -1: padding."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (u * u * u * vocab).to(torch.int32).clamp(max=vocab - 1)
    return torch.where(torch.rand(n, generator=g, device="cuda") < 0.03, torch.full_like(ids, -1), ids)


def _distinct(n, vocab):
    """How many different ids n of `_tokens` hold, on average."""
    edge = np.cbrt(np.arange(vocab + 1, dtype=np.float64) / vocab)
    return float(np.sum(1.0 - (1.0 - 0.97 * np.diff(edge)) ** n))


# ---- token embedding: y[i] = scale table[ids[i]], zero where ids[i] is no row ---------------------
def _embed_inputs(c, seed):
    g = _generator(seed)
    return {"ids": _tokens(g, c["n"], c["vocab"]), "table": _normal(g, (c["vocab"], c["dim"]), c["table"], 0.02)}


def _embed_plain(c, s):
    valid = (s["ids"] >= 0) & (s["ids"] < c["vocab"])
    rows = s["table"].index_select(0, s["ids"].clamp(0, c["vocab"] - 1)).float()
    return (rows * (valid.float() * math.sqrt(c["dim"]))[:, None]).to(_TORCH[c["out"]])


def _embed_prepare(c, s):
    out = _empty((c["n"], c["dim"]), c["out"])
    return {"ids": _put(s["ids"]), "table": _put(s["table"]), "out": out, "result": _torch(out)}


def _embed_own(c, s, kernels, q):
    kernels.embedding_fwd(q, s["table"], s["ids"], s["out"], scale=math.sqrt(c["dim"]))
    return s["result"]


def _embed_work(c):
    n, d = c["n"], c["dim"]
    return {"bytes": 4 * n + _distinct(n, c["vocab"]) * d * _BYTES[c["table"]] + n * d * _BYTES[c["out"]], "flops": n * d}


def _embed_exact(c, seed):
    s = _embed_inputs(c, seed)
    ids = s["ids"].long()
    table = torch.cat([s["table"].double(), torch.zeros((1, c["dim"]), dtype=torch.float64, device="cuda")])
    return table[torch.where((ids < 0) | (ids >= c["vocab"]), c["vocab"], ids)] * math.sqrt(c["dim"])


# ---- its gradient: dtable[v] = scale sum of dy[i] over the i with ids[i] = v ----------------------
def _embed_grad_inputs(c, seed):
    g = _generator(seed)
    return {"ids": _tokens(g, c["n"], c["vocab"]), "dy": _normal(g, (c["n"], c["dim"]), c["dy"])}


def _embed_grad_plain(c, s):
    valid = (s["ids"] >= 0) & (s["ids"] < c["vocab"])
    at = torch.where(valid, s["ids"], torch.full_like(s["ids"], c["vocab"]))
    sums = torch.zeros((c["vocab"] + 1, c["dim"]), device="cuda").index_add_(0, at, s["dy"].float())
    return sums[:-1] * math.sqrt(c["dim"])


def _embed_grad_prepare(c, s):
    from vernondsl_amd import kernels
    dtable = _empty((c["vocab"], c["dim"]), "f32")
    return {"ids": _put(s["ids"]), "dy": _put(s["dy"]), "dtable": dtable, "result": _torch(dtable),
            "workspace": _workspace(kernels.embedding_bwd_workspace_bytes(c["n"], c["vocab"], c["dim"]))}


def _embed_grad_own(c, s, kernels, q):
    kernels.embedding_bwd(q, s["ids"], s["dy"], s["dtable"], scale=math.sqrt(c["dim"]), workspace=s["workspace"])
    return s["result"]


def _embed_grad_work(c):
    n, d = c["n"], c["dim"]
    return {"bytes": 4 * n + n * d * _BYTES[c["dy"]] + 4 * c["vocab"] * d, "flops": n * d}


def _embed_grad_exact(c, seed):
    # differences of running sums over the tokens in sorted order
    s = _embed_grad_inputs(c, seed)
    ids, order = s["ids"].long().sort(stable=True)
    run = torch.cat([torch.zeros((1, c["dim"]), dtype=torch.float64, device="cuda"), s["dy"].double()[order].cumsum(0)])
    end = torch.searchsorted(ids, torch.arange(c["vocab"] + 1, device="cuda"))
    return (run[end[1:]] - run[end[:-1]]) * math.sqrt(c["dim"])


# ---- layer norm: y = (x - mean) rstd gamma + beta over each row ------------------------------------
def _norm_inputs(c, seed):
    g = _generator(seed)
    rows, cols = c["rows"], c["cols"]
    # activations with a spread and an offset of their own in each column
    x = torch.randn((rows, cols), generator=g, device="cuda") * (0.5 + torch.rand(cols, generator=g, device="cuda"))
    x = (x + 0.5 * torch.randn(cols, generator=g, device="cuda") + 0.25).to(_TORCH[c["x"]])
    return {"x": x, "gamma": 1.0 + _normal(g, (cols,), sigma=0.2), "beta": _normal(g, (cols,), sigma=0.2), "g": g}


def _norm_plain(c, s):
    x = s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((d * d).mean(1) + _EPS)
    return [(d * rstd[:, None] * s["gamma"] + s["beta"]).to(_TORCH[c["y"]]), mean, rstd]


def _norm_prepare(c, s):
    t = {k: _put(s[k]) for k in ("x", "gamma", "beta")}
    out = [_empty((c["rows"], c["cols"]), c["y"]), _empty((c["rows"],), "f32"), _empty((c["rows"],), "f32")]
    return {**t, "out": out, "result": [_torch(o) for o in out]}


def _norm_own(c, s, kernels, q):
    y, mean, rstd = s["out"]
    kernels.layer_norm_fwd(q, s["x"], s["gamma"], s["beta"], y, mean=mean, rstd=rstd, eps=_EPS)
    return s["result"]


def _norm_work(c):
    n = c["rows"] * c["cols"]
    return {"bytes": n * (_BYTES[c["x"]] + _BYTES[c["y"]]) + 8 * c["rows"] + 8 * c["cols"], "flops": 8 * n}


def _norm_exact(c, seed):
    s = _norm_inputs(c, seed)
    var, mean = torch.var_mean(s["x"].double(), 1, unbiased=False)
    y = torch.nn.functional.layer_norm(s["x"].double(), (c["cols"],), s["gamma"].double(), s["beta"].double(), _EPS)
    return [y, mean, (var + _EPS) ** -0.5]


def _norm_grad_inputs(c, seed):
    s = _norm_inputs(c, seed)
    var, mean = torch.var_mean(s["x"].double(), 1, unbiased=False)  # as the forward pass left them, in 32 bits
    s["mean"], s["rstd"] = mean.float(), ((var + _EPS) ** -0.5).float()
    s["dy"] = _normal(s["g"], (c["rows"], c["cols"]), c["dy"])
    return s


def _norm_grad_plain(c, s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["gamma"]
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return [dx.to(_TORCH[c["dx"]]), (dy * h).sum(0), dy.sum(0)]


def _norm_grad_prepare(c, s):
    from vernondsl_amd import kernels
    t = {k: _put(s[k]) for k in ("dy", "x", "gamma", "mean", "rstd")}
    out = [_empty((c["rows"], c["cols"]), c["dx"]), _empty((c["cols"],), "f32"), _empty((c["cols"],), "f32")]
    return {**t, "out": out, "result": [_torch(o) for o in out],
            "workspace": _workspace(kernels.layer_norm_bwd_workspace_bytes(c["rows"], c["cols"]))}


def _norm_grad_own(c, s, kernels, q):
    dx, dgamma, dbeta = s["out"]
    kernels.layer_norm_bwd(q, s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], dx, dgamma=dgamma, dbeta=dbeta,
                           workspace=s["workspace"])
    return s["result"]


def _norm_grad_work(c):
    n = c["rows"] * c["cols"]
    return {"bytes": n * (_BYTES[c["x"]] + _BYTES[c["dy"]] + _BYTES[c["dx"]]) + 8 * c["rows"] + 12 * c["cols"], "flops": 14 * n}


def _norm_grad_exact(c, seed):
    s = _norm_grad_inputs(c, seed)
    x, gamma, beta = (s[k].double().requires_grad_(True) for k in ("x", "gamma", "beta"))
    y = torch.nn.functional.layer_norm(x, (c["cols"],), gamma, beta, _EPS)
    return list(torch.autograd.grad(y, (x, gamma, beta), s["dy"].double()))


# ---- output layer and softmax cross entropy: loss = mean over counted rows of
# ---- logsumexp(z_i) - z_i[label_i], z = x w^T; rows whose label is no column are not counted -------
def _xent_inputs(c, seed):
    g = _generator(seed)
    n, d, v = c["n"], c["dim"], c["vocab"]
    w = _normal(g, (v, d), "bf16", 2.0 / math.sqrt(d))  # logits of spread 2
    labels = _tokens(g, n, v)
    # hidden states that know their label to a different degree: some rows are certain, some are not
    towards = w[labels.clamp(min=0).long()].float()
    towards = towards / towards.norm(dim=1, keepdim=True)
    x = torch.randn((n, d), generator=g, device="cuda") + towards * (7.0 * torch.rand((n, 1), generator=g, device="cuda"))
    return {"x": x.to(torch.bfloat16), "w": w, "labels": labels}


def _xent_parts(c, s):
    """(x, w and the logits in 32 bits, rows that count, a label for every row, 1 / rows that count, lse, loss)."""
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    valid = (s["labels"] >= 0) & (s["labels"] < c["vocab"])
    label = s["labels"].clamp(0, c["vocab"] - 1).long()[:, None]
    top = z.max(1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    inv = 1.0 / valid.sum().clamp(min=1).float()
    each = (lse - z.gather(1, label))[:, 0]
    loss = torch.where(valid, each, torch.zeros_like(each)).sum() * inv
    return x, w, z, valid, label, inv, lse, loss.reshape(1)


def _xent_loss_plain(c, s):
    *_, lse, loss = _xent_parts(c, s)
    return [loss, lse[:, 0]]


def _xent_plain(c, s):
    x, w, z, valid, label, inv, lse, loss = _xent_parts(c, s)
    z.sub_(lse).exp_()
    z.scatter_add_(1, label, torch.full_like(lse, -1.0))
    z.mul_((valid.float() * inv)[:, None])
    return [loss, lse[:, 0], (z @ w).to(_TORCH[c["grads"]]), (z.t() @ x).to(_TORCH[c["grads"]])]


def _xent_tensors(c, s, backward):
    from vernondsl_amd import kernels
    t = {k: _put(s[k]) for k in ("x", "w", "labels")}
    out = [_empty((1,), "f32"), _empty((c["n"],), "f32")]
    if backward:
        out += [_empty((c["n"], c["dim"]), c["grads"]), _empty((c["vocab"], c["dim"]), c["grads"])]
        need = kernels.linear_xent_workspace_bytes(c["n"], c["vocab"], c["dim"], piece=c["piece"])
    else:
        need = kernels.linear_xent_workspace_bytes(c["n"], c["vocab"], c["dim"], backward=False)
    return {**t, "out": out, "result": [_torch(o) for o in out], "workspace": _workspace(need)}


def _xent_loss_prepare(c, s):
    return _xent_tensors(c, s, False)


def _xent_prepare(c, s):
    return _xent_tensors(c, s, True)


def _xent_loss_own(c, s, kernels, q):
    loss, lse = s["out"]
    kernels.linear_xent_fwd(q, s["x"], s["w"], s["labels"], loss, lse=lse, workspace=s["workspace"])
    return s["result"]


def _xent_own(c, s, kernels, q):
    loss, lse, dx, dw = s["out"]
    kernels.linear_xent_fwd_bwd(q, s["x"], s["w"], s["labels"], loss, dx, dw, lse=lse, piece=c["piece"], workspace=s["workspace"])
    return s["result"]


def _xent_loss_work(c):
    n, d, v = c["n"], c["dim"], c["vocab"]
    return {"bytes": 2 * n * d + 2 * v * d + 8 * n, "flops": 2 * n * v * d}


def _xent_work(c):
    n, d, v = c["n"], c["dim"], c["vocab"]
    return {"bytes": (n * d + v * d) * (2 + _BYTES[c["grads"]]) + 8 * n, "flops": 6 * n * v * d}


def _xent_exact(c, seed, backward=True):
    s = _xent_inputs(c, seed)
    x, w = (s[k].double().requires_grad_(backward) for k in ("x", "w"))
    labels = torch.where((s["labels"] < 0) | (s["labels"] >= c["vocab"]), -100, s["labels"].long())
    z = x @ w.t()
    if bool((labels >= 0).any()):
        loss = torch.nn.functional.cross_entropy(z, labels, ignore_index=-100)
    else:
        loss = (z * 0.0).sum()
    outs = [loss.detach().reshape(1), torch.logsumexp(z.detach(), 1)]
    return outs + list(torch.autograd.grad(loss, (x, w))) if backward else outs


def _xent_loss_exact(c, seed):
    with torch.no_grad():
        return _xent_exact(c, seed, backward=False)


# ---- the kinds: inputs, plain form, buffers, the framework's call, work, 64 bits -------------------
_KINDS = {
    "embed": (_embed_inputs, _embed_plain, _embed_prepare, _embed_own, _embed_work, _embed_exact),
    "embed_grad": (_embed_grad_inputs, _embed_grad_plain, _embed_grad_prepare, _embed_grad_own, _embed_grad_work,
                   _embed_grad_exact),
    "norm": (_norm_inputs, _norm_plain, _norm_prepare, _norm_own, _norm_work, _norm_exact),
    "norm_grad": (_norm_grad_inputs, _norm_grad_plain, _norm_grad_prepare, _norm_grad_own, _norm_grad_work, _norm_grad_exact),
    "xent_loss": (_xent_inputs, _xent_loss_plain, _xent_loss_prepare, _xent_loss_own, _xent_loss_work, _xent_loss_exact),
    "xent": (_xent_inputs, _xent_plain, _xent_prepare, _xent_own, _xent_work, _xent_exact),
}


def listed():
    return [
        # the tokens of a few requests that are being served, one each: the smallest call, all latency
        {"name": "embed_8x4096", "kind": "embed", "n": 8, "dim": 4096, "vocab": 32768, "table": "bf16", "out": "bf16"},
        # a training batch's tokens into a 32-bit residual stream
        {"name": "embed_16384x4096", "kind": "embed", "n": 16384, "dim": 4096, "vocab": 32768, "table": "bf16", "out": "f32"},
        # a small model's table: sizes that are no multiple of a tile or of 16 bytes
        {"name": "embed_grad_300x1001", "kind": "embed_grad", "n": 300, "dim": 1001, "vocab": 5003, "dy": "f32"},
        # the table's gradient of a training batch: every row of the table is written, frequent tokens
        # have hundreds of terms and most rows few or none
        {"name": "embed_grad_16384x4096", "kind": "embed_grad", "n": 16384, "dim": 4096, "vocab": 32768, "dy": "bf16"},
        # one token of each of a few requests
        {"name": "norm_8x4096", "kind": "norm", "rows": 8, "cols": 4096, "x": "bf16", "y": "bf16"},
        # a training batch: the 32-bit residual stream into the next product's bf16 operand
        {"name": "norm_16384x4096", "kind": "norm", "rows": 16384, "cols": 4096, "x": "f32", "y": "bf16"},
        # a small model's backward pass, rows that are not whole 16-byte units
        {"name": "norm_grad_300x1001", "kind": "norm_grad", "rows": 300, "cols": 1001, "x": "f32", "dy": "f32", "dx": "f32"},
        # a training batch's backward pass, all in bf16
        {"name": "norm_grad_16384x4096", "kind": "norm_grad", "rows": 16384, "cols": 4096, "x": "bf16", "dy": "bf16", "dx": "bf16"},
        # evaluating a model on a batch of held-out text: no gradient
        {"name": "xent_loss_2048x4096", "kind": "xent_loss", "n": 2048, "dim": 4096, "vocab": 32768},
        # a short sequence's step on a small model: launches and short products
        {"name": "xent_16x512", "kind": "xent", "n": 16, "dim": 512, "vocab": 5003, "grads": "bf16", "piece": 0},
        # a ragged batch, width and vocabulary, the vocabulary in three pieces, the last one short
        {"name": "xent_300x1000", "kind": "xent", "n": 300, "dim": 1000, "vocab": 5003, "grads": "bf16", "piece": 2048},
        # the output layer of a training step, the largest product of the model
        {"name": "xent_8192x4096", "kind": "xent", "n": 8192, "dim": 4096, "vocab": 32768, "grads": "bf16", "piece": 0},
    ]


def _spread(rng, lo, hi):
    """An integer in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _extent(rng, lo, hi, grains):
    """Such an integer, made a multiple of one of `grains`."""
    g = rng.choice(grains)
    return max(g, _spread(rng, lo, hi) // g * g)


def draw(rng):
    kind = rng.choice(sorted(_KINDS))
    dim = _extent(rng, 64, 4096, (1, 8, 64, 256))
    vocab = _extent(rng, 1000, 32768, (1, 1, 8, 256))
    types = ["f32", "bf16"]
    if kind == "embed":
        return {"kind": kind, "n": _spread(rng, 1, 16384), "dim": dim, "vocab": vocab, "table": rng.choice(types),
                "out": rng.choice(types)}
    if kind == "embed_grad":
        return {"kind": kind, "n": _spread(rng, 1, 16384), "dim": dim, "vocab": vocab, "dy": rng.choice(types)}
    cols = _extent(rng, 8, 16384, (1, 1, 8, 256))
    rows = _spread(rng, 1, min(16384, (1 << 26) // cols))
    if kind == "norm":
        return {"kind": kind, "rows": rows, "cols": cols, "x": rng.choice(types), "y": rng.choice(types)}
    if kind == "norm_grad":
        return {"kind": kind, "rows": rows, "cols": cols, "x": rng.choice(types), "dy": rng.choice(types), "dx": rng.choice(types)}
    n = _extent(rng, 1, 8192, (1, 1, 8, 128))
    if kind == "xent_loss":
        return {"kind": kind, "n": n, "dim": dim, "vocab": vocab}
    # 0: the library's own choice of a piece
    piece = rng.choice([0, 0, _extent(rng, 512, 8192, (1, 256))])
    return {"kind": kind, "n": n, "dim": dim, "vocab": vocab, "grads": "bf16", "piece": piece}


def prepare(case, seed):
    inputs, plain, buffers, call = _KINDS[case["kind"]][:4]
    s = inputs(case, seed)
    s.pop("g", None)
    if not own:
        return {"case": case, "s": s, "run": plain}
    from vernondsl_amd import kernels
    state = {"case": case, "s": buffers(case, s), "run": call, "more": (kernels, _open()[1])}
    torch.cuda.synchronize()  # the inputs are in place before the framework's own queue reads them
    return state


def run(state):
    return state["run"](state["case"], state["s"], *state.get("more", ()))


def work(case):
    return _KINDS[case["kind"]][4](case)


def exact(case, seed):
    return _KINDS[case["kind"]][5](case, seed)
