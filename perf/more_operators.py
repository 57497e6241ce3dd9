"""What the operators that let the rows of a sequence see each other are measured on.

Rotary positions (forward and gradient), attention over packed sequences (forward and gradient), the
append of new rows to a paged cache, and attention of new rows over such a cache.  A case is a dict
whose "kind" selects the functions below.

With `own` false, `run` computes the plain form: elementary torch operations in 32 bits, rounded once
at the end (angles in 64 bits: those of far positions hold nothing in 32).  With `own` true it makes
the framework's calls, on the framework's own buffers, as perf/operators.py does.

Sequences are rows [starts[s], starts[s + 1]) of the tensors; rows behind the last one belong to none
(a padded batch).  Their lengths follow from a case's "rows", "seqs" and "split" alone.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}


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


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(c):
    """Lengths of the case's sequences: they add up to "rows" and are of all sizes, some of them empty; one row
    each where there are as many of both (single tokens that are being served)."""
    rng, seqs, rows = random.Random(c["split"]), c["seqs"], c["rows"]
    if seqs in (1, rows):
        return [rows // seqs] * seqs
    share = [0.0 if rng.random() < 0.1 else rng.uniform(0.1, 1.0) ** 2 for _ in range(seqs - 1)] + [0.5]
    out = [int(rows * x / sum(share)) for x in share]
    out[-1] += rows - sum(out)
    return out


def _starts(lengths):
    return [sum(lengths[:s]) for s in range(len(lengths) + 1)]


def _scale(c):
    return 1.0 / math.sqrt(c["dim"])


# ---- rotary positions: the pair (a, b) of a head at position p turned by the angle p f --------------
# ---- pairs: columns (i, i + rot / 2) or (2 i, 2 i + 1) of the head's first `rot`; the rest stays ----
_ROPE_BASE, _ROPE_TRAINED = 10000.0, 4096  # positions up to 4096 are the trained ones; a factor stretches them


def _frequency(c, i):
    """Radians per position of pair i.  With a factor: frequencies that turn less than once over the trained
    positions are divided by it, those that turn more than 32 times are kept, a ramp between."""
    f = _ROPE_BASE ** (-2.0 * i / c["rot"])
    if c["factor"] == 1.0:
        return f
    edge = [c["rot"] * math.log(_ROPE_TRAINED / (2.0 * math.pi * turns)) / (2.0 * math.log(_ROPE_BASE)) for turns in (32.0, 1.0)]
    lo, hi = max(0, math.floor(edge[0])), min(c["rot"] - 1, math.ceil(edge[1]))
    ramp = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
    return f * (1.0 - ramp) + f / c["factor"] * ramp


def _magnitude(c):
    return 0.1 * math.log(c["factor"]) + 1.0


def _rope_inputs(c, seed):
    g = _generator(seed)
    width = (c["heads"] + c["rest"]) * c["dim"]
    # far into a long context, each sequence from a place of its own
    lengths = _lengths(c)
    first = torch.randint(0, c["reach"], (len(lengths),), generator=g, device="cuda").tolist()
    positions = [torch.arange(n, device="cuda") + p for n, p in zip(lengths, first)]
    return {"x": _normal(g, (c["rows"], width), c["x"]), "positions": torch.cat(positions).to(torch.int32)}


def _rope_plain(c, s):
    dim, rot, heads = c["dim"], c["rot"], c["heads"]
    x = s["x"].float().reshape(c["rows"], -1, dim)
    f = torch.tensor([_frequency(c, i) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    angle = s["positions"].double()[:, None] * f
    sign = -1.0 if c["inverse"] else 1.0
    cos, sin = (torch.cos(angle) * _magnitude(c)).float()[:, None], (torch.sin(angle) * (sign * _magnitude(c))).float()[:, None]
    y = x.clone()
    at = [slice(0, rot, 2), slice(1, rot, 2)] if c["interleaved"] else [slice(0, rot // 2), slice(rot // 2, rot)]
    a, b = (x[:, :heads, k] for k in at)
    y[:, :heads, at[0]] = a * cos - b * sin
    y[:, :heads, at[1]] = a * sin + b * cos
    return y.reshape(c["rows"], -1).to(_TORCH[c["y"]])


def _rope_prepare(c, s):
    from vernondsl_amd import kernels
    freqs = kernels.rope_frequencies(c["rot"], _ROPE_BASE, factor=c["factor"], trained=_ROPE_TRAINED)
    out = _empty(tuple(s["x"].shape), c["y"])
    return {"x": _put(s["x"]), "positions": _put(s["positions"]), "freqs": _put(torch.from_numpy(freqs)), "out": out,
            "result": _torch(out)}


def _rope_own(c, s, kernels, q):
    kernels.rope(q, s["x"], s["positions"], s["freqs"], s["out"], c["heads"], c["dim"], interleaved=c["interleaved"],
                 inverse=c["inverse"], magnitude=_magnitude(c))
    return s["result"]


def _rope_work(c):
    n = c["rows"] * (c["heads"] + c["rest"]) * c["dim"]
    return {"bytes": n * (_BYTES[c["x"]] + _BYTES[c["y"]]) + 4 * c["rows"], "flops": 3 * c["rows"] * c["heads"] * c["rot"]}


def _rope_exact(c, seed):
    # complex numbers a + i b times m e^(i t)
    s = _rope_inputs(c, seed)
    rows, rot, half = c["rows"], c["rot"], c["rot"] // 2
    x = s["x"].double().reshape(rows, -1, c["dim"])
    turned = x[:, :c["heads"], :rot]
    pairs = turned.reshape(rows, -1, half, 2) if c["interleaved"] else turned.reshape(rows, -1, 2, half).transpose(2, 3)
    f = np.array([_frequency(c, i) for i in range(half)])
    t = torch.outer(s["positions"].double(), torch.from_numpy(f).cuda()) * (-1.0 if c["inverse"] else 1.0)
    w = torch.polar(torch.full_like(t, _magnitude(c)), t)[:, None]
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
    z = z.reshape(rows, -1, rot) if c["interleaved"] else z.transpose(2, 3).reshape(rows, -1, rot)
    return torch.cat([torch.cat([z, x[:, :c["heads"], rot:]], 2), x[:, c["heads"]:]], 1).reshape(rows, -1)


# ---- attention over packed sequences: o_i = sum_j p_ij v_j, p_ij = exp(scale q_i k_j - lse_i), over the --
# ---- visible j of i's sequence (j <= i where causal), lse_i = log sum_j exp(scale q_i k_j) ------------
# ---- rows of no sequence: o = 0, lse = -inf, no gradient --------------------------------------------
def _attn_inputs(c, seed):
    g = _generator(seed)
    n, h, kv, d = c["rows"] + c["pad"], c["heads"], c["kv_heads"], c["dim"]
    # scores of spread 2.5: a row looks mostly at a part of its keys
    qkv = torch.cat([_normal(g, (n, h * d), sigma=1.6), _normal(g, (n, kv * d), sigma=1.6), _normal(g, (n, kv * d))], 1)
    return {"qkv": qkv.to(torch.bfloat16), "starts": _ints(_starts(_lengths(c))), "g": g}


def _split(c, x):
    """q [n][kv_heads][group][dim], k and v [n][kv_heads][dim] of the rows of a projection."""
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    q, k, v = x.split([h * d, kv * d, kv * d], 1)
    return q.reshape(-1, kv, h // kv, d), k.reshape(-1, kv, d), v.reshape(-1, kv, d)


def _parts(c, lengths, queries=None):
    """(sequence, its rows, its kv heads a few at a time: as many as make scores of 1 GiB)."""
    at = _starts(queries or lengths)
    group = c["heads"] // c["kv_heads"]
    for s, n in enumerate(lengths):
        m = at[s + 1] - at[s]
        if m == 0:
            continue
        step = max(1, (1 << 28) // max(1, group * m * n))
        for k in range(0, c["kv_heads"], step):
            yield s, slice(at[s], at[s + 1]), slice(k, min(k + step, c["kv_heads"]))


def _softmax_parts(c, q, k, hidden):
    """Of q [m][kv][group][dim] and k [n][kv][dim] in 32 bits: q as [kv][group m][dim], exp(s - lse) [kv][group m][n] and
    lse [kv][group m]; hidden [m][n]: what is not seen."""
    m, kv, group, d = q.shape
    q = q.permute(1, 2, 0, 3).reshape(kv, group * m, d)
    s = torch.bmm(q, k.permute(1, 2, 0).contiguous()).mul_(_scale(c))
    if hidden is not None:
        s.view(kv, group, m, -1).masked_fill_(hidden, -math.inf)
    if s.shape[2] == 0:
        return q, s, torch.full(s.shape[:2], -math.inf, device="cuda")
    top = s.max(2, keepdim=True).values.clamp(min=-3e38)
    p = s.sub_(top).exp_()
    total = p.sum(2, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    return q, p, (top + torch.log(total))[:, :, 0]


def _hidden(c, m, n):
    """Of m rows at the end of n keys: whether key j lies behind row i."""
    if not c["causal"]:
        return None
    return torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]


def _attn_plain(c, s):
    q, k, v = _split(c, s["qkv"])
    n, kv, group, d = q.shape
    out = torch.zeros((n, kv, group, d), device="cuda")
    lse = torch.full((kv, group, n), -math.inf, device="cuda")
    for _, r, h in _parts(c, _lengths(c)):
        m = r.stop - r.start
        _, p, l = _softmax_parts(c, q[r, h].float(), k[r, h].float(), _hidden(c, m, m))
        o = torch.bmm(p, v[r, h].float().transpose(0, 1).contiguous())
        out[r, h] = o.view(-1, group, m, d).permute(2, 0, 1, 3)
        lse[h, :, r] = l.view(-1, group, m)
    return [out.reshape(n, -1).to(torch.bfloat16), lse.reshape(-1, n)]


def _heads_of(c, kernels, qkv):
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    return (kernels.Heads(qkv, h, d), kernels.Heads(qkv, kv, d, h * d), kernels.Heads(qkv, kv, d, (h + kv) * d))


def _attn_prepare(c, s):
    n = c["rows"] + c["pad"]
    out = [_empty((n, c["heads"] * c["dim"]), "bf16"), _empty((c["heads"], n), "f32")]
    return {"qkv": _put(s["qkv"]), "starts": _put(s["starts"]), "out": out, "result": [_torch(o) for o in out]}


def _attn_own(c, s, kernels, q):
    out, lse = s["out"]
    kernels.attention_fwd(q, *_heads_of(c, kernels, s["qkv"]), s["starts"], out, lse=lse, causal=c["causal"], scale=_scale(c))
    return s["result"]


def _pairs(c):
    return sum(n * (n + 1) // 2 if c["causal"] else n * n for n in _lengths(c))


def _attn_work(c):
    n, h, kv, d = c["rows"] + c["pad"], c["heads"], c["kv_heads"], c["dim"]
    return {"bytes": 2 * c["rows"] * (h + 2 * kv) * d + 2 * n * h * d + 4 * n * h, "flops": 4 * d * h * _pairs(c)}


def _attn_exact(c, seed):
    s = _attn_inputs(c, seed)
    n, h, kv, d = c["rows"] + c["pad"], c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().reshape(n, h + 2 * kv, d)
    out = torch.zeros((n, h, d), dtype=torch.float64, device="cuda")
    lse = torch.full((h, n), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for m in _lengths(c):
        r, at = slice(at, at + m), at + m
        seen = torch.ones((m, m), device="cuda").tril().bool() if c["causal"] else None
        for j in range(h if m else 0):
            z = x[r, j] @ x[r, h + j * kv // h].t() / math.sqrt(d)
            z = z if seen is None else z.masked_fill(~seen, -math.inf)
            lse[j, r] = torch.logsumexp(z, 1)
            out[r, j] = torch.softmax(z, 1) @ x[r, h + kv + j * kv // h]
    return [out.reshape(n, -1), lse]


# ---- its gradient: ds = p (do v - do o), dq = scale ds k, dk = scale ds^T q, dv = p^T do -------------
def _attn_grad_inputs(c, seed):
    s = _attn_inputs(c, seed)
    s["out"], s["lse"] = _attn_plain(c, s)  # as the forward pass left them
    s["dout"] = _normal(s["g"], tuple(s["out"].shape), "bf16")
    return s


def _attn_grad_plain(c, s):
    q, k, v = _split(c, s["qkv"])
    n, kv, group, d = q.shape
    do, o = (s[key].reshape(n, kv, group, d) for key in ("dout", "out"))
    grads = [torch.zeros(x.shape, device="cuda") for x in (q, k, v)]
    for _, r, h in _parts(c, _lengths(c)):
        m = r.stop - r.start
        rows, p, _ = _softmax_parts(c, q[r, h].float(), k[r, h].float(), _hidden(c, m, m))
        dr = do[r, h].float().permute(1, 2, 0, 3).reshape(-1, group * m, d)
        delta = (dr * o[r, h].float().permute(1, 2, 0, 3).reshape(-1, group * m, d)).sum(2, keepdim=True)
        grads[2][r, h] = torch.bmm(p.transpose(1, 2).contiguous(), dr).transpose(0, 1)
        ds = torch.bmm(dr, v[r, h].float().permute(1, 2, 0).contiguous()).sub_(delta).mul_(p).mul_(_scale(c))
        grads[0][r, h] = torch.bmm(ds, k[r, h].float().transpose(0, 1).contiguous()).view(-1, group, m, d).permute(2, 0, 1, 3)
        grads[1][r, h] = torch.bmm(ds.transpose(1, 2).contiguous(), rows).transpose(0, 1)
    return torch.cat([g.reshape(n, -1) for g in grads], 1).to(torch.bfloat16)


def _attn_grad_prepare(c, s):
    from vernondsl_amd import kernels
    t = {k: _put(s[k]) for k in ("qkv", "starts", "out", "lse", "dout")}
    grad = _empty(tuple(s["qkv"].shape), "bf16")
    need = kernels.attention_bwd_workspace_bytes(c["rows"] + c["pad"], c["seqs"], c["heads"], c["kv_heads"], c["dim"])
    return {**t, "grad": grad, "result": _torch(grad), "workspace": _workspace(need)}


def _attn_grad_own(c, s, kernels, q):
    kernels.attention_bwd(q, s["dout"], *_heads_of(c, kernels, s["qkv"]), s["starts"], s["out"], s["lse"],
                          *_heads_of(c, kernels, s["grad"]), causal=c["causal"], scale=_scale(c), workspace=s["workspace"])
    return s["result"]


def _attn_grad_work(c):
    n, h, kv, d = c["rows"] + c["pad"], c["heads"], c["kv_heads"], c["dim"]
    return {"bytes": 2 * c["rows"] * (3 * h + 2 * kv) * d + 4 * c["rows"] * h + 2 * n * (h + 2 * kv) * d, "flops": 10 * d * h * _pairs(c)}


def _attn_grad_exact(c, seed):
    s = _attn_grad_inputs(c, seed)
    n, h, kv, d = c["rows"] + c["pad"], c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().reshape(n, h + 2 * kv, d)
    do = s["dout"].double().reshape(n, h, d)
    grad = torch.zeros_like(x)
    at = 0
    for m in _lengths(c):
        r, at = slice(at, at + m), at + m
        seen = torch.ones((m, m), device="cuda").tril().bool() if c["causal"] else None
        for j in range(h if m else 0):
            of = (j, h + j * kv // h, h + kv + j * kv // h)
            a, b, v = (x[r, i].clone().requires_grad_(True) for i in of)
            z = a @ b.t() / math.sqrt(d)
            z = z if seen is None else z.masked_fill(~seen, -math.inf)
            for i, g in zip(of, torch.autograd.grad(torch.softmax(z, 1) @ v, (a, b, v), do[r, j])):
                grad[r, i] += g
    return grad.reshape(n, -1)


# ---- a paged cache: [pages][kv_heads][page][dim], k and v each; row i of a sequence's m new ones is ----
# ---- position p = length - m + i of it, in slot p % page of page table[sequence][p / page] -------------
def _cache_lengths(c):
    """(new rows, rows in the cache with the new ones) of each sequence: contexts of a quarter of "context" or more."""
    rng = random.Random(c["split"] + 1)
    new = _lengths(c)
    return new, [min(c["context"], m + int(c["context"] * rng.uniform(0.25, 1.0))) for m in new]


def _per_sequence(c):
    return -(-c["context"] // c["page"])


def _cache_inputs(c, seed):
    g = _generator(seed)
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    new, lengths = _cache_lengths(c)
    per = _per_sequence(c)
    pages = c["seqs"] * per
    # pages in the order in which a server that has run for a while hands them out: any
    table = torch.randperm(pages, generator=g, device="cuda").reshape(c["seqs"], per).to(torch.int32)
    used = -(-torch.tensor(lengths, device="cuda") // c["page"])
    table = torch.where(torch.arange(per, device="cuda")[None] < used[:, None], table, torch.full_like(table, -1))
    shape = (pages, kv, c["page"], d)
    n = c["rows"] + c["pad"]
    qkv = torch.cat([_normal(g, (n, h * d), "bf16", 1.6), _normal(g, (n, kv * d), "bf16", 1.6), _normal(g, (n, kv * d), "bf16")], 1)
    return {"qkv": qkv, "starts": _ints(_starts(new)), "lengths": _ints(lengths), "table": table.contiguous(),
            "k_cache": _normal(g, shape, "bf16", 1.6), "v_cache": _normal(g, shape, "bf16")}


def _append_plain(c, s):
    _, k, v = _split(c, s["qkv"])
    starts = s["starts"].long()
    row = torch.arange(c["rows"], device="cuda")
    of = torch.searchsorted(starts[1:], row, right=True)
    p = s["lengths"].long()[of] - (starts[of + 1] - row)
    page = s["table"].long()[of, p // c["page"]]
    s["k_cache"][page, :, p % c["page"]] = k[:c["rows"]]
    s["v_cache"][page, :, p % c["page"]] = v[:c["rows"]]
    return [s["k_cache"], s["v_cache"]]


def _cache_tensors(s):
    return {k: _put(s[k]) for k in ("qkv", "starts", "lengths", "table", "k_cache", "v_cache")}


def _append_prepare(c, s):
    t = _cache_tensors(s)
    return {**t, "result": [_torch(t["k_cache"]), _torch(t["v_cache"])]}


def _append_own(c, s, kernels, q):
    _, k, v = _heads_of(c, kernels, s["qkv"])
    kernels.cache_append(q, k, v, s["starts"], s["lengths"], s["table"], s["k_cache"], s["v_cache"])
    return s["result"]


def _append_work(c):
    return {"bytes": 8 * c["rows"] * c["kv_heads"] * c["dim"] + 4 * c["rows"], "flops": 0}


def _append_exact(c, seed):
    # row by row through the table; nothing is computed, so the values are the inputs'
    s = _cache_inputs(c, seed)
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].reshape(-1, h + 2 * kv, d)
    table, page = s["table"].tolist(), c["page"]
    at, to, slot = 0, [], []
    for q, (m, length) in enumerate(zip(*_cache_lengths(c))):
        for p in range(length - m, length):
            to.append(table[q][p // page])
            slot.append(p % page)
        at += m
    flat = (torch.tensor(to, device="cuda")[:, None] * kv + torch.arange(kv, device="cuda")) * page + torch.tensor(slot, device="cuda")[:, None]
    caches = []
    for name, first in (("k_cache", h), ("v_cache", h + kv)):
        new = s[name].reshape(-1, d).index_copy(0, flat.reshape(-1), x[:at, first:first + kv].reshape(-1, d))
        caches.append(new.reshape(s[name].shape).double())
    return caches


# ---- attention of the new rows over the cache, which holds them already: row i sees positions <= p -------
def _context_of(c, s, cache, q, length):
    pages = s["table"][q, :-(-length // c["page"])].long()
    return cache[pages].transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])[:length]


def _paged_plain(c, s):
    q, _, _ = _split(c, s["qkv"])
    n, kv, group, d = q.shape
    out = torch.zeros((n, kv, group, d), device="cuda")
    lse = torch.full((kv, group, n), -math.inf, device="cuda")
    new, lengths = _cache_lengths(c)
    last = None
    for i, r, h in _parts(c, lengths, new):
        if last != i:
            k, v = (_context_of(c, s, s[name], i, lengths[i]) for name in ("k_cache", "v_cache"))
            last = i
        m = r.stop - r.start
        _, p, l = _softmax_parts(c, q[r, h].float(), k[:, h].float(), _hidden(c, m, lengths[i]))
        o = torch.bmm(p, v[:, h].float().transpose(0, 1).contiguous())
        out[r, h] = o.view(-1, group, m, d).permute(2, 0, 1, 3)
        lse[h, :, r] = l.view(-1, group, m)
    return [out.reshape(n, -1).to(torch.bfloat16), lse.reshape(-1, n)]


def _paged_prepare(c, s):
    from vernondsl_amd import kernels
    n = c["rows"] + c["pad"]
    out = [_empty((n, c["heads"] * c["dim"]), "bf16"), _empty((c["heads"], n), "f32")]
    need = kernels.paged_attention_workspace_bytes(n, c["seqs"], c["heads"], c["kv_heads"], c["dim"], _per_sequence(c) * c["page"])
    return {**_cache_tensors(s), "out": out, "result": [_torch(o) for o in out], "workspace": _workspace(need)}


def _paged_own(c, s, kernels, q):
    out, lse = s["out"]
    kernels.paged_attention(q, _heads_of(c, kernels, s["qkv"])[0], s["k_cache"], s["v_cache"], s["starts"], s["lengths"], s["table"],
                            out, lse=lse, scale=_scale(c), workspace=s["workspace"])
    return s["result"]


def _paged_work(c):
    n, h, kv, d = c["rows"] + c["pad"], c["heads"], c["kv_heads"], c["dim"]
    new, lengths = _cache_lengths(c)
    pairs = sum(m * (length - m) + m * (m + 1) // 2 for m, length in zip(new, lengths))
    keys = sum(length for m, length in zip(new, lengths) if m)
    return {"bytes": 4 * keys * kv * d + 2 * (c["rows"] + n) * h * d + 4 * n * h, "flops": 4 * d * h * pairs}


def _paged_exact(c, seed):
    s = _cache_inputs(c, seed)
    n, h, kv, d = c["rows"] + c["pad"], c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().reshape(n, h + 2 * kv, d)
    out = torch.zeros((n, h, d), dtype=torch.float64, device="cuda")
    lse = torch.full((h, n), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for i, (m, length) in enumerate(zip(*_cache_lengths(c))):
        r, at = slice(at, at + m), at + m
        if m == 0:
            continue
        where = [s["table"][i, p].item() for p in range(-(-length // c["page"]))]
        keys, values = (torch.cat([cache[p] for p in where], 1)[:, :length].double() for cache in (s["k_cache"], s["v_cache"]))
        seen = torch.ones((m, length), device="cuda").tril(length - m).bool()
        for j in range(h):
            z = (x[r, j] @ keys[j * kv // h].t() / math.sqrt(d)).masked_fill(~seen, -math.inf)
            lse[j, r] = torch.logsumexp(z, 1)
            out[r, j] = torch.softmax(z, 1) @ values[j * kv // h]
    return [out.reshape(n, -1), lse]


# ---- the kinds: inputs, plain form, buffers, the framework's call, work, 64 bits -------------------
_KINDS = {
    "rope": (_rope_inputs, _rope_plain, _rope_prepare, _rope_own, _rope_work, _rope_exact),
    "attn": (_attn_inputs, _attn_plain, _attn_prepare, _attn_own, _attn_work, _attn_exact),
    "attn_grad": (_attn_grad_inputs, _attn_grad_plain, _attn_grad_prepare, _attn_grad_own, _attn_grad_work, _attn_grad_exact),
    "append": (_cache_inputs, _append_plain, _append_prepare, _append_own, _append_work, _append_exact),
    "paged": (_cache_inputs, _paged_plain, _paged_prepare, _paged_own, _paged_work, _paged_exact),
}


def listed():
    return [
        # one token of each of a few requests, far into a stretched context; q and k turn, v is handed on
        {"name": "rope_8x40x128", "kind": "rope", "rows": 8, "seqs": 8, "split": 1, "heads": 40, "rest": 8, "dim": 128, "rot": 128,
         "interleaved": False, "inverse": False, "factor": 8.0, "reach": 32768, "x": "bf16", "y": "bf16"},
        # a training batch's gradient of a projection, back through the positions of half of each head
        {"name": "rope_grad_16384x40x128", "kind": "rope", "rows": 16384, "seqs": 8, "split": 2, "heads": 40, "rest": 8, "dim": 128,
         "rot": 64, "interleaved": True, "inverse": True, "factor": 1.0, "reach": 1, "x": "f32", "y": "bf16"},
        # a few short texts in a padded batch, heads of an odd size
        {"name": "attn_300x6x80", "kind": "attn", "rows": 293, "pad": 7, "seqs": 5, "split": 3, "heads": 6, "kv_heads": 2, "dim": 80,
         "causal": True},
        # a training batch: texts of different lengths packed into one row of 8192
        {"name": "attn_8192x32x128", "kind": "attn", "rows": 8192, "pad": 0, "seqs": 6, "split": 4, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True},
        # one long prompt
        {"name": "attn_16384x32x128", "kind": "attn", "rows": 16384, "pad": 0, "seqs": 1, "split": 5, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True},
        # the backward pass of the padded batch
        {"name": "attn_grad_300x6x80", "kind": "attn_grad", "rows": 293, "pad": 7, "seqs": 5, "split": 3, "heads": 6, "kv_heads": 2,
         "dim": 80, "causal": True},
        # the backward pass of a training batch
        {"name": "attn_grad_8192x32x128", "kind": "attn_grad", "rows": 8192, "pad": 0, "seqs": 2, "split": 6, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True},
        # one new token of each request of a running server
        {"name": "append_64x8x128", "kind": "append", "rows": 64, "pad": 0, "seqs": 64, "split": 7, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "context": 1000},
        # the prompts of a few requests
        {"name": "append_16384x8x128", "kind": "append", "rows": 16384, "pad": 0, "seqs": 6, "split": 8, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "context": 16384},
        # a few requests' next tokens over short contexts: all latency
        {"name": "paged_8x32x128", "kind": "paged", "rows": 8, "pad": 0, "seqs": 8, "split": 9, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "context": 1000, "causal": True},
        # a full server's next tokens over long contexts: the cache is read once
        {"name": "paged_64x32x128", "kind": "paged", "rows": 64, "pad": 0, "seqs": 64, "split": 10, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "context": 16384, "causal": True},
        # a long prompt taken in chunks beside other requests: its next rows over what is cached
        {"name": "paged_1024x32x128", "kind": "paged", "rows": 1024, "pad": 0, "seqs": 4, "split": 11, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "context": 16384, "causal": True},
    ]


def _spread(rng, lo, hi):
    """An integer in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(sorted(_KINDS))
    split = rng.randrange(1 << 16)
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 5, 8])
    dim = rng.choice([64, 128, 128, 8 * rng.randrange(4, 17)])
    case = {"kind": kind, "split": split, "dim": dim}
    if kind == "rope":
        rows = _spread(rng, 1, 16384)
        rot = rng.choice([dim, dim, 2 * rng.randrange(4, dim // 2 + 1)])
        return {**case, "rows": rows, "seqs": rng.randint(1, 8), "heads": heads, "rest": rng.choice([0, kv_heads]), "rot": rot,
                "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.5, "factor": rng.choice([1.0, 4.0, 32.0]),
                "reach": rng.choice([1, 4096, 1 << 17, 1 << 20]), "x": rng.choice(["f32", "bf16"]), "y": rng.choice(["f32", "bf16"])}
    case = {**case, "heads": heads, "kv_heads": kv_heads, "pad": rng.choice([0, 0, rng.randint(1, 40)])}
    if kind in ("attn", "attn_grad"):
        return {**case, "rows": _spread(rng, 1, 8192), "seqs": rng.choice([1, rng.randint(2, 8), rng.randint(9, 64)]),
                "causal": rng.random() < 0.75}
    page = rng.choice([16, 16, 32, 64, 256])
    if kind == "append":
        rows = _spread(rng, 1, 8192)
        return {**case, "rows": rows, "seqs": rng.randint(1, 8), "page": page, "context": rows + _spread(rng, 1, 4096)}
    # one new row of each sequence or so, or chunks of them
    seqs = _spread(rng, 1, 64)
    rows = rng.choice([seqs, seqs, seqs + rng.randint(0, seqs), _spread(rng, 1, 1024)])
    return {**case, "rows": rows, "seqs": seqs, "page": page, "context": rows + _spread(rng, 1, (1 << 18) // seqs), "causal": True}


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
