"""Op-class calls on the HIP device, one function per `vdsl_op_*` entry point of include/vdsl.h.

Each function checks operand shapes and dtypes on the host before anything is enqueued (the C
ABI checks buffer sizes again), then enqueues the op on `q` and returns without waiting.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import numpy as np

from . import _lib
from ._lib import call
from .mapchain import Program
from .rhi import Queue, Tensor, dtype_code


def _h(t):
    return None if t is None else t.handle


def _expect(t: Tensor, shape, dtype, name):
    if t is None:
        return
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {t.shape}, expected {tuple(shape)}")
    if t.dtype != dtype_code(dtype):
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")


# ---- op class 1: escape-time iterative map (fractal.py:16-25) -------------------------------
def escape_time_params(**kw) -> _lib.EscapeTimeParams:
    p = _lib.EscapeTimeParams()
    defaults = dict(family=_lib.ESC_MANDELBROT, escape_test=_lib.ESC_MAG2_GT, rounding=_lib.ESC_ROUND_FMA,
                    out_kind=_lib.ESC_OUT_I32_COUNT, max_iter=256, bound=4.0,
                    re_den=1.0, re_off=0.0, re_scale=1.0, re_post=0.0,
                    im_den=1.0, im_off=0.0, im_scale=1.0, im_post=0.0,
                    c_re=0.0, c_im=0.0, out_base=0.0, out_scale=1.0)
    defaults.update(kw)
    for k, v in defaults.items():
        setattr(p, k, v)
    return p


def escape_time(q: Queue, p: _lib.EscapeTimeParams, out: Tensor):
    dt = "i32" if p.out_kind == _lib.ESC_OUT_I32_COUNT else "f32"
    _expect(out, (p.ni, p.nj), dt, "out")
    call("vdsl_op_escape_time", q.handle, C.byref(p), out.handle)


# ---- op class 2: fused map chain --------------------------------------------------------------
def map_chain(q: Queue, prog: Program, inputs, out: Tensor):
    """inputs[k] is the Tensor for Input(k); its broadcast comes from the program."""
    rows, cols = out.shape
    if len(inputs) != prog.n_inputs:
        raise ValueError(f"program reads {prog.n_inputs} inputs, {len(inputs)} given")
    arr = (_lib.MapInput * max(1, len(inputs)))()
    for k, t in enumerate(inputs):
        bc = prog.bcast[k]
        want = {_lib.BCAST_FULL: (rows, cols), _lib.BCAST_ROW: (cols,), _lib.BCAST_COL: (rows,), _lib.BCAST_SCALAR: (1,)}[bc]
        _expect(t, want, "f32", f"input{k}")
        arr[k].buf, arr[k].bcast, arr[k].dtype = t.handle.value, bc, _lib.F32
    _expect(out, (rows, cols), "f32", "out")
    code = prog.instr_array()
    call("vdsl_op_map_chain", q.handle, rows, cols, code, len(prog.code), arr, len(inputs), prog.out_reg, out.handle)


def map_chain_v(q: Queue, prog: Program, inputs, out: Tensor):
    """A chain over vector operands (vdsl_op_map_chain_v).  inputs[k] is the Tensor of input k:
    [rows][cols][w] for a full input of width w > 1 ([rows][cols] when w = 1), [cols][w] / [rows][w]
    / [w] when broadcast.  out: [rows][cols][len(prog.out_regs)] ([rows][cols] for one component)."""
    rows, cols = out.shape[:2]
    ow = len(prog.out_regs)
    _expect(out, (rows, cols, ow) if ow > 1 else (rows, cols), "f32", "out")
    if len(inputs) != prog.n_inputs:
        raise ValueError(f"program reads {prog.n_inputs} inputs, {len(inputs)} given")
    arr = (_lib.MapVInput * max(1, len(inputs)))()
    for k, t in enumerate(inputs):
        bc, w, d = prog.bcast[k], prog.widths[k], prog.dims.get(k, 0)
        want = {_lib.BCAST_FULL: (rows, cols), _lib.BCAST_ROW: (cols,), _lib.BCAST_COL: (rows,), _lib.BCAST_SCALAR: ()}[bc]
        if d:
            want = want + (d, d)
        elif w > 1 or bc == _lib.BCAST_SCALAR:
            want = want + (w,)
        _expect(t, want, "f32", f"input{k}")
        arr[k].buf, arr[k].bcast, arr[k].dtype, arr[k].width, arr[k].mat_dim = t.handle.value, bc, _lib.F32, w, d
    regs = (C.c_int32 * 4)(*(prog.out_regs + [0] * (4 - ow)))
    call("vdsl_op_map_chain_v", q.handle, rows, cols, prog.instr_array(), len(prog.code), arr, len(inputs), regs, ow,
         out.handle)


# ---- vertex transform (color.mlir:10-39) ----------------------------------------------------------
def vec_transform(q: Queue, pos: Tensor, mats: Tensor, out: Tensor, varying: Tensor | None = None):
    """out [n][4] = M_k ... M_1 vec4(pos, 1) for pos [n][3] (or M... pos for [n][4]); mats [k][4][4]
    row-major (model, view, proj order), k = 1..3; varying (optional) [n][3|4] = pos."""
    n, w = pos.shape
    nm = mats.shape[0]
    _expect(pos, (n, w), "f32", "pos")
    _expect(mats, (nm, 4, 4), "f32", "mats")
    _expect(out, (n, 4), "f32", "out")
    _expect(varying, (n, w), "f32", "varying")
    call("vdsl_op_vec_transform", q.handle, n, w, pos.handle, nm, mats.handle, out.handle, _h(varying))


def mat_transform(q: Queue, pos: Tensor, mats: Tensor, out: Tensor, varying: Tensor | None = None):
    """out [n][d] = M_k ... M_1 vec(pos, 1) for pos [n][d-1] (or M... pos for [n][d]); mats [k][d][d]
    row-major, d = 2, 3 or 4, k = 1..3; varying (optional) [n][d-1|d] = pos."""
    n, w = pos.shape
    nm, d = mats.shape[0], mats.shape[1]
    _expect(pos, (n, w), "f32", "pos")
    _expect(mats, (nm, d, d), "f32", "mats")
    _expect(out, (n, d), "f32", "out")
    _expect(varying, (n, w), "f32", "varying")
    call("vdsl_op_mat_transform", q.handle, n, d, w, pos.handle, nm, mats.handle, out.handle, _h(varying))


# ---- op class 3: row reductions + softmax ------------------------------------------------------
def row_reduce_softmax(q: Queue, x: Tensor, row_sum=None, row_max=None, softmax=None):
    rows, cols = x.shape
    _expect(row_sum, (rows,), "f32", "row_sum")
    _expect(row_max, (rows,), "f32", "row_max")
    _expect(softmax, (rows, cols), x.dtype, "softmax")
    call("vdsl_op_row_reduce_softmax", q.handle, rows, cols, x.dtype, x.handle, _h(row_sum), _h(row_max), _h(softmax))


def col_reduce(q: Queue, x: Tensor, col_sum=None, col_max=None):
    rows, cols = x.shape
    _expect(col_sum, (cols,), "f32", "col_sum")
    _expect(col_max, (cols,), "f32", "col_max")
    call("vdsl_op_col_reduce", q.handle, rows, cols, x.dtype, x.handle, _h(col_sum), _h(col_max))


# ---- op class 4: bf16 GEMM + layout + autodiff blocks ------------------------------------------
def gemm_bf16_workspace_bytes(trans_a, trans_b, M, N, K) -> int:
    n = C.c_size_t()
    call("vdsl_gemm_bf16_workspace_bytes", int(trans_a), int(trans_b), M, N, K, C.byref(n))
    return n.value


def gemm_bf16(q: Queue, A: Tensor, B: Tensor, Cout: Tensor, trans_a=False, trans_b=False,
              epilogue=_lib.EPI_NONE, pre_act=None, workspace=None):
    if trans_a:
        K, M = A.shape
    else:
        M, K = A.shape
    if trans_b:
        N, K2 = B.shape
    else:
        K2, N = B.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    _expect(A, A.shape, "bf16", "A")
    _expect(B, B.shape, "bf16", "B")
    if Cout.shape != (M, N):
        raise ValueError(f"C: shape {Cout.shape}, expected {(M, N)}")
    _expect(pre_act, (M, N), "f32", "pre_act")
    call("vdsl_op_gemm_bf16", q.handle, int(trans_a), int(trans_b), M, N, K, A.handle, B.handle, Cout.handle,
         Cout.dtype, int(epilogue), _h(pre_act), _h(workspace))


def gemm_bf16_mse_packed(q: Queue, A: Tensor, Bp: Tensor, T: Tensor, Y, loss: Tensor, dy: Tensor, dy_t=None,
                         partials: Tensor = None):
    """Y = A Bp^T fused with loss = mean((Y - T)^2), dy = bf16(2 (Y - T) / n), dy_t = dy^T
    (vdsl_op_gemm_bf16_mse_packed); Y (f32) and dy_t may be None.  Bp: packed [N][K] weights."""
    M, K = A.shape
    N = Bp.shape[0]
    _expect(A, (M, K), "bf16", "A")
    _expect(Bp, (N, K), "bf16", "Bp")
    _expect(T, (M, N), "f32", "T")
    _expect(Y, (M, N), "f32", "Y")
    _expect(loss, (1,), "f32", "loss")
    _expect(dy, (M, N), "bf16", "dy")
    _expect(dy_t, (N, M), "bf16", "dy_t")
    call("vdsl_op_gemm_bf16_mse_packed", q.handle, M, N, K, A.handle, Bp.handle, T.handle, _h(Y), loss.handle, dy.handle,
         _h(dy_t), partials.handle)


def pack_bf16_weights(q: Queue, w: Tensor, wp: Tensor):
    """Writes w (bf16 [N][K]) into wp in the MFMA fragment order gemm_bf16_packed reads."""
    N, K = w.shape
    _expect(w, (N, K), "bf16", "w")
    _expect(wp, (N, K), "bf16", "wp")
    call("vdsl_op_pack_bf16_weights", q.handle, N, K, w.handle, wp.handle)


def gemm_bf16_packed(q: Queue, A: Tensor, Bp: Tensor, Cout: Tensor, epilogue=_lib.EPI_NONE, pre_act=None):
    """gemm_bf16(A, B, trans_b=True) with B packed by pack_bf16_weights (Bp keeps the logical
    shape [N][K]); bit-identical results."""
    M, K = A.shape
    N, K2 = Bp.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    _expect(A, (M, K), "bf16", "A")
    _expect(Bp, (N, K), "bf16", "Bp")
    if Cout.shape != (M, N):
        raise ValueError(f"C: shape {Cout.shape}, expected {(M, N)}")
    _expect(pre_act, (M, N), "f32", "pre_act")
    call("vdsl_op_gemm_bf16_packed", q.handle, M, N, K, A.handle, Bp.handle, Cout.handle, Cout.dtype, int(epilogue),
         _h(pre_act))


def transpose(q: Queue, src: Tensor, dst: Tensor):
    rows, cols = src.shape
    _expect(dst, (cols, rows), src.dtype, "dst")
    call("vdsl_op_transpose", q.handle, rows, cols, src.dtype, src.handle, dst.handle)


def cast(q: Queue, src: Tensor, dst: Tensor):
    if src.numel != dst.numel:
        raise ValueError("cast: element counts differ")
    call("vdsl_op_cast", q.handle, src.numel, src.dtype, src.handle, dst.dtype, dst.handle)


def gelu_fwd(q: Queue, x: Tensor, y: Tensor):
    """y = GELU(x) elementwise (exact-erf form); x, y f32 or bf16 of one element count."""
    if x.numel != y.numel:
        raise ValueError(f"gelu_fwd: x has {x.numel} elements, y {y.numel}")
    call("vdsl_op_gelu_fwd", q.handle, x.numel, x.dtype, x.handle, y.dtype, y.handle)


def gelu_bwd(q: Queue, dh: Tensor, pre: Tensor, da: Tensor, da_t=None, act: str = "gelu"):
    """da = bf16(dh * act'(pre)) (+ its transpose da_t); act "gelu" or "relu"."""
    rows, cols = dh.shape
    _expect(dh, (rows, cols), "f32", "dh")
    _expect(pre, (rows, cols), "f32", "pre")
    _expect(da, (rows, cols), "bf16", "da")
    _expect(da_t, (cols, rows), "bf16", "da_t")
    fn = {"gelu": "vdsl_op_gelu_bwd", "relu": "vdsl_op_relu_bwd"}[act]
    call(fn, q.handle, rows, cols, dh.handle, pre.handle, da.handle, _h(da_t))


def add(q: Queue, a: Tensor, b: Tensor, out: Tensor):
    """out = a + b elementwise (f32 or bf16 each; one f32 addition rounded to out's dtype)."""
    if not (a.numel == b.numel == out.numel):
        raise ValueError(f"add: {a.numel}, {b.numel} and {out.numel} elements")
    call("vdsl_op_add", q.handle, out.numel, a.dtype, a.handle, b.dtype, b.handle, out.dtype, out.handle)


def gemm_bf16_gelu_bwd(q: Queue, A: Tensor, B: Tensor, pre: Tensor, da: Tensor, da_t=None, packed=False):
    """da = (A B^T) * GELU'(pre) as bf16 (and da_t = da^T): the GEMM forming dL/dy fused with the
    GELU backward (A bf16 [M][K], B bf16 [N][K] - packed by pack_bf16_weights if `packed` -, pre
    f32 [M][N])."""
    M, K = A.shape
    N, K2 = B.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    _expect(A, (M, K), "bf16", "A")
    _expect(B, (N, K), "bf16", "B")
    _expect(pre, (M, N), "f32", "pre")
    _expect(da, (M, N), "bf16", "da")
    _expect(da_t, (N, M), "bf16", "da_t")
    call("vdsl_op_gemm_bf16_gelu_bwd_packed" if packed else "vdsl_op_gemm_bf16_gelu_bwd", q.handle, M, N, K, A.handle,
         B.handle, pre.handle, da.handle, _h(da_t))


def gemm_bf16_mul_packed(q: Queue, A: Tensor, Bp: Tensor, g: Tensor, c: Tensor, c_t=None):
    """c = bf16((A Bp^T) * g) (and c_t = c^T): the GEMM forming dL/dh fused with the multiply by a
    stored local derivative g (f32 [M][N], e.g. GELU'(pre) from a forward GEMM with the
    EPI_GELU_DERIV epilogue).  Bp: packed [N][K] weights."""
    M, K = A.shape
    N, K2 = Bp.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    _expect(A, (M, K), "bf16", "A")
    _expect(Bp, (N, K), "bf16", "Bp")
    _expect(g, (M, N), "f32", "g")
    _expect(c, (M, N), "bf16", "c")
    _expect(c_t, (N, M), "bf16", "c_t")
    call("vdsl_op_gemm_bf16_mul_packed", q.handle, M, N, K, A.handle, Bp.handle, g.handle, c.handle, _h(c_t))


def pixel_program(q: Queue, prog, inputs, out: Tensor | None, grid=None):
    """Runs a compiled per-pixel program (vernondsl_amd.pixprog.PixelProgram) over out's [ni][nj]
    grid: out f32 [ni][nj] or [ni][nj][out_width] (the program stores registers) or i32 [ni][nj]
    (it stores its loop count); inputs: f32 fields [ni][nj] or [ni][nj][in_widths[k]], read at
    each pixel, or of their own extents [in_rows[k]][in_cols[k]] (gathered, or scatter-added
    into).  A program that stores nothing (pixprog.OUT_NONE) takes out None and grid (ni, nj)."""
    if prog.out_kind == 3:
        if out is not None or grid is None or len(grid) != 2:
            raise ValueError("a program that stores nothing takes out=None and grid=(ni, nj)")
        ni, nj = (int(v) for v in grid)
    else:
        if out is None or len(out.shape) not in (2, 3):
            raise ValueError("out must be a 2-D field of scalars or vectors")
        ni, nj = out.shape[:2]
        if grid is not None and tuple(grid) != (ni, nj):
            raise ValueError(f"grid {tuple(grid)} is not out's [{ni}][{nj}]")

    def field_shape(w, r=ni, c=nj):
        return (r, c) if w == 1 else (r, c, w)

    if prog.out_kind in (1, 2):  # the loop count, or an int32 field
        _expect(out, (ni, nj), "i32", "out")
    elif prog.out_kind != 3:
        _expect(out, field_shape(prog.out_width), "f32", "out")
    for k, t in enumerate(inputs):
        r, c = (prog.in_rows[k], prog.in_cols[k]) if prog.in_rows[k] else (ni, nj)  # an input of its own extents
        _expect(t, field_shape(prog.in_widths[k], r, c), "i32" if prog.in_dtypes[k] == _lib.I32 else "f32", f"input{k}")
    hs = (C.c_void_p * max(1, len(inputs)))(*[t.handle for t in inputs])
    call("vdsl_op_pixel_program", q.handle, ni, nj, C.byref(prog), hs, len(inputs), _h(out))


def mse_partials_count(rows, cols) -> int:
    return int(_lib.lib.vdsl_mse_partials_count(rows, cols))


def mse_fwd_bwd(q: Queue, y: Tensor, t: Tensor, loss: Tensor, dy: Tensor, dy_t, partials: Tensor):
    rows, cols = y.shape
    _expect(t, (rows, cols), "f32", "t")
    _expect(loss, (1,), "f32", "loss")
    _expect(dy, (rows, cols), "bf16", "dy")
    _expect(dy_t, (cols, rows), "bf16", "dy_t")
    call("vdsl_op_mse_fwd_bwd", q.handle, rows, cols, y.handle, t.handle, loss.handle, dy.handle, _h(dy_t),
         partials.handle)


# ---- op class 5: int8 W8A8 -----------------------------------------------------------------------
def quantize_rows_i8(q: Queue, x: Tensor, qx: Tensor, scale: Tensor):
    rows, cols = x.shape
    _expect(qx, (rows, cols), "i8", "qx")
    _expect(scale, (rows,), "f32", "scale")
    call("vdsl_op_quantize_rows_i8", q.handle, rows, cols, x.dtype, x.handle, qx.handle, scale.handle)


def gemm_w8a8_workspace_bytes(M, N, K) -> int:
    n = C.c_size_t()
    call("vdsl_gemm_w8a8_workspace_bytes", M, N, K, C.byref(n))
    return n.value


def gemm_w8a8(q: Queue, xq: Tensor, x_scale: Tensor, w: Tensor, w_scale: Tensor, y: Tensor, relu=False,
              acc_out=None, workspace=None):
    M, K = xq.shape
    N, K2 = w.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    _expect(xq, (M, K), "i8", "xq")
    _expect(w, (N, K), "i8", "w")
    _expect(x_scale, (M,), "f32", "x_scale")
    _expect(w_scale, (N,), "f32", "w_scale")
    if y.shape != (M, N):
        raise ValueError(f"y: shape {y.shape}, expected {(M, N)}")
    _expect(acc_out, (M, N), "i32", "acc_out")
    call("vdsl_op_gemm_w8a8", q.handle, M, N, K, xq.handle, x_scale.handle, w.handle, w_scale.handle, y.handle,
         y.dtype, int(bool(relu)), _h(acc_out), _h(workspace))


def pack_w8a8_weights(q: Queue, w: Tensor, wp: Tensor):
    """Writes w (int8 [N][K]) into wp in the MFMA fragment order gemm_w8a8_packed reads."""
    N, K = w.shape
    _expect(w, (N, K), "i8", "w")
    _expect(wp, (N, K), "i8", "wp")
    call("vdsl_op_pack_w8a8_weights", q.handle, N, K, w.handle, wp.handle)


def gemm_w8a8_packed_workspace_bytes(M, N, K) -> int:
    n = C.c_size_t()
    call("vdsl_gemm_w8a8_packed_workspace_bytes", M, N, K, C.byref(n))
    return n.value


def gemm_w8a8_packed(q: Queue, xq: Tensor, x_scale: Tensor, wp: Tensor, w_scale: Tensor, y: Tensor, relu=False,
                     acc_out=None, workspace=None):
    """gemm_w8a8 with weights packed by pack_w8a8_weights (wp keeps the logical shape [N][K]).
    workspace: gemm_w8a8_packed_workspace_bytes(M, N, K) bytes (split-K partials)."""
    M, K = xq.shape
    N, K2 = wp.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    _expect(xq, (M, K), "i8", "xq")
    _expect(wp, (N, K), "i8", "wp")
    _expect(x_scale, (M,), "f32", "x_scale")
    _expect(w_scale, (N,), "f32", "w_scale")
    if y.shape != (M, N):
        raise ValueError(f"y: shape {y.shape}, expected {(M, N)}")
    _expect(acc_out, (M, N), "i32", "acc_out")
    call("vdsl_op_gemm_w8a8_packed", q.handle, M, N, K, xq.handle, x_scale.handle, wp.handle, w_scale.handle,
         y.handle, y.dtype, int(bool(relu)), _h(acc_out), _h(workspace))


def gemm_w8a8_packed_noalloc(q: Queue, xq: Tensor, x_scale: Tensor, wp: Tensor, w_scale: Tensor, y: Tensor,
                             relu=False, acc_out=None):
    """gemm_w8a8_packed without a workspace (vdsl_op_gemm_w8a8_packed_noalloc): the split-K
    partials live in the library's own per-GPU array, so the call allocates nothing.  Calls that
    overlap in time on one GPU share that array and race."""
    M, K = xq.shape
    N, K2 = wp.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    _expect(xq, (M, K), "i8", "xq")
    _expect(wp, (N, K), "i8", "wp")
    _expect(x_scale, (M,), "f32", "x_scale")
    _expect(w_scale, (N,), "f32", "w_scale")
    if y.shape != (M, N):
        raise ValueError(f"y: shape {y.shape}, expected {(M, N)}")
    _expect(acc_out, (M, N), "i32", "acc_out")
    call("vdsl_op_gemm_w8a8_packed_noalloc", q.handle, M, N, K, xq.handle, x_scale.handle, wp.handle,
         w_scale.handle, y.handle, y.dtype, int(bool(relu)), _h(acc_out))


# ---- op class 6: what makes an MLP a model of tokens -------------------------------------------------
def embedding_fwd(q: Queue, table: Tensor, ids: Tensor, out: Tensor, scale: float = 1.0):
    """out [n][dim] = scale * table [vocab][dim][ids[i]] (f32 or bf16 each; ids i32 [n]); zeros where an
    id is outside the table."""
    vocab, dim = table.shape
    (n,) = ids.shape
    _expect(ids, (n,), "i32", "ids")
    if out.shape != (n, dim):
        raise ValueError(f"out: shape {out.shape}, expected {(n, dim)}")
    call("vdsl_op_embedding_fwd", q.handle, n, dim, vocab, table.dtype, table.handle, ids.handle, scale, out.dtype, out.handle)


def embedding_bwd_workspace_bytes(n, vocab, dim) -> int:
    b = C.c_size_t()
    call("vdsl_embedding_bwd_workspace_bytes", n, vocab, dim, C.byref(b))
    return b.value


def embedding_bwd(q: Queue, ids: Tensor, dy: Tensor, dtable: Tensor, scale: float = 1.0, workspace=None):
    """dtable (f32 [vocab][dim], every row written) = scale * the sum of dy [n][dim] over each row's tokens.
    workspace: embedding_bwd_workspace_bytes(n, vocab, dim) bytes."""
    vocab, dim = dtable.shape
    (n,) = ids.shape
    _expect(ids, (n,), "i32", "ids")
    if dy.shape != (n, dim):
        raise ValueError(f"dy: shape {dy.shape}, expected {(n, dim)}")
    _expect(dtable, (vocab, dim), "f32", "dtable")
    call("vdsl_op_embedding_bwd", q.handle, n, dim, vocab, ids.handle, dy.dtype, dy.handle, scale, dtable.handle, _h(workspace))


def _norm_params(cols, *params) -> int:
    """The one dtype of gamma and beta, each [cols] or None."""
    dt = _lib.F32
    given = [p for p in params if p is not None]
    for p in given:
        dt = given[0].dtype
        _expect(p, (cols,), dt, "gamma / beta")
    return dt


def layer_norm_fwd(q: Queue, x: Tensor, gamma, beta, y: Tensor, mean=None, rstd=None, eps: float = 1e-5):
    """y = (x - mean) * rstd * gamma + beta over the rows of x [rows][cols]; gamma, beta [cols] or None
    (1 and 0); mean and rstd (f32 [rows], optional) are kept for layer_norm_bwd."""
    rows, cols = x.shape
    if y.shape != (rows, cols):
        raise ValueError(f"y: shape {y.shape}, expected {(rows, cols)}")
    _expect(mean, (rows,), "f32", "mean")
    _expect(rstd, (rows,), "f32", "rstd")
    pdt = _norm_params(cols, gamma, beta)
    call("vdsl_op_layer_norm_fwd", q.handle, rows, cols, x.dtype, x.handle, pdt, _h(gamma), _h(beta), eps, y.dtype, y.handle,
         _h(mean), _h(rstd))


def layer_norm_bwd_workspace_bytes(rows, cols) -> int:
    b = C.c_size_t()
    call("vdsl_layer_norm_bwd_workspace_bytes", rows, cols, C.byref(b))
    return b.value


def layer_norm_bwd(q: Queue, dy: Tensor, x: Tensor, gamma, mean: Tensor, rstd: Tensor, dx: Tensor, dgamma=None, dbeta=None,
                   workspace=None):
    """dx [rows][cols], dgamma and dbeta (f32 [cols], optional) from dy, x and the forward pass's mean and
    rstd.  workspace: layer_norm_bwd_workspace_bytes(rows, cols) bytes, where dgamma or dbeta is wanted."""
    rows, cols = x.shape
    if dy.shape != (rows, cols):
        raise ValueError(f"dy: shape {dy.shape}, expected {(rows, cols)}")
    if dx.shape != (rows, cols):
        raise ValueError(f"dx: shape {dx.shape}, expected {(rows, cols)}")
    _expect(mean, (rows,), "f32", "mean")
    _expect(rstd, (rows,), "f32", "rstd")
    _expect(dgamma, (cols,), "f32", "dgamma")
    _expect(dbeta, (cols,), "f32", "dbeta")
    pdt = _norm_params(cols, gamma)
    call("vdsl_op_layer_norm_bwd", q.handle, rows, cols, dy.dtype, dy.handle, x.dtype, x.handle, pdt, _h(gamma), mean.handle,
         rstd.handle, dx.dtype, dx.handle, _h(dgamma), _h(dbeta), _h(workspace))


def linear_xent_workspace_bytes(n, vocab, dim, piece=0, backward=True) -> int:
    b = C.c_size_t()
    call("vdsl_linear_xent_workspace_bytes", n, vocab, dim, piece, int(bool(backward)), C.byref(b))
    return b.value


def _xent_operands(x, w, labels, loss, row_loss, lse):
    n, dim = x.shape
    vocab = w.shape[0]
    _expect(x, (n, dim), "bf16", "x")
    _expect(w, (vocab, dim), "bf16", "w")
    _expect(labels, (n,), "i32", "labels")
    _expect(loss, (1,), "f32", "loss")
    _expect(row_loss, (n,), "f32", "row_loss")
    _expect(lse, (n,), "f32", "lse")
    return n, dim, vocab


def linear_xent_fwd(q: Queue, x: Tensor, w: Tensor, labels: Tensor, loss: Tensor, row_loss=None, lse=None, workspace=None):
    """loss = the mean over the rows of x (bf16 [n][dim]) that count of logsumexp(x w^T) - (x w^T)[label], w
    bf16 [vocab][dim]; a row whose label (i32 [n]) is outside [0, vocab) does not count.  row_loss and lse
    (f32 [n], optional): the rows' losses and log sums.  workspace:
    linear_xent_workspace_bytes(n, vocab, dim, backward=False) bytes."""
    n, dim, vocab = _xent_operands(x, w, labels, loss, row_loss, lse)
    call("vdsl_op_linear_xent_fwd", q.handle, n, dim, vocab, x.handle, w.handle, labels.handle, loss.handle, _h(row_loss), _h(lse),
         _h(workspace))


def linear_xent_fwd_bwd(q: Queue, x: Tensor, w: Tensor, labels: Tensor, loss: Tensor, dx: Tensor, dw: Tensor, row_loss=None,
                        lse=None, piece: int = 0, grad_scale: float = 1.0, workspace=None):
    """linear_xent_fwd with the gradients of grad_scale * loss: dx [n][dim] and dw [vocab][dim], f32 or bf16
    each.  piece: columns of the vocabulary worked on at a time (0: the library's choice); workspace:
    linear_xent_workspace_bytes(n, vocab, dim, piece) bytes."""
    n, dim, vocab = _xent_operands(x, w, labels, loss, row_loss, lse)
    if dx.shape != (n, dim):
        raise ValueError(f"dx: shape {dx.shape}, expected {(n, dim)}")
    if dw.shape != (vocab, dim):
        raise ValueError(f"dw: shape {dw.shape}, expected {(vocab, dim)}")
    call("vdsl_op_linear_xent_fwd_bwd", q.handle, n, dim, vocab, x.handle, w.handle, labels.handle, piece, grad_scale, loss.handle,
         _h(row_loss), _h(lse), dx.dtype, dx.handle, dw.dtype, dw.handle, _h(workspace))


# ---- op class 7: what lets the rows of a sequence see each other ---------------------------------------
class Heads(NamedTuple):
    """Heads in the columns of a tensor [rows][width]: head h is columns [first + h * dim, first + (h + 1) * dim).  A tensor
    [rows][heads][dim] stands for all of its columns wherever the calls below take Heads."""
    tensor: Tensor
    heads: int
    dim: int
    first: int = 0


def _columns(x, name):
    """Heads, or a tensor [rows][heads][dim], as (tensor, heads, dim, first, elements of a row)."""
    if isinstance(x, Heads):
        t, heads, dim, first = x
        if len(t.shape) != 2:
            raise ValueError(f"{name}: Heads are columns of a tensor [rows][width], got shape {t.shape}")
        width = t.shape[1]
        if first < 0 or heads < 0 or dim < 0 or first + heads * dim > width:
            raise ValueError(f"{name}: columns {first} to {first + heads * dim} of a tensor of width {width}")
        return t, heads, dim, first, width
    if len(x.shape) != 3:
        raise ValueError(f"{name}: shape {x.shape}, expected [rows][heads][dim] or Heads of [rows][width]")
    _, heads, dim = x.shape
    return x, heads, dim, 0, heads * dim


# The params of the calls below as the bytes of their C structs (ctypes structs take as long to fill as a launch takes).
_ROPE_PARAMS = struct.Struct("=qqqiiiiif")
_ATTENTION_PARAMS = struct.Struct("=qqiiiifi12q")
_PAGED_PARAMS = struct.Struct("=qqqqiiiifi6q")


def _pack(params: struct.Struct, *values) -> bytes:
    try:
        return params.pack(*values)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"{values}: {e}") from None


def rope_frequencies(rot: int, base: float = 10000.0, factor: float = 1.0, trained: int = 0, kind: str = "ramp") -> np.ndarray:
    """The frequencies of rope's rot / 2 pairs, f32 [2][rot / 2]: turns per position (base^(-2 i / rot) / 2 pi, formed in 64
    bits) and what 32 bits leave of them.  factor > 1 stretches them for contexts that much longer than the trained ones:
    kind "linear" divides every frequency by it; "base" raises the base to base * factor^(rot / (rot - 2)), which leaves the
    fastest pair and divides the slowest one; "ramp" (YaRN, Peng et al. 2023) divides the pairs that turn less than once
    over the `trained` positions, keeps those that turn more than 32 times, and goes from one to the other linearly between
    (its magnitude is 0.1 log(factor) + 1)."""
    if rot < 0 or rot % 2:
        raise ValueError(f"rope_frequencies: rot {rot} is not an even number of columns")
    if not (base > 1.0 and factor >= 1.0 and np.isfinite(base) and np.isfinite(factor)):
        raise ValueError("rope_frequencies: base must be above 1 and factor at least 1")
    i = np.arange(rot // 2, dtype=np.float64)
    if kind == "base" and factor > 1.0:
        if rot <= 2:
            raise ValueError("rope_frequencies: kind 'base' needs two pairs or more")
        base = base * factor ** (rot / (rot - 2.0))
    f = base ** (-2.0 * i / max(rot, 1))
    if kind == "linear":
        f = f / factor
    elif kind == "ramp":
        if factor > 1.0:
            if trained <= 0:
                raise ValueError("rope_frequencies: kind 'ramp' needs the number of trained positions")
            pair = [rot * np.log(trained / (2.0 * np.pi * turns)) / (2.0 * np.log(base)) for turns in (32.0, 1.0)]
            lo, hi = max(0.0, np.floor(pair[0])), min(rot - 1.0, np.ceil(pair[1]))
            ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
            f = f * (1.0 - ramp) + f / factor * ramp
    elif kind != "base":
        raise ValueError(f"rope_frequencies: unknown kind {kind!r}")
    turns = f / (2.0 * np.pi)
    hi = turns.astype(np.float32)
    return np.stack([hi, (turns - hi).astype(np.float32)])


def rope(q: Queue, x: Tensor, positions: Tensor, freqs: Tensor, y: Tensor, heads: int, dim: int, first: int = 0,
         interleaved: bool = False, inverse: bool = False, magnitude: float = 1.0):
    """y = x [rows][width] with `heads` heads of `dim` columns, from column `first` on, turned by positions (i32 [rows]): the first
    2 * pairs columns of each, freqs f32 [2][pairs] (rope_frequencies); the other columns are handed on.  Pairs are columns
    (i, i + pairs), or (2 i, 2 i + 1) if interleaved.  inverse: the gradient, dx from dy.  y may be x (one dtype)."""
    rows, width = x.shape
    if y.shape != (rows, width):
        raise ValueError(f"y: shape {y.shape}, expected {(rows, width)}")
    _expect(positions, (rows,), "i32", "positions")
    _expect(freqs, (2, freqs.shape[-1]), "f32", "freqs")
    p = _pack(_ROPE_PARAMS, rows, width, first, heads, dim, freqs.shape[1], bool(interleaved), bool(inverse), magnitude)
    call("vdsl_op_rope", q.handle, p, x.dtype, x.handle, positions.handle, freqs.handle, y.dtype, y.handle)


def _attention_operands(qh, k, v, starts, out, lse, scale):
    """q, k and v as _columns gives them, checked against each other, and the scale."""
    qt, heads, dim, _, _ = qc = _columns(qh, "q")
    kt, kv_heads, _, _, _ = kc = _columns(k, "k")
    vc = _columns(v, "v")
    n = qt.shape[0]
    for name, (t, of, columns, _, _), expected in (("q", qc, heads), ("k", kc, kv_heads), ("v", vc, kv_heads)):
        if t.dtype != _lib.BF16:
            raise ValueError(f"{name}: dtype {t.dtype}, expected bf16")
        if t.shape[0] != n or columns != dim or of != expected:
            raise ValueError(f"{name}: {t.shape[0]} rows of {of} heads of {columns}, expected {n} rows of {expected} heads of {dim}")
    if len(starts.shape) != 1 or starts.numel < 1:
        raise ValueError(f"starts: shape {starts.shape}, expected one more element than there are sequences")
    if starts.dtype != _lib.I32:
        raise ValueError(f"starts: dtype {starts.dtype}, expected i32")
    if out.numel != n * heads * dim or out.shape[0] != n:
        raise ValueError(f"out: shape {out.shape}, expected {(n, heads * dim)}")
    _expect(lse, (heads, n), "f32", "lse")
    return qc, kc, vc, float(dim) ** -0.5 if scale is None and dim else scale


def attention_fwd(q: Queue, qh, k, v, starts: Tensor, out: Tensor, lse=None, causal: bool = True, scale=None):
    """out [n][heads * dim] (f32 or bf16) = softmax(scale q k^T) v over packed sequences: rows starts[s] to starts[s + 1] (i32
    [seqs + 1]) see each other, earlier ones only if causal.  q, k, v: bf16 Heads, or tensors [n][heads][dim]; kv heads divide
    the heads.  scale: 1 / sqrt(dim) if None.  lse (f32 [heads][n], optional): log of the scores' exponentials' sum, kept for
    attention_bwd.  Rows of no sequence get 0, lse -inf."""
    qc, kc, vc, scale = _attention_operands(qh, k, v, starts, out, lse, scale)
    qt, kt, vt = qc[0], kc[0], vc[0]
    p = _pack(_ATTENTION_PARAMS, qt.shape[0], starts.numel - 1, qc[1], kc[1], qc[2], bool(causal), scale, 0, *qc[3:], *kc[3:], *vc[3:],
              0, 0, 0, 0, 0, 0)
    call("vdsl_op_attention_fwd", q.handle, p, qt.handle, kt.handle, vt.handle, starts.handle, out.dtype, out.handle, _h(lse))


def attention_bwd_workspace_bytes(n, seqs, heads, kv_heads, dim) -> int:
    """Never less for more rows or sequences: a workspace for the largest batch serves smaller ones."""
    b = C.c_size_t()
    call("vdsl_attention_bwd_workspace_bytes", n, seqs, heads, kv_heads, dim, C.byref(b))
    return b.value


def attention_bwd(q: Queue, dout: Tensor, qh, k, v, starts: Tensor, out: Tensor, lse: Tensor, dq, dk, dv, causal: bool = True,
                  scale=None, workspace=None):
    """The gradients dq, dk, dv (Heads or tensors [n][heads][dim], all f32 or all bf16; disjoint columns of one tensor if they
    like) of attention_fwd from dout [n][heads * dim] (f32 or bf16) and the forward pass's out and lse.  workspace:
    attention_bwd_workspace_bytes(n, seqs, heads, kv_heads, dim) bytes."""
    qc, kc, vc, scale = _attention_operands(qh, k, v, starts, out, lse, scale)
    qt, kt, vt = qc[0], kc[0], vc[0]
    n = qt.shape[0]
    if dout.numel != out.numel or dout.shape[0] != n:
        raise ValueError(f"dout: shape {dout.shape}, expected {out.shape}")
    dqc, dkc, dvc = _columns(dq, "dq"), _columns(dk, "dk"), _columns(dv, "dv")
    dtype = dqc[0].dtype
    for name, (t, of, columns, _, _), x in (("dq", dqc, qc), ("dk", dkc, kc), ("dv", dvc, vc)):
        if t.shape[0] != n or of != x[1] or columns != x[2]:
            raise ValueError(f"{name}: {t.shape[0]} rows of {of} heads of {columns}, expected {n} rows of {x[1]} heads of {x[2]}")
        if t.dtype != dtype:
            raise ValueError("dq, dk and dv must be of one dtype")
    p = _pack(_ATTENTION_PARAMS, n, starts.numel - 1, qc[1], kc[1], qc[2], bool(causal), scale, 0, *qc[3:], *kc[3:], *vc[3:],
              *dqc[3:], *dkc[3:], *dvc[3:])
    call("vdsl_op_attention_bwd", q.handle, p, dout.dtype, dout.handle, qt.handle, kt.handle, vt.handle, starts.handle, out.dtype,
         out.handle, _h(lse), dtype, dqc[0].handle, dkc[0].handle, dvc[0].handle, _h(workspace))


def _paged_params(n, dim, kv_heads, heads, scale, starts, lengths, table, k_cache, v_cache, *layouts):
    """starts, lengths and table against the caches [pages][kv_heads][page][dim]; the params, with first and stride of q, k and v."""
    shape = k_cache.shape
    if len(shape) != 4 or shape[1] != kv_heads or shape[3] != dim:
        raise ValueError(f"k_cache: shape {shape}, expected [pages][{kv_heads}][page][{dim}]")
    if k_cache.dtype != _lib.BF16:
        raise ValueError(f"k_cache: dtype {k_cache.dtype}, expected bf16")
    _expect(v_cache, shape, "bf16", "v_cache")
    (seqs,) = lengths.shape
    _expect(starts, (seqs + 1,), "i32", "starts")
    _expect(lengths, (seqs,), "i32", "lengths")
    if len(table.shape) != 2:
        raise ValueError(f"table: shape {table.shape}, expected [seqs][pages of a sequence]")
    _expect(table, (seqs, table.shape[1]), "i32", "table")
    return _pack(_PAGED_PARAMS, n, seqs, shape[0], table.shape[1], shape[2], heads, kv_heads, dim, scale, 0, *layouts)


def cache_append(q: Queue, k, v, starts: Tensor, lengths: Tensor, table: Tensor, k_cache: Tensor, v_cache: Tensor):
    """The new rows' k and v (bf16 Heads or tensors [n][kv_heads][dim]) into their slots of the paged caches (bf16
    [pages][kv_heads][page][dim], page a power of two from 16 on): row i of the m new rows starts[s] to starts[s + 1] of sequence s is
    position p = lengths[s] - m + i, slot p % page of page table[s][p / page] (i32; lengths counts the new rows).  Rows without
    a page are dropped."""
    kt, heads, dim, k_first, k_stride = _columns(k, "k")
    vt, v_heads, v_dim, v_first, v_stride = _columns(v, "v")
    n = kt.shape[0]
    for t, name in ((kt, "k"), (vt, "v")):
        if t.dtype != _lib.BF16:
            raise ValueError(f"{name}: dtype {t.dtype}, expected bf16")
    if vt.shape[0] != n or v_heads != heads or v_dim != dim:
        raise ValueError(f"v: {vt.shape[0]} rows of {v_heads} heads of {v_dim}, expected {n} rows of {heads} heads of {dim}")
    p = _paged_params(n, dim, heads, heads, 1.0, starts, lengths, table, k_cache, v_cache, 0, 0, k_first, k_stride, v_first, v_stride)
    call("vdsl_op_cache_append", q.handle, p, kt.handle, vt.handle, starts.handle, lengths.handle, table.handle, k_cache.handle, v_cache.handle)


def paged_attention_workspace_bytes(n, seqs, heads, kv_heads, dim, positions) -> int:
    """positions: those that a row of the page table has room for (its pages times the page size).  May be more for fewer rows, which
    are split into more parts: one workspace for calls of several sizes is the largest of theirs."""
    b = C.c_size_t()
    call("vdsl_paged_attention_workspace_bytes", n, seqs, heads, kv_heads, dim, positions, C.byref(b))
    return b.value


def paged_attention(q: Queue, qh, k_cache: Tensor, v_cache: Tensor, starts: Tensor, lengths: Tensor, table: Tensor, out: Tensor, lse=None,
                    scale=None, workspace=None):
    """Attention of new rows over a paged cache that holds their own keys already (cache_append): the row at position p sees
    positions 0 to p of its sequence.  qh: bf16 Heads or a tensor [n][heads][dim]; out [n][heads * dim], lse and scale as
    for attention_fwd.  workspace: paged_attention_workspace_bytes(...) bytes; with fewer, or None, the positions are split into as
    many parts as fit, which takes longer."""
    qt, heads, dim, first, stride = _columns(qh, "q")
    n = qt.shape[0]
    if qt.dtype != _lib.BF16:
        raise ValueError(f"q: dtype {qt.dtype}, expected bf16")
    if out.numel != n * heads * dim or out.shape[0] != n:
        raise ValueError(f"out: shape {out.shape}, expected {(n, heads * dim)}")
    _expect(lse, (heads, n), "f32", "lse")
    kv_heads = k_cache.shape[1] if len(k_cache.shape) == 4 else 0
    p = _paged_params(n, dim, kv_heads, heads, float(dim) ** -0.5 if scale is None and dim else scale, starts, lengths, table, k_cache,
                      v_cache, first, stride, 0, 0, 0, 0)
    call("vdsl_op_paged_attention", q.handle, p, qt.handle, k_cache.handle, v_cache.handle, starts.handle, lengths.handle,
         table.handle, out.dtype, out.handle, _h(lse), _h(workspace))
