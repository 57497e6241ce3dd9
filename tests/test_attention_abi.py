"""The structs of the attention operators as the C header and ctypes lay them out, and what their workspaces' sizes take and refuse."""
import ctypes as C
import os
import subprocess

import pytest

from vernondsl_amd import _lib, kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"vdsl_heads": _lib.Heads, "vdsl_rope_params": _lib.RopeParams, "vdsl_attention_params": _lib.AttentionParams,
           "vdsl_paged_params": _lib.PagedParams}


def test_struct_layouts(tmp_path):
    lines, want = [], []
    for name, struct in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(struct))
        for field, _ in struct._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(struct, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "vdsl.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{os.path.join(ROOT, 'include')}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def test_workspace_sizes():
    # one row and head: -lse / scale, -delta, dout in bf16
    base = kernels.attention_bwd_workspace_bytes(0, 1, 4, 2, 64)
    assert kernels.attention_bwd_workspace_bytes(10, 1, 4, 2, 64) == base + 10 * 4 * (8 + 2 * 64)
    # one sequence of few positions is not split; a long one is, by less than its share of 64 positions
    assert kernels.paged_attention_workspace_bytes(1, 1, 32, 8, 128, 64) == 0
    need = kernels.paged_attention_workspace_bytes(1, 1, 32, 8, 128, 1 << 17)
    assert need % (32 * (8 + 4 * 128)) == 0 and 2 <= need // (32 * (8 + 4 * 128)) <= 256
    assert kernels.paged_attention_workspace_bytes(0, 0, 32, 8, 128, 1 << 17) == 0


@pytest.mark.parametrize("args", [(-1, 1, 4, 2, 64), (1, -1, 4, 2, 64), (1, 1, 4, 3, 64), (1, 1, 0, 0, 64), (1, 1, 4, 2, 0), (1, 1, 4, 2, 60),
                                  (1, 1, 4, 2, 136), (1 << 40, 1, 4, 2, 64), (1, 1 << 40, 4, 2, 64)])
def test_workspace_refusals(args):
    with pytest.raises(_lib.VdslError):
        kernels.attention_bwd_workspace_bytes(*args)
    with pytest.raises(_lib.VdslError):
        kernels.paged_attention_workspace_bytes(*args, 100)


def test_positions_are_not_negative():
    with pytest.raises(_lib.VdslError):
        kernels.paged_attention_workspace_bytes(1, 1, 4, 2, 64, -1)


@pytest.mark.parametrize("call,params,operands", [("vdsl_op_rope", _lib.RopeParams, 6), ("vdsl_op_attention_fwd", _lib.AttentionParams, 7),
                                                  ("vdsl_op_attention_bwd", _lib.AttentionParams, 14), ("vdsl_op_cache_append", _lib.PagedParams, 7),
                                                  ("vdsl_op_paged_attention", _lib.PagedParams, 10)])
def test_no_queue(call, params, operands):
    fn = getattr(_lib.lib, call)
    assert len(fn.argtypes) == 2 + operands
    assert fn(None, C.byref(params()), *[0 if t is C.c_int32 else None for t in fn.argtypes[2:]]) != 0


def flat(struct):
    """A ctypes struct's values in order."""
    out = []
    for name, kind in struct._fields_:
        value = getattr(struct, name)
        out += flat(value) if issubclass(kind, C.Structure) else [value]
    return out


@pytest.mark.parametrize("packed,struct", [(kernels._ROPE_PARAMS, _lib.RopeParams), (kernels._ATTENTION_PARAMS, _lib.AttentionParams),
                                           (kernels._PAGED_PARAMS, _lib.PagedParams)])
def test_packed_params(packed, struct):
    raw = bytes((7 * i + 1) % 113 for i in range(C.sizeof(struct)))
    x = struct.from_buffer_copy(raw)
    assert kernels._pack(packed, *flat(x)) == bytes(x) == raw


def test_params_that_do_not_fit():
    fine = [1, 1, 1, 1, 8, 1, 1.0, 0] + [0] * 12
    kernels._pack(kernels._ATTENTION_PARAMS, *fine)
    for at, value in ((0, 1 << 63), (2, 1 << 31), (6, 1e39), (6, None)):
        with pytest.raises(ValueError):
            kernels._pack(kernels._ATTENTION_PARAMS, *(value if i == at else x for i, x in enumerate(fine)))
