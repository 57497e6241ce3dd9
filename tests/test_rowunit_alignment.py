"""The units of a row start at any element, so the kernels' vector accesses may promise the compiler no more than an
element's alignment, and must stay one instruction each all the same: rowunit.h's loads and stores as compiled here."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vernondsl_amd", "csrc")
HIPCC = os.environ.get("HIPCC") or shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
KINDS = [(dt, u, stream) for dt in ("F32", "BF16") for u in (4, 8) for stream in ("false", "true")]


@pytest.fixture(scope="module")
def compiled(tmp_path_factory):
    """{(type, unit, stream): (LLVM IR, assembly)} of a kernel that copies one unit."""
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    d = tmp_path_factory.mktemp("rowunit")
    src = '#include "rowunit.h"\nusing namespace vdsl;\n'
    for dt, u, stream in KINDS:
        src += (f'extern "C" __global__ void copy_{dt}_{u}_{stream}(const void* a, void* b, int64_t e) {{\n'
                f"  float v[{u}];\n  e += threadIdx.x;\n  load_whole<VDSL_{dt}, {u}>(a, e, v);\n  store_whole<VDSL_{dt}, {u}, {stream}>(b, e, v);\n}}\n")
    (d / "unit.hip").write_text(src)
    cmd = [HIPCC, "--offload-arch=gfx950", "--cuda-device-only", "-O3", "-std=c++17", "-I", CSRC, "-I",
           os.path.join(CSRC, "..", "..", "include"), "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", str(d / "unit.hip")]
    for extra in (["-S", "-emit-llvm", "-o", str(d / "unit.ll")], ["-S", "-o", str(d / "unit.s")]):
        subprocess.run(cmd + extra, check=True, capture_output=True)
    ir, asm, out = (d / "unit.ll").read_text(), (d / "unit.s").read_text(), {}
    for dt, u, stream in KINDS:
        name = f"copy_{dt}_{u}_{stream}"
        out[dt, u, stream] = (re.search(r"define[^\n]*@%s\(.*?\n}" % name, ir, re.S).group(0),
                              re.search(r"\n%s:.*?s_endpgm" % name, asm, re.S).group(0))
    return out


@pytest.mark.parametrize("dt,u,stream", KINDS)
def test_accesses_promise_an_elements_alignment_and_stay_whole(compiled, dt, u, stream):
    ir, asm = compiled[dt, u, stream]
    element = 4 if dt == "F32" else 2
    aligns = [int(a) for a in re.findall(r"(?:load|store) <\d+ x \w+>.*?align (\d+)", ir)]
    accesses = 2 * (u // 4 if dt == "F32" else 1)
    assert len(aligns) == accesses and set(aligns) == {element}
    width = "dwordx2" if dt == "BF16" and u == 4 else "dwordx4"
    assert len(re.findall(r"global_(?:load|store)_" + width, asm)) == accesses
    assert len(re.findall(r"global_(?:load|store)_", asm)) == accesses
    assert len(re.findall(r"global_store_\w+ .* nt\b", asm)) == (accesses // 2 if stream == "true" else 0)
