"""Host-side checks of the fine-tuning operators that need no GPU: struct layouts, refusals that
come before any device work, and the scan of their assembly."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import REPO
from test_isa_cpu import HIPCC, PKG, scc_reads_live_into_a_block

OPERATOR_FILES = ("losses", "checkpoint8", "linear_grad8")


def test_struct_layouts_match_the_header(tmp_path):
    from ttperf import _lib as L
    structs = {"ttp_matrix": L.Matrix, "ttp_preference_args": L.PreferenceArgs,
               "ttp_policy_args": L.PolicyArgs, "ttp_checkpoint8": L.Checkpoint8}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ttperf/ttperf.h"',
             "int main(void) {"]
    for cname, ct in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for f, _ in ct._fields_:
            lines.append(f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));')
    lines.append("return 0; }")
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(REPO, "include"), "-o", str(exe),
                    str(src)], check=True)
    got = dict(line.rsplit(" ", 1) for line in
               subprocess.run([str(exe)], capture_output=True, text=True,
                              check=True).stdout.splitlines())
    for cname, ct in structs.items():
        assert int(got[f"{cname} size"]) == C.sizeof(ct), cname
        for f, _ in ct._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(ct, f).offset, f"{cname}.{f}"


def test_a_null_context_is_refused():
    from ttperf import _lib as L
    m = L.Matrix()
    assert L.lib.ttp_token_logprobs(None, C.byref(m), None, None) == L.ERR_INVALID
    assert L.lib.ttp_preference_loss(None, C.byref(L.PreferenceArgs())) == L.ERR_INVALID
    assert L.lib.ttp_policy_loss(None, C.byref(L.PolicyArgs())) == L.ERR_INVALID
    k = L.Checkpoint8()
    assert L.lib.ttp_checkpoint8_pack(None, C.byref(m), C.byref(k)) == L.ERR_INVALID
    assert L.lib.ttp_checkpoint8_restore(None, C.byref(k), C.byref(m)) == L.ERR_INVALID
    assert L.lib.ttp_gelu_checkpoint8(None, C.byref(m), 0, C.byref(m), C.byref(k)) == \
        L.ERR_INVALID
    assert L.lib.ttp_accumulate_linear_grad8(None, 0, 1, C.byref(k), C.byref(m), 0) == \
        L.ERR_INVALID
    assert L.lib.ttp_gelu_backward8(None, C.byref(k), 0, C.byref(m), C.byref(m)) == L.ERR_INVALID


@pytest.mark.parametrize("name", OPERATOR_FILES)
def test_no_scc_read_is_live_into_a_block(name, tmp_path):
    """The scan of tests/test_isa_cpu.py on the operators' assembly."""
    if not os.access(HIPCC, os.X_OK):
        pytest.skip("hipcc absent")
    subprocess.run(["make", "-s", "-C", PKG, f"isa-{name}", f"ISA_DIR={tmp_path}"], check=True,
                   capture_output=True, timeout=900)
    asm = open(tmp_path / f"{name}.s").read()
    bad = scc_reads_live_into_a_block(asm.splitlines())
    assert not bad, "SCC read before any write in its block:\n" + "\n".join(
        f"  {name}.s:{ln} {fn[:80]} {blk}: {ins}" for ln, fn, blk, ins in bad[:20])
    assert "v_pk_add_f32" not in asm and "v_pk_mul_f32" not in asm and "v_pk_fma_f32" not in asm
