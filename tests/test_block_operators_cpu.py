"""Host-side checks of a block's operators that need no GPU: struct layouts, refusals that come
before any device work, the scan of their assembly, and the tests' own generator."""
import ctypes as C
import os
import subprocess

import pytest

import block_util as B
from conftest import REPO
from test_isa_cpu import HIPCC, PKG, scc_reads_live_into_a_block

FILES = ("dropout", "layer_norm", "embedding", "linear", "linear_to_bf16", "linear_to_fp32")


def test_struct_layouts_match_the_header(tmp_path):
    from ttperf import _lib as L
    structs = {"ttp_dropout": L.Dropout, "ttp_linear_args": L.LinearArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ttperf/ttperf.h"',
             "int main(void) {"]
    for cname, ct in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        for f, _ in ct._fields_:
            lines.append(f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));')
    for n in ("NONE", "RELU", "GELU_ERF", "GELU_TANH"):
        lines.append(f'printf("{n} %d\\n", TTP_ACTIVATION_{n});')
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
        assert int(got[cname]) == C.sizeof(ct), cname
        for f, _ in ct._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(ct, f).offset, f"{cname}.{f}"
    for n in ("NONE", "RELU", "GELU_ERF", "GELU_TANH"):
        assert int(got[n]) == getattr(L, f"ACTIVATION_{n}")


def test_a_null_context_is_refused():
    from ttperf import _lib as L
    m, d = L.Matrix(), L.Dropout()
    assert L.lib.ttp_dropout_forward(None, d, m, None, m) == L.ERR_INVALID
    assert L.lib.ttp_embedding(None, 0, None, 1.0, L.NO_TENSOR, None, m) == L.ERR_INVALID
    assert L.lib.ttp_accumulate_embedding_grad(None, 0, None, 1.0, m) == L.ERR_INVALID
    assert L.lib.ttp_layer_norm(None, 0, 1, m, 1e-5, m, None, None) == L.ERR_INVALID
    assert L.lib.ttp_layer_norm_backward(None, 0, 1, m, m, None, None, None, m) == L.ERR_INVALID
    assert L.lib.ttp_linear(None, L.LinearArgs()) == L.ERR_INVALID


@pytest.mark.parametrize("name", FILES)
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


def test_the_generator_gives_the_published_known_answers():
    """Philox 4x32-10's known answers, as its authors' library lists them."""
    ones, pi = 2 ** 32 - 1, (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344)
    for key, counter, want in (
            ((0, 0), (0, 0, 0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones, ones), (ones,) * 4, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0xA4093822, 0x299F31D0), pi, (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w) for w in B.philox(key, counter)) == want
