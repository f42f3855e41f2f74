"""No kernel of the built library reads an SGPR in a vector-memory instruction too soon after a vector instruction wrote
it (wait_states.py), and the reader of the listings finds such pairs where there are any.  No GPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

from laya_cuda import _lib
from wait_states import functions, hazards

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"


def listing(*lines):
    return "\n".join(["0000000000001000 <kernel>:"] + [f"\t{line:60s}// {0x1000 + 4 * i:012X}: 00000000" for i, line in enumerate(lines)])


LOAD = "buffer_load_dwordx4 v1, s[8:11], s20 offen lds"


@pytest.mark.parametrize("lines,states", [
    (["v_readfirstlane_b32 s20, v3", "s_nop 0", LOAD], 1),
    (["v_readfirstlane_b32 s9, v3", "s_nop 2", LOAD], 3),
    (["v_readlane_b32 s11, v40, 3", "s_nop 1", "v_mov_b32_e32 v5, v6", LOAD], 3),
    (["v_cmp_eq_u32_e64 s[20:21], v0, v1", LOAD], 0),
    (["v_add_co_u32 v1, vcc, v2, v3", "global_load_dword v4, v5, vcc"], 0),
    (["s_branch 2", "v_readfirstlane_b32 s20, v3", "s_branch 2", "s_nop 0", "s_nop 0", LOAD], 1),  # over a forward branch
    ([LOAD, "s_nop 4", "v_readfirstlane_b32 s20, v3", "s_cbranch_scc1 65532"], 1),  # over a loop's end
])
def test_planted_pairs_are_found(lines, states):
    found = hazards(listing(*lines))
    assert [f[3] for f in found] == [states]


@pytest.mark.parametrize("lines", [
    ["v_readfirstlane_b32 s20, v3", "s_nop 4", LOAD],
    ["v_readfirstlane_b32 s21, v3", LOAD],  # another register
    ["v_readfirstlane_b32 s21, v3", "s_mov_b32 s20, s21", LOAD],  # a scalar copy, a read that the hardware checks
    ["v_readfirstlane_b32 s20, v3", "s_nop 1", "v_mov_b32_e32 v5, v6", "v_mov_b32_e32 v5, v6", "s_add_u32 s3, s3, 1", LOAD],
    ["v_readfirstlane_b32 s20, v3", "s_endpgm", LOAD],
])
def test_allowed_pairs_are_not(lines):
    assert not hazards(listing(*lines))


@pytest.mark.skipif(not Path(OBJDUMP).is_file(), reason="llvm-objdump is not installed")
@pytest.mark.skipif(not _lib.LIBRARY.is_file(), reason="the library is not built")
def test_the_built_kernels_have_none(tmp_path):
    library = tmp_path / "lib.so"
    shutil.copy(_lib.LIBRARY, library)
    subprocess.run([OBJDUMP, "--offloading", str(library)], cwd=tmp_path, check=True, capture_output=True, timeout=60)
    kernels, loads, found = 0, 0, []
    for code in sorted(tmp_path.glob("*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(code)], check=True, capture_output=True, text=True, timeout=60).stdout
        kernels += len(functions(text))
        loads += text.count(" lds ")
        found += hazards(text)
    assert kernels > 200 and loads > 1000  # the listing was read
    assert not found, found[:5]
