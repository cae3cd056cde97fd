"""The transfers to LDS of the tiled products read scalar registers in inline assembly: compile their sources for gfx950 and check
that no such register was written by a vector instruction fewer than five wait states before (CPU only).  The check itself is
tested on hand-written fragments."""
import subprocess
from pathlib import Path

import pytest

import scalar_wait_check as S

REPO = Path(__file__).resolve().parents[1]
CSRC = REPO / "coding-basic-hw-2_amd" / "csrc"
SOURCES = ("mx4gemm.hip", "w8gemm.hip", "glu.hip")


def test_check_counts_wait_states():
    def asm(n, between=()):
        return ["\tv_readlane_b32 s1, v96, 3", *between, "\ts_mov_b32 m0, s7", f"\ts_nop {n}", "\tglobal_load_lds_dwordx4 v4, s[0:1]",
                "\ts_endpgm"]
    assert [(t, r) for _, t, r in S.check_kernel(asm(0))] == [("global_load_lds_dwordx4 v4, s[0:1]", (1,))]
    assert S.check_kernel(asm(2)) and not S.check_kernel(asm(3))
    assert not S.check_kernel(asm(0, ["\tv_add_u32_e32 v1, v2, v3"] * 3)) and S.check_kernel(asm(0, ["\tv_add_u32_e32 v1, v2, v3"] * 2))
    assert not S.check_kernel(asm(0, ["\ts_addc_u32 s1, s1, 0"]))          # written again, by the scalar unit
    assert S.check_kernel(["\tv_cmp_eq_u32_e64 s[2:3], v0, v1", "\tbuffer_load_dwordx4 v1, s[0:3], 0 offen lds", "\ts_endpgm"])
    assert not S.check_kernel(["\tv_cmp_eq_u32_e64 s[4:5], v0, v1", "\tbuffer_load_dwordx4 v1, s[0:3], 0 offen lds", "\ts_endpgm"])


def test_check_takes_the_shortest_way():
    asm = ["\tv_readfirstlane_b32 s0, v1", "\ts_cbranch_scc1 .LBB0_2", "\ts_nop 4", ".LBB0_2:", "\ts_nop 2",
           "\tbuffer_load_dwordx4 v1, s[0:3], 0 offen lds", "\ts_endpgm"]
    assert [r for _, _, r in S.check_kernel(asm)] == [(0,)]
    asm[4] = "\ts_nop 3"
    assert not S.check_kernel(asm)
    # around a loop
    assert S.check_kernel([".LBB0_1:", "\tbuffer_load_dwordx4 v1, s[0:3], 0 offen lds", "\tv_readlane_b32 s2, v9, 1", "\ts_cbranch_scc1 .LBB0_1",
                           "\ts_endpgm"])


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """{source: (compiler, its output)}, all of them under way at once."""
    def start(source):
        out = tmp_path_factory.mktemp("asm") / "kernels.s"
        cmd = ["/opt/rocm/bin/hipcc", "-O3", "-std=c++17", "-fPIC", f"-I{REPO / 'include'}", f"-I{CSRC}", "-x", "hip", "--offload-arch=gfx950",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unused-command-line-argument", "--cuda-device-only", "-S",
               str(CSRC / source), "-o", str(out)]
        return subprocess.Popen(cmd, stderr=subprocess.DEVNULL), out
    return {source: start(source) for source in SOURCES}


@pytest.mark.parametrize("source", SOURCES)
def test_transfers_wait_for_scalar_registers(assembly, source):
    compiler, out = assembly[source]
    assert compiler.wait(timeout=600) == 0
    found, transfers = S.check(out)
    assert transfers > 500
    assert not found, [(k[:60], v[:2]) for k, v in found.items()]
