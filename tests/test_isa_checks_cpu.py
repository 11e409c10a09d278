"""CPU: the checks of the kernels' ISA (tools/scan_*.py) on planted sequences."""
import importlib.util
import os

from conftest import ROOT


def _tool(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "tools", name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


LOOP = """
_Z4kernPf:
; %bb.0:
\tv_mov_b32_e32 v0, 0
.LBB0_1:                                ; =>This Inner Loop Header: Depth=1
\ts_barrier
\tds_read_b32 v1, v0
\ts_waitcnt lgkmcnt(0){wait}
\tds_write_b32 v0, v1
\ts_cbranch_scc1 .LBB0_1
; %bb.2:
\ts_endpgm
.section .rodata
"""


def test_barrier_check_follows_loops_whose_header_carries_a_comment():
    """A loop header's label has a comment behind it; the write at the loop's end reaches the barrier at its top."""
    scan = _tool("scan_barrier_waits")
    ins = scan._kernels(LOOP.format(wait="").split("\n"))["_Z4kernPf"]
    assert ".LBB0_1:" in ins
    assert scan._scan_function(ins) == (1, 1)
    waited = LOOP.replace("\ts_barrier", "\ts_waitcnt lgkmcnt(0)\n\ts_barrier")
    assert scan._scan_function(scan._kernels(waited.format(wait="").split("\n"))["_Z4kernPf"]) == (1, 0)
