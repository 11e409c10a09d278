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


def _hits(*lines):
    scan = _tool("scan_asm_hazards")
    text = ["_Z4kernPf:"]
    for l in lines:
        text += [";;#ASMSTART", *("\t" + x for x in l), ";;#ASMEND"] if isinstance(l, tuple) else [l if l.endswith(":") else "\t" + l]
    return [h[:2] for hits in scan.scan_lines(scan.marked("\n".join([*text, "\ts_endpgm"]))).values() for h in hits]


DMA = "buffer_load_dwordx4 v55, s[44:47], s2 offen lds"
MFMA = "v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], a[0:15]"


def test_wait_state_check():
    """What an asm block reads too early is found, over block ends and round loops; what waits, and what hipcc issues itself, is not."""
    assert _hits("v_readlane_b32 s2, v254, 18", (DMA,)) == [(0, 5)]
    assert _hits("v_readlane_b32 s2, v254, 18", DMA) == []
    assert _hits("v_readfirstlane_b32 s45, v1", ("s_mov_b32 m0, s7", "s_nop 0", DMA)) == [(2, 5)]
    assert _hits("v_readfirstlane_b32 s45, v1", ("s_mov_b32 m0, s7", "s_nop 3", DMA)) == []
    assert _hits("v_readlane_b32 s2, v254, 18", "s_mov_b32 s2, s3", (DMA,)) == []
    assert _hits("s_cbranch_scc0 .LBB0_2", "v_readfirstlane_b32 s2, v1", ".LBB0_2:", (DMA,)) == [(0, 5)]
    assert _hits(".LBB0_1:", (DMA,), "v_readfirstlane_b32 s2, v1", "s_cbranch_scc1 .LBB0_1") == [(1, 5)]
    assert _hits("v_cmp_gt_f32_e64 s[4:5], v1, v2", ("v_addc_co_u32 v0, vcc, v0, v0, s[4:5]",)) == [(0, 2)]
    assert _hits("v_cmp_gt_f32_e64 s[4:5], v1, v2", ("s_nop 1", "v_addc_co_u32 v0, vcc, v0, v0, s[4:5]")) == []
    assert _hits(MFMA, ("v_accvgpr_read_b32 v9, a3",)) == [(0, 12)]
    assert _hits(MFMA, ("s_nop 11", "v_accvgpr_read_b32 v9, a3")) == []
    assert _hits(("v_max_f32 v1, v2, v3",), "v_permlane32_swap_b32_e32 v1, v4") == [(0, 2)]
    assert _hits(("v_max_f32 v1, v2, v3",), "s_nop 1", "v_permlane32_swap_b32_e32 v1, v4") == []
    load = ("buffer_load_dwordx4 v[0:3], v9, s[0:3], s4 offen",)
    assert _hits(load, "v_mov_b32_e32 v9, v2") == [(-1, 0)]
    assert _hits(load, "buffer_store_dword v8, v9, s[0:3], 0 offen", ("s_waitcnt vmcnt(1)",), "v_mov_b32_e32 v9, v2") == []
    assert _hits(load, "buffer_store_dword v8, v9, s[0:3], 0 offen", ("s_waitcnt vmcnt(2)",), "v_mov_b32_e32 v9, v2") == [(-1, 0)]
    group = ("s_mov_b32 m0, s9", "s_nop 0"), ("s_nop 4", DMA), "v_add_u32_e32 v1, v1, v2", ("s_nop 4", "buffer_load_dwordx4 v55, s[44:47], s2 offen offset:1024 lds")
    assert _hits(*group) == []
    assert _hits(*group[:3], "s_mov_b32 m0, s3", group[3]) == [(-2, 0)]


def _scan(path):
    return path, _tool("scan_asm_hazards").scan(path)


def test_no_asm_block_reads_too_early():
    """Every kernel of the sources whose asm blocks hold vector or memory instructions, themselves or in a source that they include."""
    import concurrent.futures as cf
    import glob
    import re

    csrc = os.path.join(ROOT, "satflow_amd", "csrc")

    def has_asm(path):
        text = open(path).read()
        return re.search(r'\basm(?: volatile)?\((?:\s*"[^"]*")*?\s*"(?:[^"]*(?:\\t|\s))?(?:buffer_|global_|ds_|v_)', text) is not None or any(
            has_asm(os.path.join(csrc, m)) for m in re.findall(r'#include "([^"/]+\.hip)"', text))

    files = [f for f in sorted(glob.glob(os.path.join(csrc, "*.hip"))) if has_asm(f)]
    assert {"conv3x3_bf16.hip", "conv3x3_f16.hip", "conv3x3_bf16_persist4.hip", "convgru_seq.hip"} <= {os.path.basename(f) for f in files}
    bad = []
    with cf.ProcessPoolExecutor(max_workers=min(7, len(files))) as ex:
        for f, found in ex.map(_scan, files):
            assert found is not None, f"{f} did not compile"
            bad += [f"{os.path.basename(f)}: {k[:100]}: {have} of {want} wait states before {text}" for k, hits in found.items() for have, want, text in hits]
    assert not bad, "\n".join(bad[:20])
