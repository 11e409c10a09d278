"""ISA check: wait states that the hardware needs between two instructions and that hipcc does not put there, because one of the two stands in inline assembly (its
hazard recognizer does not look into asm blocks).  For every kernel, along every path of its control-flow graph:

  * a vector-ALU instruction writes an SGPR (v_readfirstlane, v_readlane - also the reload of a spilled SGPR -, a comparison, a carry) and a vector-memory
    instruction reads it: 5 wait states.  Too early it reads the old value: an LDS-DMA piece then comes from another offset or another descriptor's memory.
  * a vector-ALU instruction writes an SGPR and another one reads it: 2
  * a matrix instruction writes a register and a vector-ALU, LDS or memory instruction reads it: passes + 4 (32x32x16 bf16: 12)
  * a vector-ALU instruction writes a register and a v_permlane*_swap, a DPP or a matrix instruction reads it: 2; v_readlane / v_readfirstlane: 1
  * a load writes a register, which is read or written before an `s_waitcnt vmcnt` covers it (-1 of 0 wait states in the report)
  * a load to LDS in an asm block takes the M0 of an earlier block, and hipcc has written M0 since (-2 of 0)

Pairs of which neither instruction stands in an asm block are hipcc's own and left out.  An instruction is one wait state, `s_nop n` is n + 1.  Usage: python tools/scan_asm_hazards.py [file.hip ...] (default: all of csrc)."""
import functools, glob, importlib.util, os, re, sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_spec = importlib.util.spec_from_file_location("scan_barrier_waits", os.path.join(ROOT, "tools", "scan_barrier_waits.py"))
_isa = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_isa)

CAP = 24   # no hazard here is longer
_REG = re.compile(r"(?<![\w.])([sva])(?:\[(\d+):(\d+)\]|(\d+)\b)|\b(vcc)(_lo|_hi)?\b|\b(m0)\b")


@functools.lru_cache(maxsize=None)
def _regs(text):
    out = []
    for m in _REG.finditer(text):
        if m.group(7):
            out.append(("s", 1002))
        elif m.group(5):
            out += [("s", 1000), ("s", 1001)] if not m.group(6) else [("s", 1000 if m.group(6) == "_lo" else 1001)]
        elif m.group(4) is not None:
            out.append((m.group(1), int(m.group(4))))
        else:
            out += [(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)]
    return out


def _passes(op):
    """Wait states between a matrix instruction and a vector, LDS or memory read of its result."""
    m = re.match(r"v_s?mfmac?_\w+?_(\d+)x(\d+)x(\d+)_?(\w*)", op)
    rows, kind = int(m.group(1)), m.group(4)
    if kind in ("f32", "f64"):   # (not on the XDL path: passes + 2)
        return 18 if rows == 32 else 10
    return 12 if rows == 32 else 8 if rows == 16 else 6


@functools.lru_cache(maxsize=None)
def _decode(text):
    """(kind, defs, uses, wait states) of an instruction; kind: valu, mfma, vmem, lds, salu, wait, other."""
    op, _, rest = text.partition(" ")
    ops = [o.strip() for o in re.split(r",(?![^\[]*\])", rest)] if rest else []
    if op == "s_nop":
        return "salu", [], [], int(ops[0], 0) + 1
    if "mfma" in op or "smfmac" in op:
        return "mfma", _regs(ops[0]), _regs(" ".join(ops[1:])), 1
    if op.startswith("v_"):
        if op.startswith(("v_permlane16_swap", "v_permlane32_swap", "v_swap")):
            return "valu", _regs(rest), _regs(rest), 1
        n = 2 if re.match(r"v_(add|sub|subrev|addc|subb|subbrev)_co_|v_(addc|subb|subbrev)_co|v_div_scale|v_mad_[ui]64", op) else 1
        uses = _regs(" ".join(ops[n:]))
        if op.startswith("v_cndmask") and len(ops) == 3 or op.startswith("v_div_fmas"):
            uses = [*uses, ("s", 1000), ("s", 1001)]
        if op.startswith(("v_fmac", "v_mac", "v_dot2c", "v_writelane")):
            uses = [*uses, *_regs(ops[0])]
        return "valu", _regs(" ".join(ops[:n])), uses, 1
    if op.startswith(("buffer_", "global_", "flat_", "scratch_")):
        return "vmem", [] if re.search("store|atomic|lds", text) else _regs(ops[0]), _regs(rest), 1
    if op.startswith("ds_"):
        return "lds", _regs(ops[0]) if re.search(r"read|load|permute|swizzle|rtn", op) else [], _regs(rest), 1
    if op == "s_waitcnt":
        return "wait", [], [], 1
    if op.startswith("s_"):
        dst = [] if op.startswith(("s_cmp", "s_waitcnt", "s_barrier", "s_cbranch", "s_branch", "s_bitcmp", "s_setprio", "s_sleep", "s_endpgm", "s_store")) or not ops else _regs(ops[0])
        return "salu", dst, [], 1
    return "other", [], [], 1


@functools.lru_cache(maxsize=None)
def _needs(kind, text, bank):
    """[(class of the earlier write, wait states)] that a read of a register of this bank (s, v, a) by this instruction asks for."""
    op = text.split(" ", 1)[0]
    need = []
    if bank == "s":
        if kind == "vmem":
            need.append(("valu", 5))
        elif kind == "valu":
            need.append(("valu", 2))
        return need
    if kind in ("valu", "vmem", "lds"):
        need.append(("mfma", None))
    if kind == "mfma":
        need.append(("valu", 2))
    if kind == "valu":
        if op.startswith("v_permlane"):
            need.append(("valu", 2))
        elif re.search(r"quad_perm|row_|wave_|dpp", text):
            need.append(("valu", 2))
        elif op.startswith(("v_readlane", "v_readfirstlane")):
            need.append(("valu", 1))
    return need


def _blocks(ins):
    blocks, cur, label_of = [], [], {}
    for t in ins:
        if t.endswith(":"):
            if cur:
                blocks.append(cur)
            cur = [t]
            continue
        cur.append(t)
        if t.startswith(("s_branch", "s_cbranch", "s_endpgm", "s_setpc")):
            blocks.append(cur)
            cur = []
    if cur:
        blocks.append(cur)
    for i, b in enumerate(blocks):
        if b[0].endswith(":"):
            label_of[b[0][:-1]] = i
    succ = []
    for i, b in enumerate(blocks):
        last, to = b[-1], []
        if last.startswith(("s_branch", "s_cbranch")) and last.split()[-1] in label_of:
            to.append(label_of[last.split()[-1]])
        if not last.startswith(("s_branch", "s_endpgm", "s_setpc")) and i + 1 < len(blocks):
            to.append(i + 1)
        succ.append(to)
    return blocks, succ


ASM = " @asm"
M0 = ("m0", ("s", 1002))   # written by hipcc behind the last write of an asm block


def scan_function(ins):
    """Hits (wait states there are, needed, the reading instruction) of one function, whose instructions from asm blocks end in ASM.
    State: (class, register) -> (age of the write, states that a matrix result needs, written in an asm block); ("load", register): age in younger memory operations."""
    blocks, succ = _blocks(ins)
    decoded = [[(t, t.endswith(ASM), *_decode(t.removesuffix(ASM))) for t in b if not t.endswith(":")] for b in blocks]
    state_in = [None] * len(blocks)
    state_in[0] = {}
    hits, work = {}, [0]
    while work:
        i = work.pop()
        clock, memory = 0, 0   # wait states, memory operations since the block's start
        s = {k: (-age, n, a) for k, (age, n, a) in state_in[i].items()}
        for j, (text, in_asm, kind, defs, uses, wait) in enumerate(decoded[i]):
            for reg in uses:
                for cls, need in _needs(kind, text, reg[0]):
                    at = s.get((cls, reg))
                    if at is not None and (in_asm or at[2]):
                        want = at[1] if need is None else need
                        if clock - at[0] < want:
                            hits[(i, j)] = (clock - at[0], want, text)
            if in_asm and kind == "vmem" and "lds" in text and M0 in s:
                hits[(i, j)] = (-2, 0, text)
            if M0[1] in defs:
                s.pop(M0, None)
                if not in_asm:
                    s[M0] = (0, 0, False)
            for reg in (*uses, *defs):
                if ("load", reg) in s and (in_asm or s[("load", reg)][2]):
                    hits[(i, j)] = (-1, 0, text)
            clock += wait
            if kind == "wait":
                s = {k: x for k, x in s.items() if k[0] != "load" or memory - x[0] < wait_count(text)}
            for reg in defs:
                for cls in ("valu", "mfma", "load"):
                    s.pop((cls, reg), None)
                if kind == "valu":
                    s[("valu", reg)] = (clock, 0, in_asm)
                elif kind == "mfma":
                    s[("mfma", reg)] = (clock, _passes(text.split(" ", 1)[0]), in_asm)
            if kind == "vmem":
                memory += 1
                for reg in defs:
                    s[("load", reg)] = (memory, 0, in_asm)
        out = {}
        for k, (at, n, a) in s.items():
            if k[0] == "load":
                out[k] = (min(memory - at, 64), n, a)
            elif k == M0:
                out[k] = (0, n, a)
            elif clock - at < CAP:
                out[k] = (clock - at, n, a)
        for j in succ[i]:
            old = state_in[j]
            new = dict(out) if old is None else dict(old)
            if old is not None:
                for k, x in out.items():
                    if k not in new or x[0] < new[k][0] or x[2] and not new[k][2]:
                        new[k] = (min(x[0], new.get(k, x)[0]), max(x[1], new.get(k, x)[1]), x[2] or new.get(k, x)[2])
            if new != old:
                state_in[j] = new
                work.append(j)
    return list(hits.values())


def wait_count(text):
    """How many memory operations may still be in flight behind an s_waitcnt (64: it does not look at them)."""
    m = re.search(r"vmcnt\((\d+)\)", text)
    return int(m.group(1)) if m else 0 if re.match(r"s_waitcnt\s+(0x0|0)\b", text) else 64


def marked(text):
    """The assembly with the instructions of asm blocks marked."""
    out, inside = [], False
    for line in text.split("\n"):
        if "#ASMSTART" in line or "#ASMEND" in line:
            inside = "#ASMSTART" in line
        elif inside and line.strip() and not line.strip().startswith(";"):
            line = line.split(";")[0].rstrip() + ASM
        out.append(line)
    return out


def scan_lines(lines):
    return {name: h for name, ins in _isa._kernels(lines).items() if ins and (h := scan_function(ins))}


def scan_text(text):
    return scan_lines(marked(text))


def scan(path):
    text = _isa.isa_of(path)
    return None if text is None else scan_text(text)


if __name__ == "__main__":
    worst = 0
    for f in sys.argv[1:] or sorted(glob.glob(os.path.join(ROOT, "satflow_amd", "csrc", "*.hip"))):
        found = scan_text(open(f).read()) if f.endswith(".s") else scan(f)
        if found is None:
            print(os.path.basename(f), "did not compile")
            worst += 1
            continue
        worst += len(found)
        print(f"{os.path.basename(f):36s} {sum(map(len, found.values()))} reads too early in {len(found)} kernels")
        for name, hits in found.items():
            for have, want, text in hits[:4]:
                print(f"       {name[:110]}: {have} of {want} wait states before  {text}")
    sys.exit(1 if worst else 0)
