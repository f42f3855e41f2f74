"""Reads gfx950 listings (llvm-objdump -d) for one hazard: a vector-memory instruction may read an SGPR that a vector
instruction wrote (readfirstlane, readlane, a comparison, a carry) only five wait states later.  The hardware does not check it; the
compiler does for its own instructions, not for the loads inside inline assembly."""
import re

STATES = 5
MEMORY = ("buffer_", "global_", "scratch_", "flat_")
LINE = re.compile(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):")
REGISTER = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc|vcc_lo|vcc_hi)\b")
VCC = {"vcc": {106, 107}, "vcc_lo": {106}, "vcc_hi": {107}}


def registers(text):
    found = set()
    for m in REGISTER.finditer(text):
        found |= set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])} if m[3] else VCC[m[4]]
    return found


def written(op, operands):
    """SGPRs that an instruction writes, by its class."""
    parts = operands.split(", ")
    if op.startswith("s_"):
        return set() if op.startswith(("s_cmp", "s_bitcmp", "s_waitcnt", "s_branch", "s_cbranch")) else registers(parts[0])
    if op.startswith(("v_readlane", "v_readfirstlane", "v_cmp")):
        return registers(parts[0])
    if op.startswith("v_") and len(parts) > 1 and ("_co_" in op or "div_scale" in op or op.startswith(("v_mad_u64", "v_mad_i64"))):
        return registers(parts[1])
    return set()


def functions(listing):
    """[(name, [(address, op, operands)])] of a disassembly."""
    out = []
    for line in listing.splitlines():
        head = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if head:
            out.append((head[1], []))
            continue
        m = LINE.match(line)
        if m and out:
            out[-1][1].append((int(m[3], 16), m[1], m[2]))
    return out


def hazards(listing):
    """[(function, the memory instruction, the write before it, wait states between)]."""
    found = []
    for name, code in functions(listing):
        place = {address: i for i, (address, _, _) in enumerate(code)}
        into = {}
        for i, (address, op, operands) in enumerate(code):
            if op.startswith(("s_branch", "s_cbranch")):
                step = int(operands.split()[0])
                target = place.get(address + 4 + 4 * (step - 65536 if step >= 32768 else step))
                if target is not None:
                    into.setdefault(target, []).append(i)
        for i, (_, op, operands) in enumerate(code):
            reads = registers(operands) if op.startswith(MEMORY) else set()
            if not reads:
                continue
            todo, seen = [(i, reads, 0)], set()
            while todo:
                at, wanted, states = todo.pop()
                before = list(into.get(at, []))
                if at and not code[at - 1][1].startswith(("s_branch", "s_endpgm", "s_setpc")):
                    before.append(at - 1)
                for b in before:
                    _, bop, boperands = code[b]
                    writes = written(bop, boperands) & wanted
                    if writes and bop.startswith("v_"):
                        found.append((name, f"{op} {operands}", f"{bop} {boperands}", states))
                        continue
                    after = states + (int(boperands.split()[0], 0) + 1 if bop == "s_nop" else 1)
                    left = wanted - writes
                    if left and after < STATES and (b, after) not in seen:
                        seen.add((b, after))
                        todo.append((b, left, after))
    return found
