"""Wait states in the assembly that hipcc makes of our own sources for gfx950.

A scalar register that a vector instruction wrote (v_readlane, v_readfirstlane, a
comparison) may be read by a memory instruction as its base, its descriptor or
its offset five wait states later at the earliest.  The hardware does not hold
such an instruction back; the compiler puts the missing states in, but it does not
look into inline assembly."""
from __future__ import annotations

import re

STATES = 5  # between the vector instruction and the memory instruction
MEMORY = ("global", "buffer", "flat", "scratch")
SECOND_IS_SCALAR = re.compile(r"v_(add|sub|subrev|addc|subb|subbrev)_co|v_div_scale|v_mad_[iu]64")


def scalars(operand):
    """The scalar registers of an operand."""
    words = operand.split()
    name = words[0] if words else ""
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", name)
    if m:
        return [f"s{i}" for i in range(int(m[1]), int(m[2]) + 1)]
    return ["vcc_lo", "vcc_hi"] if name == "vcc" else [name] if re.fullmatch(r"s\d+|vcc_lo|vcc_hi", name) else []


def functions(text):
    """{name: [(opcode, operands) or ("label", name)]}"""
    out, cur = {}, None
    for line in text.splitlines():
        line = line.split(";", 1)[0].rstrip()
        if not line:
            continue
        m = re.match(r"(\S+):$", line)
        if m and m[1].startswith(".LBB"):
            if cur is not None:
                cur.append(("label", m[1]))
        elif m and m[1].startswith(".Lfunc_end"):
            cur = None
        elif m and not m[1].startswith("."):
            cur = out.setdefault(m[1], [])
        elif cur is not None and not line.strip().startswith("."):
            op, _, rest = line.strip().partition("\t") if "\t" in line.strip() else line.strip().partition(" ")
            cur.append((op, [x.strip() for x in re.split(r",(?![^\[]*\])", rest)] if rest.strip() else []))
    return out


def early(code):
    """(index, states) of every memory instruction of a function that may read a scalar
    register too early, over all ways through it: an instruction counts one state, s_nop n n + 1."""
    labels = {x[1]: i for i, x in enumerate(code) if x[0] == "label"}
    entry, work, bad = {0: {}}, [0], {}

    def meet(at, state):  # the fewest states of any way there
        old = entry.get(at)
        if old is None:
            entry[at] = dict(state)
            work.append(at)
            return
        less = {r: n for r, n in state.items() if n < old.get(r, STATES)}
        if less:
            old.update(less)
            work.append(at)

    while work:
        i = start = work.pop()
        state = dict(entry[start])
        while i < len(code):
            op, args = code[i]
            if op == "label":
                if i != start:
                    meet(i, state)
                    break
                i += 1
                continue
            if op.split("_")[0] in MEMORY:
                since = [state[r] for a in args for r in scalars(a) if r in state]
                if since:
                    bad[i] = min(since + [bad.get(i, STATES)])
            n = int(args[0], 0) + 1 if op == "s_nop" else 1
            state = {r: s + n for r, s in state.items() if s + n < STATES}
            if op.startswith("v_") and args:
                for r in scalars(args[0]) or (scalars(args[1]) if SECOND_IS_SCALAR.match(op) else []):
                    state[r] = 0
            elif op.startswith("s_") and args:
                for r in scalars(args[0]):
                    state.pop(r, None)
            if op.startswith("s_cbranch"):
                meet(labels[args[0]], state)
            if op == "s_branch":
                meet(labels[args[0]], state)
                break
            if op in ("s_endpgm", "s_setpc_b64"):
                break
            i += 1
    return sorted(bad.items())
