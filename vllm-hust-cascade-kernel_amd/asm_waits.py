"""Looks for missing waits around hand-written instructions in gfx950 assembly.

The hardware does not hold an instruction back until everything it needs is there: for some
pairs the program has to keep a number of wait states (other instructions, or ``s_nop``) between
the two. The compiler inserts them for its own instructions, but does not see those inside
inline assembly (``#ASMSTART`` .. ``#ASMEND``). ``missing_waits`` walks back from each of
those over all paths and names the pairs that are too close. The distances are the ones that
the compiler itself keeps between such instructions for gfx950:

* a matrix product's result, before anything but a product's own sum reads or overwrites it:
  8 (16x16x16, 16x16x32) and 12 (32x32x16),
* a vector instruction's result, before a matrix product reads it: 2,
* a scalar register written by a vector instruction, before a memory instruction reads it: 5,
* M0, before a load to LDS reads it: 1.
"""
import collections
import re

PRODUCT_WAITS = {"16x16x16": 8, "16x16x32": 8, "32x32x16": 12}
VECTOR_TO_PRODUCT, VECTOR_TO_MEMORY, M0_TO_LDS_LOAD = 2, 5, 1
FURTHEST = max(*PRODUCT_WAITS.values(), VECTOR_TO_PRODUCT, VECTOR_TO_MEMORY, M0_TO_LDS_LOAD)

Instr = collections.namedtuple("Instr", "line text op inline writes reads product states")
_REG = re.compile(r"\b([vas])(?:(\d+)\b|\[(\d+):(\d+)\])|\b(m0)\b")


def _regs(text):
    out = set()
    for kind, one, lo, hi, m0 in _REG.findall(text):
        if m0:
            out.add("m0")
        else:
            out.update("%s%d" % (kind, i) for i in range(int(one or lo), int(one or hi) + 1))
    return out


def _is_memory(op):
    return op.startswith(("buffer_", "global_", "flat_", "scratch_"))


def _decode(line, text, inline):
    op, _, rest = text.partition(" ")
    ops = [o for o in re.split(r",\s*(?![^\[]*\])", rest.strip()) if o]
    to_lds = re.search(r"\blds\b", rest) is not None or "_load_lds_" in op
    stores = "store" in op or "write" in op and op.startswith("ds_") or to_lds or op.startswith(("s_cmp", "s_barrier"))
    count = 0 if stores else 2 if "_swap" in op else 1
    writes = set().union(*(_regs(o) for o in ops[:count])) if ops else set()
    reads = set().union(*(_regs(o) for o in (ops if "_swap" in op else ops[count:]))) if ops else set()
    if to_lds:
        reads.add("m0")
    product = None
    if "_mfma_" in op:
        product = next((k for k in PRODUCT_WAITS if k in op), None)
        if product is None:
            raise ValueError("line %d: no known distance for %s" % (line, text))
    states = int(ops[0], 0) + 1 if op == "s_nop" else 1
    return Instr(line, text, op, inline, writes, reads, product, states)


def parse(lines):
    """{function: (instructions, {label: index of the instruction after it})}"""
    funcs, code, labels, inline = {}, None, None, False
    for n, raw in enumerate(lines, 1):
        if "#ASMSTART" in raw or "#ASMEND" in raw:
            inline = "#ASMSTART" in raw
            continue
        text = raw.split(";")[0].strip()
        label = re.match(r"([.\w$]+):$", text)
        if label:
            if label.group(1).startswith(".L"):
                if code is not None:
                    labels[label.group(1)] = len(code)
            else:
                code, labels = [], {}
                funcs[label.group(1)] = (code, labels)
            continue
        if not text or text.startswith(".") or code is None:
            continue
        code.append(_decode(n, text, inline))
    return {k: v for k, v in funcs.items() if v[0]}


def _before(code, labels):
    """For each instruction the ones that can come right before it."""
    prev = [[] for _ in code]
    for i, ins in enumerate(code):
        if ins.op.startswith(("s_branch", "s_cbranch")):
            to = labels.get(ins.text.split()[-1])
            if to is not None and to < len(code):
                prev[to].append(i)
        if ins.op not in ("s_branch", "s_endpgm", "s_setpc_b64") and i + 1 < len(code):
            prev[i + 1].append(i)
    return prev


def _waits(first, then, reg):
    """Wait states that `then`, hand-written, has to keep from `first`, which writes reg."""
    if first.product:
        if then.product and reg in then.writes:  # its sum goes on where it is
            return 0 if first.writes == then.writes else PRODUCT_WAITS[first.product]
        return PRODUCT_WAITS[first.product]
    if reg == "m0":
        return M0_TO_LDS_LOAD
    if first.op.startswith("v_") and reg in then.reads:
        if reg[0] == "s":
            return VECTOR_TO_MEMORY if _is_memory(then.op) else 0
        return VECTOR_TO_PRODUCT if then.product else 0
    return 0


def missing_waits(lines):
    """(function, the earlier instruction, the hand-written one, register, states kept, states needed)"""
    found = []
    for name, (code, labels) in parse(lines).items():
        prev = _before(code, labels)
        for i, then in enumerate(code):
            if not then.inline:
                continue
            open_regs = frozenset(then.reads | then.writes)
            seen, todo = set(), [(p, 0, open_regs) for p in prev[i]]
            while todo:
                at, kept, regs = todo.pop()
                if kept >= FURTHEST or not regs or (at, kept, regs) in seen:
                    continue
                seen.add((at, kept, regs))
                first = code[at]
                for reg in regs & first.writes:
                    need = _waits(first, then, reg)
                    if kept < need:
                        found.append((name, first, then, reg, kept, need))
                todo += [(p, kept + first.states, regs - first.writes) for p in prev[at]]
    return found


def check(path):
    """Raises for the first pair that is too close in the assembly file."""
    with open(path) as f:
        found = missing_waits(f)
    if found:
        name, first, then, reg, kept, need = found[0]
        raise RuntimeError("%s:%d: %d wait states, not %d, between `%s` (line %d) and `%s` for %s; %d such pairs"
                           % (path, then.line, kept, need, first.text, first.line, then.text, reg, len(found)))
