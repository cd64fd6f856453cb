"""Looks for vector instructions that run with lanes switched off which they are meant for, in gfx950 assembly.

Where a condition of single lanes ends together with one around it, the compiler leaves out the inner one's end: the
lanes switched off by ``s_and_b64 exec, exec, ...`` (which keeps no copy of the mask) come back with the outer one's. Nothing
may stand between. The register allocator, which comes later, can put copies there when a kernel is short of registers;
the lanes that are off keep what their registers held, and results are wrong without an error.
"""
import re

from asm_waits import parse

_OFF = re.compile(r"s_and_b64 exec, exec, ")


def lost_lanes(lines):
    """(function, the instruction that switches lanes off, the vector instruction before they are back)"""
    found = []
    for name, (code, labels) in parse(lines).items():
        for i, off in enumerate(code):
            if not _OFF.match(off.text):
                continue
            to = next((c.text.split()[1] for c in code[i + 1:i + 4] if c.op == "s_cbranch_execz"), None)
            for c in code[labels[to]:] if to in labels else ():
                if re.match(r"s_\w+ exec,", c.text) or "saveexec" in c.op or c.op.startswith(("s_cbranch", "s_branch", "s_endpgm", "s_setpc")):
                    break
                if c.op.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
                    found.append((name, off, c))
    return found


def check(path):
    """Raises for the first such instruction in the assembly file."""
    with open(path) as f:
        found = lost_lanes(f)
    if found:
        name, off, then = found[0]
        raise RuntimeError("%s:%d: `%s` runs before the lanes that line %d switches off are back; %d such instructions"
                           % (path, then.line, then.text, off.line, len(found)))
