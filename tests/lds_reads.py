"""Registers that an LDS read is still to fill, in the machine code of this
library's own kernels.

Some kernels read LDS by inline assembly and wait by counts of their own
(s_waitcnt lgkmcnt); to the compiler such a read is done where it stands.  It
must therefore be seen, in what was built, that nothing reads or writes a
register between its read and the wait that covers it.  LDS operations of a
wave complete in order, so at lgkmcnt(n) all but the n last of them are done.
"""
import os
import re
import struct
import subprocess
import tempfile

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")


def code_objects(library):
    """The gfx950 code objects in a library or object file."""
    data = open(library, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24: p + 24 + length].decode()
            p += 24 + length
            if "gfx950" in name and size:
                yield data[at + offset: at + offset + size]
        at = data.find(MAGIC, at + len(MAGIC))


def kernels(code_object):
    """{name: [(address, text, branch target or None)]} of a code object."""
    with tempfile.NamedTemporaryFile(suffix=".co") as f:
        f.write(code_object)
        f.flush()
        text = subprocess.run([OBJDUMP, "-d", f.name], check=True, capture_output=True, text=True).stdout
    out, start, code = {}, 0, None
    for line in text.splitlines():
        m = re.match(r"([0-9a-f]+) <(.+)>:$", line)
        if m:
            start, code = int(m.group(1), 16), out.setdefault(m.group(2), [])
            continue
        m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):", line)
        if not m or code is None:
            continue
        to = None
        if m.group(1).startswith(("s_branch", "s_cbranch")):
            t = re.search(r"<[^>]*?(?:\+0x([0-9a-fA-F]+))?>\s*$", line)
            to = start + int(t.group(1) or "0", 16)
        code.append((int(m.group(2), 16), m.group(1), to))
    return out


REGISTERS = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(text):
    out = set()
    for kind, first, last, one in REGISTERS.findall(text):
        out |= {(kind, i) for i in (range(int(first), int(last) + 1) if first else (int(one),))}
    return frozenset(out)


NONE = frozenset()


def compiled(code):
    """Instructions as (what, argument, registers): a wait for all but `argument` LDS operations, an LDS operation that fills
    `argument` and reads the registers, or anything else that touches them."""
    out = []
    for _, text, _ in code:
        op = text.split(None, 1)[0]
        if op == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", text)
            out.append(("wait", int(m.group(1)) if m else None, NONE))
        elif op.startswith("ds_"):
            operands = text.split(None, 1)[1] if " " in text else ""
            if re.match(r"ds_(read|load|bpermute|permute|swizzle)|.*_rtn", op):
                fills, _, rest = operands.partition(",")
                out.append(("lds", registers(fills), registers(rest)))
            else:
                out.append(("lds", NONE, registers(operands)))
        else:
            out.append(("other", None, registers(text)))
    return out


def touched_in_flight(code):
    """[(address, text)] of the instructions that on some path touch a register which an LDS read is still to fill.  What is
    known before a block: for each register in flight the least number of LDS operations that follow its read on a way there."""
    steps, index = compiled(code), {a: i for i, (a, _, _) in enumerate(code)}
    starts = {index[to] for _, _, to in code if to is not None}
    bad, before, todo = set(), {0: {}}, [0]

    def goes_on(i, flight):
        if i >= len(steps):
            return
        known = before.get(i)
        merged = dict(flight) if known is None else {r: min(known.get(r, 99), flight.get(r, 99)) for r in known.keys() | flight.keys()}
        if merged != known:
            before[i] = merged
            todo.append(i)

    while todo:
        i = todo.pop()
        flight = dict(before[i])
        while True:
            what, arg, regs = steps[i]
            if what == "wait":
                if arg is not None:
                    flight = {r: n for r, n in flight.items() if n < arg}
            else:
                if not regs.isdisjoint(flight):
                    bad.add(i)
                if what == "lds":
                    flight = {r: n + 1 for r, n in flight.items()}
                    flight.update(dict.fromkeys(arg, 0))  # (a read into registers that an earlier one fills comes after it)
            _, text, to = code[i]
            i += 1
            if to is not None:
                goes_on(index[to], flight)
            if text.startswith(("s_branch", "s_endpgm", "s_setpc")):
                break
            if to is not None or i in starts or i >= len(steps):
                goes_on(i, flight)
                break
    return [code[i][:2] for i in sorted(bad)]
