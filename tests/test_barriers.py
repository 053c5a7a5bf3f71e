"""What the kernels' machine code promises at barriers: a wave that comes to one has waited for
its writes to LDS, which others read behind it. (The compiler's own wait was missing once, at a
barrier that began a loop whose end wrote to LDS: now and then a wave went on from an older
value, which tests of results do not reliably show.)

The check walks each kernel's blocks along their branches with the age of the newest LDS write
under way: the operations of the same counter issued behind it. s_waitcnt lgkmcnt(n) ends it
where it leaves no more than those under way."""
import bisect
import concurrent.futures
import os
import re
import struct
import subprocess

import pytest

from janis_amd import build

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
WRITES = re.compile(r"ds_(write|store|add|sub|rsub|max|min|or|and|xor|inc|dec|cmpst|wrxchg|mskor|append|consume)")
LINE = re.compile(r"^\t(s_barrier|s_waitcnt|s_cbranch\w+|s_branch|s_endpgm|s_setpc\w+|s_load\w+|s_buffer_load\w+|s_memtime|s_memrealtime|ds_\w+)"
                  r"\b(.*?)// ([0-9A-F]+):(.*)$")
HEAD = re.compile(r"^([0-9a-f]{16}) <(.+)>:$")
TARGET = re.compile(r"<[^>+]+(?:\+0x([0-9a-f]+))?>\s*$")


def code_objects(path):
    """The gfx950 code objects in a library's bundles."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, n = struct.unpack_from("<QQQ", data, p)
            if size and data[p + 24:p + 24 + n].endswith(b"gfx950"):
                yield data[at + offset:at + offset + size]
            p += 24 + n
        at = data.find(MAGIC, at + 1)


def functions(text):
    """(name, [(address, operation, operands, branch target or None)]) of a disassembly, of
    the operations that matter here."""
    name, start, ins = None, 0, []
    for line in text.splitlines():
        m = LINE.match(line)
        if m:
            addr, op = int(m.group(3), 16), m.group(1)
            t = TARGET.search(m.group(4)) if "branch" in op else None
            ins.append((addr, op, m.group(2), start + int(t.group(1) or "0", 16) if t else None))
        elif not line.startswith("\t"):
            m = HEAD.match(line)
            if m:
                if name:
                    yield name, ins
                name, start, ins = m.group(2), int(m.group(1), 16), []
    if name:
        yield name, ins


def behind(block, age, early):
    """The age of the pending write behind a block (-1: none); barriers that meet one are added to `early`."""
    for addr, op, args, _ in block:
        if op == "s_barrier":
            if age >= 0:
                early.add(addr)
        elif op == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", args)
            if age >= 0 and (int(m.group(1)) <= age if m else "cnt" not in args):
                age = -1
        elif WRITES.match(op):
            age = 0
        elif op.startswith(("ds_", "s_load", "s_buffer", "s_mem")):
            age += age >= 0
    return age


def early_barriers(ins):
    """Addresses of the barriers that a wave may come to with an LDS write under way."""
    addrs = [i[0] for i in ins]
    ends = lambda i: i[1] in ("s_branch", "s_endpgm") or i[1].startswith("s_setpc")  # noqa: E731
    first = {0} | {bisect.bisect_left(addrs, i[3]) for i in ins if i[3] is not None} | {n + 1 for n, i in enumerate(ins) if i[3] is not None or ends(i)}
    first = sorted(n for n in first if n < len(ins))
    number = {n: b for b, n in enumerate(first)}
    blocks = [ins[a:b] for a, b in zip(first, first[1:] + [len(ins)])]
    ages, todo, early = {0: -1}, [0] if blocks else [], set()
    while todo:
        b = todo.pop()
        last, out = blocks[b][-1], behind(blocks[b], ages[b], set())
        to = [number.get(bisect.bisect_left(addrs, last[3]))] if last[3] is not None else []
        for x in to + ([] if ends(last) else [b + 1]):
            if x is None or x >= len(blocks):
                continue
            had = ages.get(x)
            if had is None or (out >= 0 and (had < 0 or out < had)):
                ages[x] = out
                todo.append(x)
    for b, age in ages.items():
        behind(blocks[b], age, early)
    return sorted(early)


TEXT = """0000000000001000 <kernel>:
\tds_write_b32 v0, v1                                        // 000000001000: 00000000
\t{first}                                                    // 000000001008: 00000000
\ts_barrier                                                  // 00000000100C: 00000000
\tds_read_b32 v2, v0                                         // 000000001010: 00000000
\ts_waitcnt lgkmcnt(0)                                       // 000000001018: 00000000
\ts_cbranch_scc1 4                                           // 00000000101C: 00000000 <kernel+0x30>
\tds_write_b32 v0, v2                                        // 000000001020: 00000000
\tds_read_b32 v3, v4                                         // 000000001028: 00000000
\t{second}                                                   // 000000001030: 00000000
\ts_branch 65526                                             // 000000001034: 00000000 <kernel+0xc>
\ts_endpgm                                                   // 000000001038: 00000000
"""


@pytest.mark.parametrize("first,second,early", [
    ("s_waitcnt lgkmcnt(0)", "s_waitcnt lgkmcnt(0)", False), ("s_waitcnt lgkmcnt(0)", "s_waitcnt lgkmcnt(1)", False),
    ("s_waitcnt lgkmcnt(0)", "s_waitcnt lgkmcnt(2)", True), ("s_waitcnt lgkmcnt(0)", "s_waitcnt vmcnt(0)", True),
    ("s_nop 0", "s_waitcnt lgkmcnt(0)", True), ("s_waitcnt vmcnt(0) lgkmcnt(0)", "s_nop 0", True)])
def test_the_check_itself(first, second, early):
    """A write before the first barrier, and one at a loop's end whose beginning is that barrier."""
    (name, ins), = functions(TEXT.format(first=first, second=second))
    assert name == "kernel" and early_barriers(ins) == ([0x100c] if early else [])


def test_no_barrier_meets_an_lds_write_under_way(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    if not os.path.exists(build.LIB):
        build.build()
    files = []
    for n, code in enumerate(code_objects(build.LIB)):
        files.append(tmp_path / f"{n}.co")
        files[-1].write_bytes(code)
    assert len(files) >= len(build.SOURCES) - 1  # (a file may hold no kernel)

    def of(path):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True, check=True).stdout
        return [(name, len(ins), early_barriers(ins)) for name, ins in functions(text)]

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        seen = [f for part in pool.map(of, files) for f in part]
    assert any("tree_attn_kernel" in name and n > 1000 for name, n, _ in seen)
    assert [(name, [hex(b) for b in early]) for name, _, early in seen if early] == []
