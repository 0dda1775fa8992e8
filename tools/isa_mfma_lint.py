#!/usr/bin/env python3
"""Lint for the gfx950 code of a built object or library: is a matrix instruction's result left alone for long enough?

The hardware does not interlock a vector, memory or LDS instruction that touches the registers a matrix instruction (v_mfma) is still writing: the
compiler has to put the wait states between them, 8 behind one of 4 passes (16x16x64 of 8 bits), 12 behind one of 8 (32x32x32 of 8 bits).  It was
seen to count too few where a branch lies between the two, so the count is done again here over both sides of every branch.  A matrix
instruction that takes the result as its accumulator may follow at once.

usage: isa_mfma_lint.py FILE [--kernel SUBSTR]      (an object, shared library or code object built here; needs llvm-objdump)
Prints the smallest distance of each kernel; exit status 1 where one is too short."""
import glob
import os
import re
import subprocess
import sys
import tempfile

OBJDUMP = os.environ.get('LLVM_OBJDUMP', '/opt/rocm/llvm/bin/llvm-objdump')
NEEDED = {'16x16x64': 8, '32x32x32': 12, '32x32x16': 12, '16x16x32': 8}      # wait states, by the shape in the name
SYMBOL = re.compile(r'^([0-9a-f]+) <(\S+)>:')
LINE = re.compile(r'^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):')
TARGET = re.compile(r'<(\S+?)(?:\+0x([0-9a-f]+))?>\s*$')
REGS = re.compile(r'\b([av])(?:\[(\d+):(\d+)\]|(\d+))')


def regs(text):
    out = set()
    for kind, lo, hi, one in REGS.findall(text):
        out.update((kind, i) for i in (range(int(lo), int(hi) + 1) if lo else (int(one),)))
    return out


def operands(text):
    return [t.strip() for t in re.split(r',(?![^\[]*\])', text)]


def parse(listing, want=''):
    """{kernel: [(op, operands, index of the branch target or None)]} of llvm-objdump -d's output, for the kernels with `want` in their names."""
    kernels, starts, name = {}, {}, None
    for line in listing.splitlines():
        m = SYMBOL.match(line)
        if m:
            name = m.group(2) if want in m.group(2) else None
            if name is None:
                continue
            starts[name] = int(m.group(1), 16)
            kernels[name] = []
            continue
        m = LINE.match(line) if name else None
        if m:
            op, args, addr = m.group(1), m.group(2), int(m.group(3), 16)
            t = TARGET.search(line) if op.startswith(('s_cbranch', 's_branch')) else None
            kernels[name].append((op, args, addr, (t.group(1), int(t.group(2) or '0', 16)) if t else None))
    out = {}
    for name, code in kernels.items():
        at = {addr: i for i, (_, _, addr, _) in enumerate(code)}
        out[name] = [(op, args, at.get(starts.get(t[0], 0) + t[1]) if t else None) for op, args, _, t in code]
    return out


def shape(op):
    m = re.search(r'_(\d+x\d+x\d+)_', op + '_')
    return m.group(1) if m else ''


def lint(code):
    """[(distance, needed, index of the matrix instruction, index of what touches its result)], one for each matrix instruction that is followed too closely; and the smallest
    distance found."""
    bad, least = [], None
    for p, (op, args, _) in enumerate(code):
        if not op.startswith('v_mfma') or shape(op) not in NEEDED:
            continue
        need, result = NEEDED[shape(op)], regs(operands(args)[0])
        seen, stack, found = {}, [(p + 1, 0)], None
        while stack:
            q, d = stack.pop()
            if q >= len(code) or d >= need + 8 or seen.get(q, 1 << 30) <= d:
                continue
            seen[q] = d
            o, a, target = code[q]
            if o.startswith('v_mfma'):
                to, fa, fb, fc = (regs(t) for t in operands(a)[:4])
                touched = (fa | fb | (set() if fc == result else fc)) & result   # (its accumulator the hardware forwards, and results are written in order)
            else:
                to, touched = set(), regs(a) & result
            if touched:
                if found is None or d < found[0]:
                    found = (d, q)
                continue
            if o == 's_endpgm' or result <= to:               # (the newer result is looked at in its turn)
                continue
            n = d + 1 + (int(a, 0) if o == 's_nop' else 0)
            if target is not None:
                stack.append((target, n))
            if o != 's_branch':
                stack.append((q + 1, n))
        if found:
            least = found[0] if least is None else min(least, found[0])
            if found[0] < need:
                bad.append((found[0], need, p, found[1]))
    return bad, least


def disassemble(path):
    """llvm-objdump -d of every gfx950 code object in a file."""
    with open(path, 'rb') as f:
        plain = f.read(20)[18:20] == b'\xe0\x00'              # e_machine: AMDGPU
    if plain:
        return subprocess.run([OBJDUMP, '-d', path], capture_output=True, text=True, check=True).stdout
    with tempfile.TemporaryDirectory() as tmp:
        link = os.path.join(tmp, 'f')
        os.symlink(os.path.abspath(path), link)
        subprocess.run([OBJDUMP, '--offloading', link], capture_output=True, check=True, cwd=tmp)
        parts = sorted(p for p in glob.glob(os.path.join(tmp, '*')) if 'gfx950' in os.path.basename(p))
        return '\n'.join(subprocess.run([OBJDUMP, '-d', p], capture_output=True, text=True, check=True).stdout for p in parts)


def main(argv):
    want = argv[argv.index('--kernel') + 1] if '--kernel' in argv else ''
    failed = False
    for name, code in sorted(parse(disassemble(argv[0]), want).items()):
        bad, least = lint(code)
        if least is None:
            continue
        print(f'{least:4d} {name}' + ''.join(f'\n       {d} of {n} wait states: {" ".join(code[p][:2])}  ->  {" ".join(code[q][:2])}' for d, n, p, q in bad))
        failed |= bool(bad)
    return int(failed)


if __name__ == '__main__':
    sys.exit(main(sys.argv[1:]))
