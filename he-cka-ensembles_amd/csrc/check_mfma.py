"""Reads the assembly of one of this library's own sources and refuses it where a matrix instruction written as inline asm meets a
hazard that the compiler does not see (it does not know what the asm is).  Along every way through a kernel, branches and the ways back to a loop's
start included:

  * a vector instruction that writes an operand less than two issue slots before it;
  * an instruction that reads a sum less than 18 issue slots behind the instruction that made it: any vector or memory instruction, and a
    matrix instruction, whoever made it, that takes it as a factor, or as an addend other than the very sum that it goes on with;
  * an instruction that writes such a sum's registers before those slots are over.

    python3 check_mfma.py build/hecka_block8_gemm.s"""
import re
import sys

READY, SETTLED = 2, 18      # slots: an operand's writer is further away than READY, a sum's maker at least SETTLED


def registers(text):
    found = set()
    for kind, lo, hi in re.findall(r'\b([va])\[(\d+):(\d+)\]', text):
        found |= {(kind, i) for i in range(int(lo), int(hi) + 1)}
    return found | {(kind, int(n)) for kind, n in re.findall(r'\b([va])(\d+)\b', text)}


class Instruction(object):
    """slots it takes; registers it reads and writes; matrix: [factors, addend, sum] of a matrix instruction; own: written as asm."""

    def __init__(self, line, own):
        self.line, self.own = line, own
        op, _, tail = line.replace('\t', ' ').partition(' ')
        args = [a for a in re.split(r',\s*(?![^\[]*\])', tail.strip())]
        self.op, self.slots = op, 1
        self.matrix, self.reads, self.writes, self.vector = None, set(), set(), op.startswith('v_')
        if op == 's_nop':
            self.slots = int(tail) + 1
        elif op.startswith(('v_mfma', 'v_smfma')):
            self.matrix = (registers(','.join(args[1:3] + args[4:])), frozenset(registers(args[3])), frozenset(registers(args[0])))
        elif not op.startswith('s_'):
            first, rest = registers(args[0]) if args else set(), registers(','.join(args[1:]))
            gives = not ('store' in op or 'write' in op and op.startswith('ds_') or 'atomic' in op or re.search(r'\blds\b', tail))
            self.reads = rest if gives else first | rest
            self.writes = first if gives else set()
            if 'swap' in op:      # both operands change places
                self.reads = self.writes = first | rest
            if 'atomic' in op or op.startswith('ds_') and 'rtn' in op:      # may give a value back as well
                self.writes = first


def blocks(body):
    """[(label, instructions, labels that may follow; None: the next block)] of a kernel's text."""
    found, label, now, own = [], '', [], False

    def end(after):
        found.append((label, now, after))
    for line in body.split('\n'):
        if '#ASMSTART' in line or '#ASMEND' in line:
            own = '#ASMSTART' in line
            continue
        line = line.split(';')[0].strip()
        if line.endswith(':') and not line.startswith('.set'):
            end([None])
            label, now = line[:-1], []
            continue
        if not line or line.startswith('.'):
            continue
        now.append(Instruction(line, own))
        if line.startswith(('s_branch', 's_cbranch', 's_endpgm', 's_setpc')):
            to = line.split()[-1]
            end([] if line.startswith(('s_endpgm', 's_setpc')) else [to] if line.startswith('s_branch') else [to, None])
            label, now = '', []
    end([])
    return found


def later(state, slots, most):
    return {k: age + slots for k, age in state.items() if age + slots < most}


def through(instructions, written, made, fault=None):
    """State behind a block.  written: {register: slots since a vector instruction wrote it}; made: {(register, sum's registers): slots since an asm
    product made it}."""
    for i in instructions:
        written, made = later(written, i.slots, READY + 1), later(made, i.slots, SETTLED)
        fresh = {r for r, _ in made}
        if i.matrix:
            factors, addend, total = i.matrix
            if i.own:
                late = [r for r in factors | addend if r in written]
                if late and fault:
                    fault(i, 'reads %s just written' % sorted(late)[:2])
            early = factors & fresh
            early |= {r for r, whole in made if (r in addend and whole != addend) or (r in total and whole != total)}
            if addend != total:
                early |= (addend | total) & fresh
            if early and fault:
                fault(i, 'meets %s before it is settled' % sorted(early)[:2])
            made = {k: age for k, age in made.items() if k[0] not in total}
            if i.own:
                made.update({(r, total): 0 for r in total})
            written = {r: age for r, age in written.items() if r not in total}
            continue
        early = (i.reads | i.writes) & fresh
        if early and fault:
            fault(i, '%s %s before it is settled' % ('reads' if i.reads & fresh else 'writes', sorted(early)[:2]))
        made = {k: age for k, age in made.items() if k[0] not in i.writes}
        written = {r: age for r, age in written.items() if r not in i.writes}
        if i.vector:
            written.update({r: 0 for r in i.writes})
    return written, made


def join(a, b):
    return {k: min(a.get(k, 99), b.get(k, 99)) for k in set(a) | set(b)}


def check(text):
    faults, seen = [], 0
    for name, body in re.findall(r'\n(\w+):\s*; @\w+\n(.*?)\n\t\.section', text, re.S):
        parts = blocks(body)
        seen += sum(1 for _, ins, _ in parts for i in ins if i.matrix and i.own)
        at = {label: k for k, (label, _, _) in enumerate(parts) if label}
        before, todo = {0: ({}, {})}, [0]
        while todo:      # states only gain registers or get younger: this ends
            k = todo.pop()
            out = through(parts[k][1], *before[k])
            for label in parts[k][2]:
                to = k + 1 if label is None else at.get(label)
                if to is None or to >= len(parts):
                    continue
                new = tuple(join(a, b) for a, b in zip(before[to], out)) if to in before else out
                if new != before.get(to):
                    before[to] = new
                    todo.append(to)
        for k, (_, instructions, _) in enumerate(parts):
            through(instructions, *before.get(k, ({}, {})), lambda i, why: faults.append('%s: %s %s' % (name, i.line, why)))
    return seen, faults


if __name__ == '__main__':
    seen, faults = check(open(sys.argv[1]).read())
    for f in faults[:20]:
        print(f)
    print('%d matrix instructions written as asm, %d hazards' % (seen, len(faults)))
    sys.exit(1 if faults or not seen else 0)
