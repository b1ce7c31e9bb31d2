"""Reads the assembly of one of this library's own sources and refuses it where a matrix instruction written as inline asm meets a
hazard that the compiler does not see (it does not know what the asm is):

  * a vector instruction that writes an operand less than two issue slots before it;
  * an instruction other than a matrix one that reads a sum less than 18 issue slots behind the instruction that made it.

    python3 check_mfma.py build/hecka_block8_gemm.s"""
import re
import sys


def registers(text):
    found = set()
    for kind, lo, hi in re.findall(r'\b([va])\[(\d+):(\d+)\]', text):
        found |= {(kind, i) for i in range(int(lo), int(hi) + 1)}
    return found | {(kind, int(n)) for kind, n in re.findall(r'\b([va])(\d+)\b', text)}


def check(text):
    faults, seen = [], 0
    for name, body in re.findall(r'\n(\w+):\s*; @\w+\n(.*?)\n\t\.section', text, re.S):
        slot, written, made, inside = 0, {}, {}, False
        for line in body.split('\n'):
            if '#ASMSTART' in line or '#ASMEND' in line:
                inside = '#ASMSTART' in line
                continue
            line = line.split(';')[0].strip()
            if not line or line.startswith('.') or line.endswith(':'):
                continue
            op, _, rest = line.partition(' ') if ' ' in line else line.partition('\t')
            op, _, tail = line.replace('\t', ' ').partition(' ')
            if op == 's_nop':
                slot += int(tail) + 1
                continue
            slot += 1
            args = tail.split(',')
            target = registers(args[0]) if args else set()
            sources = registers(','.join(args[1:]))
            if op.startswith('v_mfma'):
                if inside:
                    seen += 1
                    late = [r for r in sources if slot - written.get(r, -99) <= 2]
                    if late:
                        faults.append('%s: %s reads %s just written' % (name, line, sorted(late)[:2]))
                    made.update({r: slot for r in target})
                else:
                    for r in target:
                        made.pop(r, None)
                for r in target:
                    written.pop(r, None)
                continue
            reads = sources if op.startswith(('v_', 'ds_write', 'buffer_store', 'global_store', 'scratch_store')) else set()
            if op.startswith(('ds_write', 'buffer_store', 'global_store', 'scratch_store')):
                reads = sources | target
            early = [r for r in reads if slot - made.get(r, -99) < 18]
            if early:
                faults.append('%s: %s reads %s before it is settled' % (name, line, sorted(early)[:2]))
            if op.startswith(('v_', 'ds_read', 'buffer_load', 'global_load', 'scratch_load')):
                for r in target:
                    made.pop(r, None)
                    written.pop(r, None)
                    if op.startswith('v_'):
                        written[r] = slot
    return seen, faults


if __name__ == '__main__':
    seen, faults = check(open(sys.argv[1]).read())
    for f in faults[:20]:
        print(f)
    print('%d matrix instructions written as asm, %d hazards' % (seen, len(faults)))
    sys.exit(1 if faults or not seen else 0)
