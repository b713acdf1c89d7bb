#!/usr/bin/env python
"""ISA lint for the hand-scheduled GEMM kernels: the fragment reads are inline-asm ds_read_b128 whose results hipcc believes
to be ready at once.  Between such a read and the next `s_waitcnt lgkmcnt(0)` NO instruction may touch the destination
registers (a compiler-made copy would copy stale data; a late LDS return would clobber a re-used register).  Followed along
the branches, not along the text: blocks are laid out in any order (a branch that no launch takes, a K loop of no tiles, counts too).
Usage: python tools/check_async_frags.py <file.s> [kernel-name-substring]"""
import re, sys


def regs(tok):
    out = set()
    for m in re.finditer(r'\bv\[(\d+):(\d+)\]', tok):
        out.update(range(int(m.group(1)), int(m.group(2)) + 1))
    for m in re.finditer(r'\bv(\d+)\b', tok):
        out.add(int(m.group(1)))
    return out


def blocks_of(body):
    """([[(line number, instruction)]], [successors]) of a kernel's text"""
    blocks, labels = [[]], {}
    for n, line in enumerate(body.split('\n')):
        label = re.match(r'(\.LBB\w+):', line)
        t = line.split(';')[0].strip()
        if label:
            if blocks[-1]:
                blocks.append([])
            labels[label.group(1)] = len(blocks) - 1
        elif t and not t.startswith('.') and not t.endswith(':'):
            blocks[-1].append((n, t))
            if t.startswith(('s_cbranch', 's_branch', 's_endpgm', 's_setpc')):
                blocks.append([])
    succ = []
    for i, b in enumerate(blocks):
        last = b[-1][1] if b else ""
        to = [labels[last.split()[1]]] if last.startswith(('s_cbranch', 's_branch')) else []
        if last.startswith('s_setpc'):          # a far branch: its target was added to the program counter a few lines above
            to = [labels[f] for _, t in b for f in re.findall(r'\((\.LBB\w+)-\.Lpost_getpc', t)][-1:]
        if not last.startswith(('s_branch', 's_endpgm', 's_setpc')) and i + 1 < len(blocks):
            to.append(i + 1)
        succ.append(to)
    return blocks, succ


def walk(block, pending, report=None):
    """registers with a read in flight behind the block; report(line, instruction, registers) for every touch of one"""
    pending = set(pending)
    for n, t in block:
        if t.startswith('s_waitcnt') and 'lgkmcnt' in t:
            pending.clear()
        elif t.startswith('ds_read_b128'):
            dst, _, addr = t.partition(',')
            touched = regs(addr) & pending      # (a destination re-used by another read = dead result of the redundant tail reads: LDS returns in order)
            if touched and report:
                report(n, t, touched)
            pending |= regs(dst)
        elif regs(t) & pending and report:
            report(n, t, regs(t) & pending)
    return pending


def main():
    s = open(sys.argv[1]).read()
    sub = sys.argv[2] if len(sys.argv) > 2 else ""
    bad = []
    for m in re.finditer(r'^(\S+):\s*; @\1\n(.*?)\.end_amdhsa_kernel', s, re.S | re.M):
        name = m.group(1)
        if sub not in name:
            continue
        blocks, succ = blocks_of(m.group(2))
        before = [set() for _ in blocks]
        todo = list(range(len(blocks)))
        while todo:
            i = todo.pop()
            after = walk(blocks[i], before[i])
            for j in succ[i]:
                if not after <= before[j]:
                    before[j] |= after
                    todo.append(j)
        found = []
        for b, p in zip(blocks, before):
            walk(b, p, lambda n, t, r: found.append(f"{name}: line {n}: {t}  touches pending {sorted(r)[:8]}"))
        print(*found, sep='\n', end='\n' if found else '')
        bad += found
        print(f"{name[-60:]}: {sum(t.startswith('ds_read_b128') for b in blocks for _, t in b)} fragment reads checked")
    print("violations:", len(bad))
    return 1 if bad else 0


if __name__ == "__main__":
    sys.exit(main())
