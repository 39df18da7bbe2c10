"""What the compiler does not look after in the kernels' assembly, checked in the code that was built (no GPU): an instruction on memory that reads a scalar register
written by a vector instruction needs five wait states in between, and a load straight into LDS one behind the write of m0; and such loads have to be waited for before the
workgroup ends and its LDS goes to another.  The compiler keeps all that for its own instructions, not for those of an assembly block."""
import os
import re
import struct
import subprocess

import pytest

import panogrf_amd

OBJDUMP = '/opt/rocm/llvm/bin/llvm-objdump'
LIB = os.path.join(os.path.dirname(panogrf_amd.__file__), 'libpanogrf_hip.so')
MEMORY = re.compile(r'(global|buffer|scratch|flat)_')
SCALARS = re.compile(r'\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc|m0)\b')


def scalars(text):
    for lo, hi, one, name in SCALARS.findall(text):
        if name:
            yield name
        elif one:
            yield int(one)
        else:
            yield from range(int(lo), int(hi) + 1)


def too_close(lines):
    """-> [(function, instruction)] of memory instructions that come too soon behind what their scalar operands come from.  `lines`: a listing of objdump."""
    bad, name, now, written, m0 = [], '', 0, {}, -9
    for line in lines:
        head = re.match(r'[0-9a-f]+ <(.*)>:$', line)
        if head:
            name, now, written, m0 = head.group(1), 0, {}, -9
            continue
        text = line.split('//')[0].strip()
        if not text or text.endswith(':'):
            continue
        op, _, rest = text.partition(' ')
        args = rest.split(',')
        if MEMORY.match(op):
            reads = list(scalars(rest)) + ['m0'] * ('_lds_' in op)
            if any(now - written.get(r, -9) - 1 < 5 for r in reads) or ('_lds_' in op and now - m0 - 1 < 1):
                bad.append((name, text))
        if op.startswith('v_'):                                      # (the destination, and the carry or comparison behind it)
            outs = args[:2] if op.startswith(('v_add_co', 'v_addc_co', 'v_sub_co', 'v_subb_co', 'v_subrev_co', 'v_div_scale', 'v_mad_u64', 'v_mad_i64')) else args[:1]
            for r in scalars(','.join(outs)):
                written[r] = now
        elif op.startswith('s_'):
            for r in scalars(args[0]):
                written.pop(r, None)
                if r == 'm0':
                    m0 = now
        now += int(args[0]) + 1 if op == 's_nop' else 1
    return bad


def ends_with_loads(lines):
    """-> [(function, end)] of ends of a program that a load straight into LDS (or a call, which may make some) reaches without a wait for all loads, on any path of branches."""
    bad, functions = [], []
    for line in lines:
        head = re.match(r'([0-9a-f]+) <(.*)>:$', line)
        if head:
            functions.append((head.group(2), int(head.group(1), 16), []))
        elif functions and '// ' in line and line.strip():
            text, _, note = line.partition('//')
            functions[-1][2].append((int(note.split(':')[0], 16), text.strip(), note))
    for name, start, code in functions:
        place = {at: i for i, (at, _, _) in enumerate(code)}
        todo, seen = [(0, False)] if code else [], set()
        while todo:
            i, flying = todo.pop()
            if (i, flying) in seen or i >= len(code):
                continue
            seen.add((i, flying))
            text, note = code[i][1], code[i][2]
            if text.startswith('s_endpgm'):
                if flying:
                    bad.append((name, hex(code[i][0])))
                continue
            if 'load_lds' in text or text.startswith('s_swappc'):
                flying = True
            elif text.startswith('s_waitcnt') and 'vmcnt(0)' in text:
                flying = False
            if text.startswith(('s_branch', 's_cbranch')):
                todo.append((place[start + int(re.search(r'\+0x([0-9a-f]+)>', note).group(1), 16)], flying))
            if not text.startswith(('s_branch', 's_setpc')):
                todo.append((i + 1, flying))
    return sorted(set(bad))


def code_objects():
    data, mark, at = open(LIB, 'rb').read(), b'__CLANG_OFFLOAD_BUNDLE__', 0
    while (at := data.find(mark, at)) >= 0:
        o = at + 32
        for _ in range(struct.unpack_from('<Q', data, at + 24)[0]):
            off, size, n = struct.unpack_from('<QQQ', data, o)
            if b'gfx950' in data[o + 24:o + 24 + n] and b'diff_attn' in data[at + off:at + off + size]:
                yield data[at + off:at + off + size]
            o += 24 + n
        at += 24


def test_the_check_itself():
    near = ['0 <f>:', '  v_readfirstlane_b32 s4, v1', '  s_mov_b32 m0, s8', '  s_nop 0', '  global_load_lds_dwordx4 v2, s[4:5]']
    assert too_close(near) == [('f', 'global_load_lds_dwordx4 v2, s[4:5]')]
    assert not too_close(near[:3] + ['  s_nop 3'] + near[4:])
    assert not too_close(['0 <f>:', '  v_readfirstlane_b32 s4, v1', '  s_nop 4', '  global_load_dword v2, v3, s[4:5]'])
    assert not too_close(['0 <f>:', '  v_readfirstlane_b32 s4, v1', '  s_add_u32 s4, s4, 1', '  global_load_dword v2, v3, s[4:5]'])
    assert too_close(['0 <f>:', '  s_mov_b32 m0, s8', '  global_load_lds_dwordx4 v2, s[4:5]'])
    loads = ['0000 <f>:', ' global_load_lds_dword v2, s[4:5] // 000: 0', ' s_cbranch_scc1 1 // 008: 0 <f+0x10>', ' s_waitcnt vmcnt(0) // 00c: 0', ' s_endpgm // 010: 0']
    assert ends_with_loads(loads) == [('f', '0x10')]
    assert not ends_with_loads(loads[:2] + loads[3:]) and not ends_with_loads(loads[:1] + loads[2:])


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason='no llvm-objdump')
def test_waits_of_memory_instructions(tmp_path):
    seen, flying = 0, []
    for i, code in enumerate(code_objects()):
        path = tmp_path / f'{i}.co'
        path.write_bytes(code)
        listing = subprocess.run([OBJDUMP, '-d', '--no-show-raw-insn', str(path)], check=True, capture_output=True, text=True).stdout.splitlines()
        seen += sum('global_load_lds' in line for line in listing)
        assert too_close(listing) == []
        flying += ends_with_loads(listing)
    assert seen > 0
    assert flying == []
