"""CPU: what the inline assembly of the kernels has to bring along, read from the sources."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_inline_asm_memory_instructions_bring_their_wait_states():
    """An SGPR written by a VALU instruction (v_readfirstlane of a buffer descriptor) may not be read by a vector-memory instruction for five wait states; the
    compiler does not look into inline asm.  Every asm statement with a buffer_* instruction spends at least five in front of it."""
    csrc = os.path.join(ROOT, 'open-solution-mapping-challenge_amd', 'csrc')
    seen = 0
    for f in sorted(os.listdir(csrc)):
        if not f.endswith(('.hip', '.h')):
            continue
        for text in re.findall(r'asm volatile\(\s*"([^"]*)"', open(os.path.join(csrc, f)).read()):
            if 'buffer_' not in text:
                continue
            seen += 1
            lines = text.replace('\\t', ' ').split('\\n')
            at = next(i for i, l in enumerate(lines) if 'buffer_' in l)
            states = sum(int(l.split()[1]) + 1 if l.split()[0] == 's_nop' else 1 for l in lines[:at])
            assert states >= 5, (f, text)
    assert seen >= 4


def asm_statements(source):
    """(template, operands) of every asm statement: the literals joined as the compiler joins them, up to the first colon outside of one"""
    for m in re.finditer(r'\basm\b(?:\s+volatile)?\s*\(', source):
        i, literals, rest = m.end(), [], None
        while rest is None:
            i += len(re.match(r'\s*', source[i:]).group())
            if source[i] == '"':
                literal = re.match(r'"((?:[^"\\]|\\.)*)"', source[i:])
                literals.append(literal.group(1))
                i += literal.end()
            else:
                rest = source[i:source.index(';', i)]
        yield ''.join(literals).replace('\\t', ' '), rest


def memory_without_waits(source):
    """the vector-memory instructions of `source`'s asm that read scalar registers, with fewer than five wait states in front of them"""
    for text, operands in asm_statements(source):
        lines = [l.strip() for l in re.split(r'\\n|;', text) if l.strip()]
        scalar = re.search(r'"[^"]*[sS][^"]*"\s*\(', operands) is not None or re.search(r'\bs\[?\d', text) is not None
        for at, line in enumerate(lines):
            if re.match(r'(buffer|global|flat|scratch|tbuffer|image)_', line) and scalar:
                states = sum(int(l.split()[1]) + 1 if l.split()[0] == 's_nop' else 1 for l in lines[:at])
                if states < 5:
                    yield line


def sources():
    csrc = os.path.join(ROOT, 'open-solution-mapping-challenge_amd', 'csrc')
    return {f: re.sub(r'//[^\n]*', '', open(os.path.join(csrc, f)).read()) for f in sorted(os.listdir(csrc)) if f.endswith(('.hip', '.h'))}


def test_every_asm_statement_is_read_whole():
    """... whatever its literals, and every kind of vector-memory instruction that takes a scalar register"""
    seen = 0
    for f, text in sources().items():
        assert list(memory_without_waits(text)) == [], f
        seen += sum('buffer_' in t for t, _ in asm_statements(text))
    assert seen == sum(len(re.findall(r'"[^"\n]*buffer_(?:load|store)_', text)) for text in sources().values()) >= 5      # none is written in a way that this misses


def test_the_reader_of_asm_statements_finds_what_it_is_for():
    split = 'asm volatile("s_mov_b32 m0, %1\\n\\t"\n   "buffer_load_dword %0, %2, 0 offen lds" : "=v"(x) : "s"(a), "s"(r) : "memory");'
    assert list(memory_without_waits(split)) == ['buffer_load_dword %0, %2, 0 offen lds']
    assert list(memory_without_waits('asm("global_load_dword %0, %1, %2" : "=v"(x) : "v"(o), "s"(p));')) == ['global_load_dword %0, %1, %2']
    assert list(memory_without_waits('asm volatile ("s_nop 4\\n\\t" "global_load_dword %0, %1, %2" : "=v"(x) : "v"(o), "s"(p));')) == []
    assert list(memory_without_waits('asm volatile("global_store_dwordx4 %0, %1, off" ::"v"(p), "v"(t) : "memory");')) == []      # no scalar register
