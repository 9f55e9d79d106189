"""Inline assembly in asr_amd/csrc changes no register that the compiler is not told about."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'asr_amd', 'csrc')
SOURCES = sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, '*.hip')) + glob.glob(os.path.join(CSRC, '*.h')))


def _statements(text):
    """(template, operands and clobbers) of every asm statement."""
    for m in re.finditer(r'\basm\b\s*(?:volatile\b|__volatile__\b)?\s*\(', text):
        depth, at, quoted = 1, m.end(), False
        while depth:
            c = text[at]
            if c == '"' and text[at - 1] != '\\':
                quoted = not quoted
            elif not quoted:
                depth += (c == '(') - (c == ')')
            at += 1
        body = text[m.end():at - 1]
        template = re.match(r'\s*((?:"(?:[^"\\]|\\.)*"\s*)*)', body).group(1)
        yield template, body[len(template):]


def _written_by_name(template):
    """Registers that are the first operand of an instruction in the template and are named there."""
    for line in re.split(r'\\n|\\t|;|"', template):
        m = re.match(r'\s*([sv]_\w+)\s+(m0|exec\w*|vcc\w*|scc|[sva]\d+|[sva]\[\d+:\d+\])\b', line)
        if m and not m.group(1).startswith(('s_cmp', 's_waitcnt', 's_nop')):
            yield m.group(2)


def test_the_scan_sees_a_hidden_register():
    text = 'asm volatile("s_mov_b32 m0, %1\\n\\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(at) : "memory");'
    (template, rest), = _statements(text)
    assert list(_written_by_name(template)) == ['m0'] and '"m0"' not in rest


@pytest.mark.parametrize('source', SOURCES)
def test_registers_that_inline_assembly_writes_are_named(source):
    with open(os.path.join(CSRC, source)) as f:
        for template, rest in _statements(f.read()):
            for register in _written_by_name(template):
                assert '"%s"' % register in rest, '%s: %s changes %s' % (source, template.strip(), register)
