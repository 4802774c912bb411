"""Inline assembly of the kernels says what it does with m0, in which the
compiler may hold a value of its own: a statement that writes it names it as
clobbered, one that copies into LDS, whose place m0 gives, takes it as an
operand or writes it itself."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stable-diffusion.assembly_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")))


def statements(text):
    """The asm statements of a source: from `asm` to the parenthesis that ends it."""
    for m in re.finditer(r"\basm\s+(?:volatile\s*)?\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if quoted:
                i += c == "\\"
                quoted = c != '"'
            else:
                quoted = c == '"'
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


def clobbers(statement):
    """What stands after the third colon outside of quotes and parentheses."""
    parts, depth, quoted, start = [], 0, False, 0
    for i, c in enumerate(statement):
        if c == '"':
            quoted = not quoted
        elif not quoted:
            depth += (c == "(") - (c == ")")
            if c == ":" and depth == 1:
                parts.append(statement[start:i])
                start = i + 1
    parts.append(statement[start:])
    return re.findall(r'"([^"]*)"', parts[3]) if len(parts) > 3 else []


def test_parsing():
    s = next(statements('x; asm volatile("s_mov_b32 m0, %0\\n\\tnop" ::"s"(f(a)), "v"(b) : "m0", "memory"); y(":")'))
    assert s.endswith('"memory")') and clobbers(s) == ["m0", "memory"]
    assert clobbers('asm volatile("s_barrier" ::: "memory")') == ["memory"]
    assert clobbers('asm("" : "+v"(x))') == []


def writes_m0(statement):
    return re.search(r"\bs_\w+ m0\b", statement) is not None


@pytest.mark.parametrize("source", SOURCES, ids=[os.path.basename(s) for s in SOURCES])
def test_m0_is_named(source):
    with open(source) as f:
        for s in statements(f.read()):
            assert not writes_m0(s) or "m0" in clobbers(s), s
            if re.search(r"load_lds|_lds_dword|buffer_load\w*[^;]* lds\b", s):
                assert '"{m0}"' in s or writes_m0(s), s
