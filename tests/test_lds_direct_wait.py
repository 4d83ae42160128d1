"""LDS-direct loads written in inline asm: the write of M0, their LDS address, and
the load need a wait state between them (CDNA3 and CDNA4 list the pair among the
hazards that software has to keep apart). The compiler adds it for its own builtin,
but cannot within an asm block."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "rusttorch_amd", "csrc")


def asm_blocks(text):
    """The instructions of every asm statement's template."""
    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)", text):
        template = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
        yield [i.strip() for i in re.split(r"\\n|\\t|;", template) if i.strip()]


def unsafe(block):
    """Loads to LDS that follow a write of M0 at once."""
    return [b for a, b in zip(block, block[1:]) if re.match(r"s_\w+\s+m0\b", a) and re.search(r"load_lds|\blds$", b)]


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.endswith((".hip", ".h", ".cpp"))))
def test_m0_is_written_a_wait_state_ahead(name):
    with open(os.path.join(CSRC, name)) as f:
        for block in asm_blocks(f.read()):
            assert not unsafe(block), block


def test_what_is_found():
    bad = 'asm volatile("s_mov_b32 m0, %1\\n\\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(x) : "memory");'
    good = bad.replace("%1\\n", "%1\\n\\ts_nop 0\\n")
    assert [unsafe(b) for b in asm_blocks(bad)] == [["global_load_lds_dwordx4 %0, off"]]
    assert [unsafe(b) for b in asm_blocks(good)] == [[]]
