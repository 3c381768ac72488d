"""Waits that inline assembly has to bring itself: the compiler's own hazard
handling ends at its border."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "trispconv_amd" / "csrc"


def _blocks():
    """(file, the lines of instructions) of every inline assembly statement."""
    for path in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.hpp")]):
        for text in re.findall(r'\basm\s*volatile\s*\(\s*((?:"[^"]*"\s*)+)', path.read_text()):
            code = "".join(re.findall(r'"([^"]*)"', text))
            # s_nop may be written as its word
            code = re.sub(r"\.long 0xbf8000(\d\d)", lambda m: f"s_nop {int(m[1], 16)}", code)
            lines = [s.strip() for s in re.split(r"\\n|;", code.replace("\\t", " "))]
            yield path.name, [s for s in lines if s]


def test_m0_settles_before_a_load_to_lds():
    """A load to LDS takes its LDS address from M0 and may not be the next
    instruction behind the one that writes M0 (one wait state on CDNA; the
    compiler puts an s_nop there around its own loads)."""
    seen = 0
    for name, lines in _blocks():
        for i, line in enumerate(lines):
            if re.match(r"s_\w+\s+m0\b", line):
                seen += 1
                assert i + 1 < len(lines) and lines[i + 1].startswith("s_nop"), (name, lines)
    assert seen >= 3


def test_a_base_in_scalar_registers_settles_before_a_load():
    """A scalar register that a vector instruction wrote may be read by a memory
    instruction five wait states later (CDNA).  Base addresses come back from
    spilled registers through v_readlane right before the statement, so it has
    to bring the five itself."""
    seen = 0
    for name, lines in _blocks():
        for i, line in enumerate(lines):
            if re.match(r"(global|buffer|scratch)_", line) and not line.endswith("off"):
                seen += 1
                waits = sum(1 + int(re.match(r"s_nop\s+(\d+)", s)[1]) if s.startswith("s_nop") else 1
                            for s in lines[:i])
                assert waits >= 5, (name, lines)
    assert seen >= 1
