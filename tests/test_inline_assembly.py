"""What inline assembly owes the compiler and the hardware (no GPU): read from the
sources, since a wrong one works until a compiler moves something."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "inferrous_amd" / "csrc"


def statements():
    """(file, line, instructions, clobbers) of every asm statement."""
    for path in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.hpp")]):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for start in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
            depth, at = 1, start.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[at], 0)
                at += 1
            body = text[start.end():at - 1]
            parts, depth, quoted, part = [], 0, False, ""
            for ch in body:
                quoted ^= ch == '"'
                depth += 0 if quoted else {"(": 1, ")": -1}.get(ch, 0)
                if ch == ":" and not quoted and depth == 0:
                    parts.append(part)
                    part = ""
                else:
                    part += ch
            parts = [*parts, part, "", "", ""]
            code = "".join(re.findall(r'"([^"]*)"', parts[0])).replace(r"\n", "\n").replace(r"\t", " ")
            yield (path.name, text.count("\n", 0, start.start()) + 1, [c.strip() for c in code.split("\n") if c.strip()],
                   re.findall(r'"([^"]*)"', parts[3]))


ALL = list(statements())
NAMED = re.compile(r"\b(m0|vcc|exec|scc|[sva]\d+)\b")


def test_finds_them():
    assert len(ALL) > 20 and any("m0" in line for s in ALL for line in s[2])


@pytest.mark.parametrize("file, line, code, clobbers", ALL)
def test_a_register_by_name_is_declared(file, line, code, clobbers):
    for c in code:
        written = NAMED.match(c.split(None, 1)[1].split(",")[0].strip()) if " " in c else None
        assert not written or written[1] in clobbers, f"{file}:{line}: {c} writes {written[1]}"


@pytest.mark.parametrize("file, line, code, clobbers", ALL)
def test_m0_is_written_a_wait_state_before_a_load_to_lds(file, line, code, clobbers):
    """A load to LDS may follow a write of m0, its LDS address, after one other instruction."""
    for before, after in zip(code, code[1:]):
        if re.match(r"s_\w+\s+m0\b", before):
            assert not re.search(r"_lds_", after), f"{file}:{line}: {before}; {after}"
