"""Every load from tensor memory waits within its own asm statement.

tcgen05.ld is asynchronous: its registers hold nothing until tcgen05.wait::ld. A wait in a
statement of its own clobbers memory, but not those registers, so the compiler may move
arithmetic on them between the two."""

import re
from pathlib import Path

CSRC = Path(__file__).parents[1] / "iron_b200" / "csrc"


def test_loads_wait_in_their_own_statement():
    loads = []
    for src in sorted(CSRC.glob("*.cu*")):
        for statement in re.findall(r"\basm\b.*?\);", src.read_text(), re.S):
            if "tcgen05.ld." in statement:
                loads.append((src.name, statement))
    assert loads
    for name, statement in loads:
        assert "tcgen05.wait::ld" in statement, (name, statement)
