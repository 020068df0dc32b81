"""Every wait for a load from tensor memory names the registers of that load."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "arctic_platform_b200" / "csrc"


def sources():
    return {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("*.cu*"))}


def test_no_wait_without_registers():
    bare = {name: len(re.findall(r"\btmem_ld_wait\s*\(\s*\)", text)) for name, text in sources().items()}
    assert not {name: n for name, n in bare.items() if n}


def test_loads_and_waits_stand_in_one_place():
    """Each instruction is wrapped once for every width, and a wait lists its registers as read and written."""
    for name, text in sources().items():
        if name != "common.cuh":
            assert "tcgen05.ld." not in text and "tcgen05.wait::ld" not in text, name
    common = sources()["common.cuh"]
    waits = re.findall(r'asm volatile\(\s*"tcgen05\.wait::ld[^"]*"\s*:\s*("\+r")?', common)
    assert waits and all(waits)

