"""The limits that the header declares for the float experts and the adapters are the ones Python names, and every entry point of that
section has its binding."""
import re
from pathlib import Path

import pytest

HEADER = (Path(__file__).resolve().parent.parent / "include" / "phx_moe.h").read_text()
SECTION = HEADER[HEADER.index("float experts, adapters, the residual's norm"):]
ENTRIES = re.findall(r"^(?:int|void) (phx_\w+)\(", SECTION, flags=re.M)


@pytest.mark.parametrize("name", ["MAX_ADAPTERS", "MAX_RANK"])
def test_python_mirror(pkg, name):
    assert f"#define PHX_{name} {getattr(pkg.PHX, name)}\n" in HEADER


def test_every_entry_point_is_bound(pkg):
    assert len(ENTRIES) == 8
    source = (Path(pkg.moe.__file__)).read_text()
    for name in ENTRIES:
        assert re.search(rf"\b{name}\b", source), name
