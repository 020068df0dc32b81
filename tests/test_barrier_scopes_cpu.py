"""Arrivals at a barrier of another block order memory only at the scope of the cluster; without a scope they have that of their own block."""
import re
from pathlib import Path

import pytest

SOURCES = sorted((Path(__file__).parents[1] / "arctic_platform_b200" / "csrc").glob("*.cu*"))
ARRIVAL = re.compile(r"mbarrier\.(?:arrive|arrive_drop)((?:\.[\w:]+)*)\s")


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_arrivals_at_other_blocks_name_the_clusters_scope(path):
    for qualifiers in ARRIVAL.findall(path.read_text()):
        names = qualifiers.split(".")
        assert "shared::cluster" not in names or "cluster" in names, f"{path.name}: mbarrier.arrive{qualifiers}"


def test_the_look_finds_arrivals():
    found = [q for p in SOURCES for q in ARRIVAL.findall(p.read_text()) if "shared::cluster" in q]
    assert ".release.cluster.shared::cluster.b64" in found and ".relaxed.cluster.shared::cluster.b64" in found
