"""What the cases of test_gpu_large_products.py are there for: by the rules as they are, each pass of a case takes the tiles
that the case says, and all tiles have a case of every type, pass and way to share them out."""
import pytest

from large_products_cases import all_cases
from product_rules import KINDS, Rules

TABLE = 1022  # experts from which on the tiles' numbers have gaps


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    return Rules(str(tmp_path_factory.mktemp("large_products")))


CASES = [c for c in all_cases() if c["ways"]]


def ways(rules, c):
    if c["op"] == "large":
        slots = c["tokens"] * c["top_k"]
        return [rules.way(kind, c["dtype"], slots, c["experts"], c["out"], c["cols"]) for kind in KINDS]
    if c["op"] == "large_four":
        return [rules.way_four(c["rows"], c["out"], c["cols"])]
    return [rules.way_four(c["tokens"] * c["top_k"], c["out"], c["cols"], c["experts"],
                           0 if c["in_order"] else c["tokens"])]


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["name"])
def test_tiles(rules, case):
    assert ways(rules, case) == case["ways"]


def test_all_tiles_have_cases(rules):
    found = set()
    for c in CASES:
        listed = "four" in c["op"] and "experts" not in c or c["experts"] < TABLE
        if c["op"] == "large":
            slots = c["tokens"] * c["top_k"]
            in_parts = rules.part(c["dtype"], slots, c["experts"], c["out"], c["cols"]) < slots
            for kind, way in zip(KINDS, c["ways"]):
                found.add((kind, c["dtype"] == "float32", way, "parts" if kind == "dweights" and in_parts else listed))
        elif c["op"] == "large_four":
            found.add(("four", -(-c["cols"] // 256) % 2, c["ways"][0], listed))
        else:
            found.add(("in order" if c["in_order"] else "gathered", -(-c["cols"] // 256) % 2, c["ways"][0], listed))
    for way in ("128", "256"):
        for kind in KINDS:
            assert (kind, False, way, True) in found and (kind, True, way, True) in found
        for odd in (0, 1):
            for kind in ("four", "gathered", "in order"):
                assert (kind, odd, way, True) in found
    assert ("dweights", False, "256", "parts") in found and ("dweights", True, "128", "parts") in found
    for kind in ("forward", "drows"):
        assert (kind, False, "256", False) in found
    for kind in ("gathered", "in order"):
        assert (kind, 1, "256", False) in found
