"""Kernels of one call that start under one another's tails (programmatic launches): what one writes, the next must not
read by the read-only path, whose loads are for memory that nobody writes while the kernel lives and which nothing orders
behind griddepcontrol.wait."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "baidu_cti_grab_b200", "csrc")
# the workspaces' fields, which kernels of the same call write
WRITTEN = {
    "attention.cu": ("rows", "tiles", "key_tiles", "delta", "part", "next", "peaks", "redo", "key_segments"),
    "embedding.cu": ("key", "row", "counts", "totals", "heads", "part"),
    "clip.cu": ("sums",),
}


def _arguments(text, call):
    """(line, argument text) of every `call(...)`."""
    at = text.find(call + "(")
    while at >= 0:
        end, depth = at + len(call) + 1, 1
        while depth:
            depth += (text[end] == "(") - (text[end] == ")")
            end += 1
        yield text.count("\n", 0, at) + 1, text[at + len(call) + 1:end - 1]
        at = text.find(call + "(", end)


@pytest.mark.parametrize("name", sorted(WRITTEN))
def test_workspaces_are_read_by_plain_loads(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    assert "griddepcontrol.wait" in text
    fields = "|".join(WRITTEN[name])
    aliases = re.findall(r"\* (\w+) = p\.(?:%s)(?:\[0\])?;" % fields, text)
    pattern = re.compile(r"p\.(?:%s)\b" % fields + "".join(r"|\b%s\b" % a for a in aliases))
    found = [(line, arg) for line, arg in _arguments(text, "__ldg") if pattern.search(arg)]
    assert not found, found
    assert "ld.global.nc" not in text
