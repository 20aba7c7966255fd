"""Kernels that round the start of their shared memory up to 1,024 bytes ask for that much more, or check that what they asked for was enough. Read from the
sources (no GPU)."""

import re

import pytest

from paged_attention_engine_b200.kernels import build

ROUNDS = re.compile(r"\(raw \+ 1023u\) & ~1023u")
SIZE = re.compile(r"SMEM_BYTES = ([^;]*);")


@pytest.mark.parametrize("path", sorted(p for p in build.CSRC.glob("*.cu") if ROUNDS.search(p.read_text()) and SIZE.search(p.read_text())), ids=lambda p: p.stem)
def test_the_alignment_has_room(path):
    text = path.read_text()
    sizes = [(m.start(), re.sub(r"/\*.*?\*/", "", m.group(1))) for m in SIZE.finditer(text)]
    for rounding in ROUNDS.finditer(text):
        size = [expression for at, expression in sizes if at < rounding.start()][-1]          # the layout that stands before the kernel
        kernel = text[rounding.start() : rounding.start() + 1500]
        room = any(int(n) >= 1023 for n in re.findall(r"\+ (\d+)", size))
        assert room or "const bool fits = (base - raw) +" in kernel, (path.name, size)
