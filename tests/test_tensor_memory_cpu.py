"""The address of a kernel's tensor memory, written to shared memory by the allocation and read by every warp."""

from __future__ import annotations

import re
from pathlib import Path

import lite_llama_b200

CSRC = Path(lite_llama_b200.__file__).parent / "csrc"
ALLOCATION = re.compile(r"tmem_alloc(?:_pair)?\(&(\w+->\w+),")


def gaps():
    """(file, source text between an allocation and the first use of what it wrote)."""
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for site in ALLOCATION.finditer(text):
            use = text.find(site.group(1), site.end())
            assert use > 0, path.name
            if not ALLOCATION.search(text, site.start() + 1, use + len(site.group(1)) + 1):      # the last of several forms
                yield path.name, text[site.end():use]


def test_the_address_is_read_behind_a_barrier_that_shows_it():
    """A barrier of the CTA, or of the cluster with release: one that arrives relaxed orders no ordinary store."""
    seen = list(gaps())
    assert len({name for name, _ in seen}) >= 8
    for name, between in seen:
        assert re.search(r"\b(__syncthreads(_or|_and|_count)?|pair_sync)\(", between), name
