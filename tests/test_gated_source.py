"""Checks of the gated product's source: what its inline assembly writes, and the polynomial that it states."""
import math
import os
import re

import sparton_amd

CSRC = os.path.join(os.path.dirname(sparton_amd.__file__), "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def test_inline_assembly_names_m0_where_it_writes_it():
    found = 0
    for name in sorted(os.listdir(CSRC)):
        for block in re.findall(r"asm volatile\((.*?)\);", source(name), re.S):
            if re.search(r"s_mov_b32 m0|\bm0, %", block):
                found += 1
                assert re.search(r':\s*"m0"', block), (name, block)
    assert found == 1
