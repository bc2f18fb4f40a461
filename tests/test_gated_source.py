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


def test_the_normal_integrals_polynomial():
    """t Q(t) exp(-g^2 / 2), with the file's coefficients and factor rounded to fp32 as the kernel has them, against
    erfc(|g| / sqrt 2) / 2, in 64 bits: the bound that the file states."""
    import struct
    body = re.search(r"float normal_below\(.*?\n}", source("sparton_gated.hip"), re.S).group(0)
    f32 = lambda s: struct.unpack("f", struct.pack("f", float(s)))[0]
    factor = f32(re.search(r"rcpf\(fmaf\(([-\d.]+)f", body).group(1))
    c = [f32(re.search(r"float q = ([-\d.]+)f;", body).group(1))]
    c += [f32(v) for v in re.findall(r"q = fmaf\(q, t, ([-\d.]+)f\);", body)]
    assert len(c) == 11 and abs(factor - 0.4 / math.sqrt(2.0)) <= 2.0 ** -26
    worst = 0.0
    for i in range(13001):
        g = i / 1000
        t, q = 1.0 / (1.0 + factor * g), 0.0
        for v in c:
            q = q * t + v
        worst = max(worst, abs(t * q * math.exp(-0.5 * g * g) / (0.5 * math.erfc(g * math.sqrt(0.5))) - 1.0))
    stated = float(re.search(r"relative\s+(?://\s*)?error \(([\d.e-]+), with", source("sparton_gated.hip")).group(1))
    assert 0.9 * stated <= worst <= stated <= 2.0 ** -24, worst
