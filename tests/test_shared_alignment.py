"""Shared arrays that a kernel reads or writes in 8- or 16-byte pieces say their alignment: an array of a scalar type has
that of the scalar alone, and where the compiler happens to put it is not a promise."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "aipu_b200", "csrc")
FILES = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")))
SIZE = {"uint8_t": 1, "char": 1, "uint16_t": 2, "int": 4, "int32_t": 4, "uint32_t": 4, "float": 4, "double": 8, "uint64_t": 8, "int64_t": 8,
        "int2": 8, "uint2": 8, "float2": 8, "int4": 16, "uint4": 16, "float4": 16, "longlong2": 16, "ulonglong2": 16}


def _short(text):
    """(array, bytes it is aligned to, bytes of a piece) of every shared array read in pieces that it is not aligned to."""
    found = []
    for align, typ, names in re.findall(r"__shared__\s+(?:(?:__align__|alignas)\((\d+)\)\s+)?(\w+)\s+([^;]*);", text):
        for name in re.findall(r"(\w+)\s*(?:\[[^,;]*?\])+", names):
            has = int(align) if align else SIZE.get(typ)
            for piece in re.findall(r"reinterpret_cast<(?:const\s+)?(?:volatile\s+)?(\w+)\s*\*>\(\s*&?" + name + r"\b", text):
                if has is not None and SIZE.get(piece, 0) > has:
                    found.append((name, has, SIZE[piece]))
    return found


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_arrays_read_in_pieces_are_aligned_to_them(path):
    with open(path) as f:
        assert _short(f.read()) == []


def test_the_check_sees_a_short_alignment():
    read = "x = *reinterpret_cast<const int4*>(key + i);"
    assert _short("__shared__ int key[256];" + read) == [("key", 4, 16)]
    assert _short("__shared__ int other, key[256];" + read) == [("key", 4, 16)]
    assert _short("__shared__ __align__(16) int key[256];" + read) == []
    assert _short("__shared__ int4 key[64];" + read) == []
