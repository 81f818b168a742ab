"""The ctypes mirrors of the cache operators' structs (busfill_b200.kv4) against include/busfill.h: a
small C program prints each struct's size and field offsets, which must equal the ctypes layout."""
import ctypes
import os
import shutil
import subprocess

import pytest

from busfill_b200 import kv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STRUCTS = {"busfill_kv4": kv4.Cache, "busfill_rope": kv4.Rope, "busfill_kv4_rows": kv4.Rows,
           "busfill_attn": kv4.Attn, "busfill_kv4_eviction": kv4.Eviction}


@pytest.fixture(scope="module")
def c_layout(tmp_path_factory):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    d = tmp_path_factory.mktemp("layout")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "busfill.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        for f, _ in cls._fields_:
            lines.append(f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));')
    lines += ["  return 0;", "}"]
    src = d / "layout.c"
    src.write_text("\n".join(lines) + "\n")
    exe = d / "layout"
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    return {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_ctypes_mirror_matches_c_layout(c_layout, name):
    cls = STRUCTS[name]
    assert ctypes.sizeof(cls) == c_layout[(name, "size")], name
    for f, _ in cls._fields_:
        assert getattr(cls, f).offset == c_layout[(name, f)], (name, f)


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_packed_bytes_are_the_struct(name):
    cls = STRUCTS[name]
    values = [float(i) if t is ctypes.c_float else i for i, (_, t) in enumerate(cls._fields_, 1)]
    data = kv4._packer(cls)(*values)
    assert len(data) == ctypes.sizeof(cls)
    back = cls.from_buffer_copy(data)
    assert [getattr(back, f) for f, _ in cls._fields_] == values
