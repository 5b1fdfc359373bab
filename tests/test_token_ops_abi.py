"""CPU: the ctypes mirrors of the token operators' descriptors have the header's layout, field by field."""
import ctypes
import os
import shutil
import subprocess

import pytest

from agents_amd import _lib

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
MIRRORS = {"aa_categorical_desc": _lib.CategoricalDesc, "aa_layer_norm_desc": _lib.LayerNormDesc}


@pytest.mark.parametrize("name", list(MIRRORS))
def test_layout(tmp_path, name):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    mirror = MIRRORS[name]
    fields = [f for f, _ in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"agents_amd.h\"\nint main(void) {\n" +
                   f'  printf("%zu", sizeof({name}));\n' +
                   "".join(f'  printf(" %zu", offsetof({name}, {f}));\n' for f in fields) +
                   "  return 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", INCLUDE, str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]
