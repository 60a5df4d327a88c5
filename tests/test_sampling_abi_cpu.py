"""The argument blocks of token sampling, steps of a paged cache and attention over shared prefixes, as the header has them."""

import ctypes
import subprocess

import pytest

from scaling_amd import _lib
from tests.test_abi_cpu import HEADER

BLOCKS = {"mi_sample_args": _lib.MiSampleArgs, "mi_paged_step_args": _lib.MiPagedStepArgs, "mi_paged_prefix_attn_args": _lib.MiPagedPrefixAttnArgs}


@pytest.mark.parametrize("name", BLOCKS)
def test_layout_matches_header(name, tmp_path):
    block = BLOCKS[name]
    fields = [f for f, _ in block._fields_]
    source = tmp_path / "layout.c"
    source.write_text(f'#include "{HEADER}"\n#include <stdio.h>\n#include <stddef.h>\nint main() {{ printf("%zu", sizeof({name}));\n'
                      + "".join(f'printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "return 0; }\n")
    subprocess.run(["gcc", str(source), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [ctypes.sizeof(block)] + [getattr(block, f).offset for f in fields]
