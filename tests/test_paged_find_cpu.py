"""The search that every workgroup of paged attention makes for its work."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

REACHED = r"""
#include "%s/scaling_amd/csrc/paged_plan.h"
#include <initializer_list>
#include <stdio.h>
int main() {
    const PagedPlan p = {0, 0x7fffffff, 0x7fffffff, 64, 0, 64, 6, 0, 0};
    for (int n = 1; n <= 1 << 22; n = n * 3 + 1)
        for (int ctx : {0, 1, 20, 300, 5000, 1 << 20, 1 << 30})
            for (int n_rep : {1, 4, 64}) {
                const PagedSeq s = paged_seq(0, n, ctx, n, 1 << 30);
                const PagedWork w = paged_work<256, 64>(p, s, n_rep);
                if ((int64_t)w.blocks * w.tiles > 0x7fffffff) continue;      // refused by the host
                for (int causal = 0; causal < 2; ++causal) {
                    const int r = paged_reached<64>(s, w, causal);
                    if (r < 0 || r > w.blocks * w.tiles) { printf("%%d tokens, %%d keys: %%d\n", n, ctx, r); return 1; }
                }
            }
    printf("ok\n");
    return 0;
}
"""


def _run(tmp_path, program):
    src, exe = tmp_path / "program.cpp", tmp_path / "program"
    src.write_text(program % ROOT)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout + done.stderr


def test_tiles_that_blocks_reach_are_no_fewer_than_none(tmp_path):
    """Of sequences of more tokens than keys, too: their sums over 64 sequences are taken as numbers without a sign."""
    _run(tmp_path, REACHED)
