"""What the packed attention's tensor maps claim (r97b_internal.h rows_extent): the copy engine reads rows that a map claims
when a box begins before them, so a map over T tokens claims their rows and no others, and the blocks that it cannot hold
without doing so (rows_map_has) are not loaded by it. Compiled on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "r97b_internal.h"
#include <cstdio>
int main() {
    for (long T = 1; T <= 700; ++T) {
        for (int claim = 1; claim <= 128; ++claim) {
            const r97b::RowsExtent e = r97b::rows_extent(3, 136, 128, T, claim);
            if (e.cols != 2 * 136 + 128 || e.rows < 1 || e.rows > claim || e.blocks < 1) return printf("shape at T = %ld\n", T), 1;
            if (e.rows - 1 + e.blocks - 1 != T - 1) return printf("T = %ld: row %ld claimed\n", T, (long)(e.rows + e.blocks - 2)), 1;
        }
        const r97b::RowsExtent e = r97b::rows_extent(3, 136, 128, T, 128);
        for (long tok = 0; tok < T; ++tok)
            if (r97b::rows_map_has(tok, T) != (T >= 128 && tok < (long)e.blocks)) return printf("T = %ld, block at %ld\n", T, tok), 1;
    }
    const long T = 0x7FFFFF00;
    return r97b::rows_map_has(T - 128, T) && !r97b::rows_map_has(T - 127, T) && r97b::rows_extent(1, 128, 128, T, 128).blocks == T - 127 ? 0 : 1;
}
"""


def test_maps_claim_no_row_behind_the_batch(tmp_path):
    src = tmp_path / "extent.cpp"
    src.write_text(SOURCE)
    cuda = "/usr/local/cuda/include"
    if not os.path.isdir(cuda):
        pytest.skip("no CUDA headers")
    subprocess.run(["g++", "-std=c++17", "-I", cuda, "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "r97training_b200", "csrc"), str(src), "-o", str(tmp_path / "extent")], check=True)
    r = subprocess.run([str(tmp_path / "extent")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
