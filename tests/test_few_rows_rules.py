"""How the kernels for few rows cut a product, from the header that both share, compiled by the host compiler.

The rules count CTAs against what the device holds at once (two per SM), so they take its SM count: on
one with fewer SMs a split still fits one wave.
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "pantheon_b200" / "csrc"
FILES = ["qg_gemm_mxfp4_rows.cu", "qg_gemm_gated_rows.cu"]

PROGRAM = r"""
#include "qg_few_rows.cuh"
#include <cstdio>
int main() {
    int M, tiles_n, nk, sms;
    while (std::scanf("%d %d %d %d", &M, &tiles_n, &nk, &sms) == 4)
        std::printf("%d %d %d\n", (int)qg::few_rows::few_tiles(M, tiles_n, sms), qg::few_rows::row_tile(M, tiles_n, sms),
                    qg::few_rows::pick_split(M, tiles_n, nk, sms));
}
"""


def _up(a, b):
    return -(-a // b)


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    assert shutil.which("g++")
    d = tmp_path_factory.mktemp("rules")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", "-x", "c++", str(d / "main.cpp"), "-o", str(d / "main")],
                   check=True, capture_output=True, text=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(d / "main")], input=text, check=True, capture_output=True, text=True).stdout.split()
        v = [int(x) for x in out]
        assert len(v) == 3 * len(cases)
        return list(zip(v[::3], v[1::3], v[2::3]))
    return run


CASES = [(M, t, nk) for M in (1, 16, 17, 33, 64, 65, 128, 200, 512, 1000, 4096) for t in (1, 2, 8, 19, 37, 64, 148, 224)
         for nk in (1, 4, 7, 8, 16, 17, 32, 112)]


@pytest.mark.parametrize("sms", [8, 64, 132, 148, 160])
def test_a_split_fits_one_wave_of_the_device(rules, sms):
    for (M, t, nk), (few, rows, split) in zip(CASES, rules([(*c, sms) for c in CASES])):
        assert few == (4 * t * _up(M, 64) <= 2 * sms)
        assert rows == (16 if M <= 16 else 32 if M <= 32 else 64 if M <= 64 or few else 128)
        tiles = t * _up(M, rows)
        assert split in (1, 2, 4, 8) and (split == 1 or (split * tiles <= 2 * sms and nk >= 4 * split))
        # and no larger one would
        assert split == 8 or 2 * split * tiles > 2 * sms or 8 * split > nk


def test_both_kernels_use_the_one_rule():
    for name in FILES:
        code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        assert "qg_few_rows.cuh" in code
        assert not re.search(r"\b148\b", code)
        assert not re.search(r"\b(bool few_tiles|int row_tile|int pick_split)\s*\(", code)
    for name in ("umma_commit_both",):
        defined = [p.name for p in CSRC.iterdir() if re.search(rf"void {name}\(", p.read_text())]
        assert len(defined) == 1, defined
