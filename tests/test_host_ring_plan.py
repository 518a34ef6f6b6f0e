"""The residual norm's rings against an SM's shared memory, for every width that they take: the plan counts on all of its blocks
being resident (a round of blocks beyond that ran almost alone, a quarter of the time at 256 to 768 columns)."""
import pathlib
import shutil
import subprocess

import pytest

HEADER = pathlib.Path(__file__).resolve().parent.parent / "loractl_b200" / "csrc" / "lq_resnorm_plan.cuh"
PROGRAM = r"""
#include <cstdio>
#include "%s"
using namespace resnorm_plan;
int main() {
    for (int backward = 0; backward < 2; ++backward)
        for (int bytes = 2; bytes <= 4; bytes += 2)
            for (int inputs = 1; inputs <= (backward ? 4 : 2); ++inputs)
                for (long h = 8; h <= 8192; h += 8)
                    printf("%%d %%d %%d %%ld %%d %%d %%d\n", backward, bytes, inputs, h, threads_of(h), blocks_per_sm(h, backward),
                           stages_of(h, bytes, inputs, backward));
}
"""


def test_every_planned_block_fits(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src = tmp_path / "plan.cpp"
    src.write_text(PROGRAM % HEADER)
    subprocess.run([gxx, "-std=c++17", "-o", str(tmp_path / "plan"), str(src)], check=True)
    rows = [tuple(map(int, line.split())) for line in subprocess.run([str(tmp_path / "plan")], check=True, capture_output=True, text=True).stdout.splitlines()]
    assert len(rows) == 1024 * 2 * (2 + 4)
    for backward, nbytes, inputs, h, threads, blocks, stages in rows:
        assert threads * 8 >= h and threads % 32 == 0 and 1 <= blocks <= 32 and blocks * threads <= 2048
        assert stages == 0 or 2 <= stages <= 8
        # dynamic ring, the kernel's barriers and sums (580 bytes), the system's kilobyte; in units of 128
        block = -(-(stages * inputs * h * nbytes + 640 + 1024) // 128) * 128
        assert stages * inputs * h * nbytes + 640 <= 227 * 1024
        resident = min(blocks, 228 * 1024 // block)
        assert resident == blocks or (resident == blocks - 1 and stages == 2), (backward, nbytes, inputs, h)
