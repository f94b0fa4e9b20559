"""CPU check of how the tensor-core kernels count the time of their waits: the counting itself, compiled for the host."""
import os
import subprocess

from compactwarprnntloss_b200 import build

PROGRAM = r"""
#include <cstdio>
#include "cwrnnt_tc.cuh"
using cwrnnt::tc::Patience;
int main()
{
    const uint64_t ms = 1000000, s = 1000 * ms;
    uint64_t now = 7 * s;
    Patience steady(now);  // looks every 5 us: over after two seconds, not before
    uint64_t looks = 0;
    while (!steady.spent(now += 5000)) ++looks;
    std::printf("%llu\n", (unsigned long long)(looks * 5000 / ms));
    Patience broken(now);  // away for three seconds, twice, then back
    int ran_out = 0;
    for (int i = 0; i < 1000; ++i) ran_out += broken.spent(now += 5000);
    ran_out += broken.spent(now += 3 * s);
    for (int i = 0; i < 1000; ++i) ran_out += broken.spent(now += 5000);
    ran_out += broken.spent(now += 3 * s);
    std::printf("%d\n", ran_out);
    Patience seldom(now);  // a look each second: it ends too
    int seconds = 0;
    while (!seldom.spent(now += s)) ++seconds;
    std::printf("%d\n", seconds);
    return 0;
}
"""


def test_time_away_from_the_gpu_does_not_run_a_wait_out(tmp_path):
    source, program = tmp_path / "waits.cu", tmp_path / "waits"
    source.write_text(PROGRAM)
    csrc = os.path.join(os.path.dirname(build.__file__), "csrc")
    subprocess.run([build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", csrc, str(source), "-o",
                    str(program)], check=True)
    steady, ran_out, seconds = (int(v) for v in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split())
    assert steady == 2000 and ran_out == 0 and seconds == 100
