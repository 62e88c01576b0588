"""The rows that the 8-bit products give to each expert, for counts of any kind: those that are summed in fixed integers against
sums of unbounded ones."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transformers-qwen3-moe-fused_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "fp8_counts.h"
using namespace mfl;
// a wave's scan, 64 experts at a time: sums of growing neighbourhoods, in the order of the lanes' moves
static void scan(uint32_t (&x)[64]) {
    for (int d = 1; d < 16; d *= 2)
        for (int i = 63; i >= 0; --i)
            if (i % 16 >= d) x[i] = fp8_sum(x[i], x[i - d]);
    for (int i = 0; i < 64; ++i)
        if (i / 16 % 2) x[i] = fp8_sum(x[i], x[i / 16 * 16 - 1]);
    for (int i = 32; i < 64; ++i) x[i] = fp8_sum(x[i], x[31]);
}
int main() {
    int wrong = 0;
    const long long kinds[] = {0, 1, 5, 37, -1, -3, 100, 1000, 0x7fffffffll, -0x80000000ll, 0x100000005ll, 0x7fffffffffffffffll,
                               -0x7fffffffffffffffll, 0x40000000ll, 0xffffffffll};
    const long long all_rows[] = {1, 64, 300, 1000, 0x2000000ll, 0x7fffffffll};
    for (int at = 0; at < 6000; ++at) {
        const long long R = all_rows[at % 6];
        const int E = at / 6 % 5 == 0 ? 3 : at / 6 % 5 == 1 ? 64 : 130;
        std::vector<long long> sizes(E);
        for (auto &v : sizes) v = at % 2 ? kinds[std::rand() % 15] : std::rand() % (2 * R / E + 2);
        if (at == 2) sizes = {0x7fffffff, 0x7fffffff, 5};
        const int n = (int)sizes.size();
        __int128 sum = 0;
        uint32_t carry = 0;
        for (int e0 = 0; e0 < n; e0 += 64) {
            uint32_t x[64], count[64];
            for (int i = 0; i < 64; ++i) x[i] = count[i] = e0 + i < n ? fp8_count_of(sizes[e0 + i], (uint32_t)R) : 0u;
            scan(x);
            for (int i = 0; i < 64 && e0 + i < n; ++i) {
                const __int128 first = sum < R ? sum : R;
                if (sizes[e0 + i] > 0) sum += sizes[e0 + i];
                const __int128 last = sum < R ? sum : R;
                const uint32_t room = (uint32_t)R - carry;
                if ((__int128)carry + fp8_begin(x[i], count[i], room) != first || (__int128)carry + fp8_end(x[i], room) != last)
                    if (wrong++ < 5) std::printf("case %d, expert %d of %d, %lld rows\n", at, e0 + i, n, R);
            }
            carry += fp8_end(x[63], (uint32_t)R - carry);
        }
    }
    return wrong ? 1 : 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_counts_of_any_kind_are_cut_at_the_last_row(tmp_path):
    src, exe = tmp_path / "counts.cpp", tmp_path / "counts"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
