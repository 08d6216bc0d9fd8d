"""The positions of a batch's rows, from the kernels' own header compiled for the host (no GPU needed) with every signed
overflow an error: lengths are read on the device and may be anything, and shared prefixes are seen by all rows."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

HIP = Path(__file__).resolve().parent.parent / "nibblemac_amd" / "csrc" / "hip"

HEAD = """
#include <climits>
#include <cstdio>
#define __host__
#define __device__
#define __forceinline__ inline
%s
static int bad;
static void same(const char *what, long long got, long long want, long long a, long long b, long long c) {
    if (got != want && bad++ < 5) printf("%%s(%%lld, %%lld, %%lld): %%lld, not %%lld\\n", what, a, b, c, got, want);
}
int main() {
    const int lens[] = {0, 1, 2, 31, 511, 512, 513, 1 << 24, (1 << 24) + 1, 1 << 30, INT_MAX - 1, INT_MAX};
    for (int len : lens)
        for (int count = 1; count <= 512; count += count < 4 ? 1 : 127)
            for (int i = 0; i < count; i += i < 4 ? 1 : 63)
                same("row_position", row_position(len, count, i), (long long)len - count + i, len, count, i);
    const int ends[] = {1, 2, 32, 300, 1 << 24};
    for (int p1 : ends)
        for (int len : lens)
            for (int count = 1; count <= 512; count += count < 4 ? 1 : 127)
                for (int i = 0; i < count; i++) {
                    const int last = row_position(len, count, 0);
                    const long long past = (long long)last + 1 + i;
                    same("positions_seen", positions_seen(last, i, p1), past < p1 ? past : p1, last, i, p1);
                }
    for (int p1 : ends)
        for (int i = 0; i < 512; i++) same("all", positions_seen(ROWS_SEE_ALL, i, p1), p1, ROWS_SEE_ALL, i, p1);
    return bad != 0;
}
"""
# what it was: the sum is formed for a row that sees everything
FORMED = """
constexpr int ROWS_SEE_ALL = 0x7ffffffe;
inline int row_position(int len, int count, int i) { return len - (count - i); }
inline int positions_seen(int last, int i, int p1) {
    volatile int past = last + 1 + i;
    return last >= p1 ? p1 : past < p1 ? past : p1;
}
"""


def run(tmp_path, text):
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(HEAD % text)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{HIP}", str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True)


def test_no_step_leaves_32_bits(tmp_path):
    p = run(tmp_path, '#include "nmx_rowpos.h"')
    assert p.returncode == 0, p.stdout + p.stderr


def test_an_overflow_is_found(tmp_path):
    p = run(tmp_path, FORMED)
    assert p.returncode and "signed integer overflow" in p.stderr, p.stdout + p.stderr


@pytest.mark.parametrize("name", ["row_position", "positions_seen", "ROWS_SEE_ALL"])
def test_the_kernels_take_them_from_there(name):
    text = (HIP / "nmx_attnbatch.hip").read_text()
    assert name in text and "0x7ffffffe" not in text
