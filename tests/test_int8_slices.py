"""How the quantizer's rows are shared out over launches, from the header that the library is built with, compiled for the
host: every row once, every grid below 2^32 threads."""
import os
import subprocess

import pytest

from conftest import ROOT

THREADS = 256
CODE = r"""
#include "int8_slices.h"
#include <stdio.h>
#include <stdlib.h>
int main(int argc, char** argv) {
    for (int i = 1; i + 1 < argc; i += 2) {
        chimere::i8_slices<256>(atoll(argv[i]), atoi(argv[i + 1]), [](int64_t r, int64_t n, int64_t groups) {
            printf("%lld %lld %lld;", (long long)r, (long long)n, (long long)groups); });
        printf("\n");
    }
}
"""


@pytest.fixture(scope="module")
def slices(tmp_path_factory):
    d = tmp_path_factory.mktemp("slices")
    (d / "s.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "chimere_amd", "csrc"), "-o", str(d / "s"),
                    str(d / "s.cpp")], check=True)

    def of(nrows, ncols):
        out = subprocess.run([str(d / "s"), str(nrows), str(ncols)], check=True, capture_output=True, text=True).stdout
        return [tuple(int(v) for v in part.split()) for part in out.strip().split(";") if part]
    return of


@pytest.mark.parametrize("ncols,per", [(1, 4), (1024, 4), (1025, 1), (100000, 1)])
def test_every_row_once(slices, ncols, per):
    for nrows in (0, 1, 5, 2**22 - 1, 2**22, 2**22 + 1, 2**24 - 1, 2**24, 2**24 + 1, 2**26 + 5, 2**31 - 1):
        at = 0
        for first, n, groups in slices(nrows, ncols):
            assert first == at and n > 0 and (groups - 1) * per < n <= groups * per
            assert groups * THREADS < 2**32
            at += n
        assert at == nrows
