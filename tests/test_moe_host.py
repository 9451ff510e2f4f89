"""Index arithmetic of the routing kernels, compiled for the host: no GPU is needed."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cuda-kernel-library_b200", "csrc")


def run_host(tmp_path, source):
    """Compiles `source` with the kernels' headers and runs it on the host; it must return 0."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc here")
    src, exe = tmp_path / "steps.cu", tmp_path / "steps"
    src.write_text(source)
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, "-I",
                    os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


def test_row_of_a_slot(tmp_path):
    """slot / slots_per_row over the whole range of slots, at the borders of every row tried."""
    run_host(tmp_path, """
#include <cstdio>
#include "moe_route.cuh"
#include "ckl_internal.h"
int main() {
    const int divisors[] = {1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 31, 32, 33, 100, 511, 512, 513, 1000, 65535, 65536, 65537,
                            16777215, 16777217, 1073741823, 1073741824, ckl::kMaxExtent, 0x7fffffff};
    for (int d : divisors) {
        const unsigned long long r = ckl::detail::reciprocal_of(d);
        auto right = [&](long long s) {
            if (s < 0 || s > 0x7fffffffll || ckl::detail::quotient(static_cast<int>(s), r) == s / d) return true;
            std::printf("%lld / %d\\n", s, d);
            return false;
        };
        unsigned int x = 1;
        for (int i = 0; i < 100000; ++i) {
            x = x * 1664525u + 1013904223u;
            const long long s = x >> 1, row = s / d * d;
            if (!right(s) || !right(row - 1) || !right(row) || !right(row + d - 1)) return 1;
        }
        for (long long at : {0ll, 1ll << 24, 1ll << 27, static_cast<long long>(ckl::kMaxExtent), 0x7fffffffll}) {
            for (long long s = at - 600; s <= at + 600; ++s) if (!right(s)) return 1;
        }
    }
    return 0;
}
""")


def test_combine_refuses_a_misaligned_row_count(ckl):
    p = 1 << 20
    for call in (lambda: ckl.moe_combine(ckl.F32, p, p, p, p, ckl.F32, 4, 2, 64, 8, kept=p + 2),
                 lambda: ckl.moe_combine_backward(ckl.F32, p, p, p, p, ckl.F32, p, p, 4, 2, 64, 8, kept=p + 1)):
        with pytest.raises(ckl.CklError) as e:
            call()
        assert e.value.status == ckl.ERR_INVALID_ARG
