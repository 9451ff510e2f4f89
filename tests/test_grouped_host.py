"""Refusals of the routing, grouped and adapter entry points: no GPU is needed to be told that an
argument is wrong, and degenerate sizes are no-ops that touch nothing."""

import ctypes

import pytest

P = 1 << 20  # an address that is never read: every call here returns before a launch


def status(ckl, f, *a, **k):
    with pytest.raises(ckl.CklError) as e:
        f(*a, **k)
    return e.value.status


def grouped(ckl, **over):
    a = dict(ab_dtype=ckl.BF16, a=P, b=P, c=P, c_dtype=ckl.F32, offsets=P, groups=4, rows=16, n=64, k=64)
    a.update(over)
    return ckl.gemm_grouped(**a)


@pytest.mark.parametrize("over,code", [
    (dict(ab_dtype=0), "INVALID_ARG"), (dict(c_dtype=7), "INVALID_ARG"), (dict(a=None), "INVALID_ARG"),
    (dict(b=None), "INVALID_ARG"), (dict(c=None), "INVALID_ARG"), (dict(offsets=None), "INVALID_ARG"),
    (dict(groups=0), "INVALID_ARG"), (dict(groups=1025), "TOO_LARGE"), (dict(lda=63), "INVALID_ARG"),
    (dict(ldb=63), "INVALID_ARG"), (dict(ldc=63), "INVALID_ARG"), (dict(lda=65), "UNSUPPORTED"),
    (dict(ldb=68), "UNSUPPORTED"), (dict(a=P + 2), "UNSUPPORTED"), (dict(b=P + 8), "UNSUPPORTED"),
    (dict(stride_b=4100), "UNSUPPORTED"), (dict(stride_b=-8), "INVALID_ARG"), (dict(c=P + 2), "INVALID_ARG"),
    (dict(offsets=P + 2), "INVALID_ARG"), (dict(a_rows=P, a_count=-1), "INVALID_ARG"),
    (dict(a_rows=P + 1, a_count=3), "INVALID_ARG"), (dict(trans_b=True, ldb=56), "INVALID_ARG"),
])
def test_grouped_refusals(ckl, over, code):
    assert status(ckl, grouped, ckl, **over) == getattr(ckl, "ERR_" + code)
    assert "gemm_grouped" in ckl.last_error()


def test_gather_needs_a_count(ckl):
    with pytest.raises(ValueError):
        grouped(ckl, a_rows=P)
    with pytest.raises(ValueError):
        ckl.gemm_grouped_wgrad(ckl.F16, P, P, P, ckl.F32, P, 1, 1, 8, 8, a_rows=P)


def wgrad(ckl, **over):
    a = dict(ab_dtype=ckl.F16, a=P, g=P, dw=P, dw_dtype=ckl.F32, offsets=P, groups=4, rows=16, m=64, n=64)
    a.update(over)
    return ckl.gemm_grouped_wgrad(**a)


@pytest.mark.parametrize("over,code", [
    (dict(ab_dtype=3), "INVALID_ARG"), (dict(dw=None), "INVALID_ARG"), (dict(a=None), "INVALID_ARG"),
    (dict(g=P + 4), "UNSUPPORTED"), (dict(ldg=72 + 1), "UNSUPPORTED"), (dict(lddw=8), "INVALID_ARG"),
    (dict(stride_dw=-1), "INVALID_ARG"), (dict(groups=2000), "TOO_LARGE"), (dict(dw=P + 1), "INVALID_ARG"),
])
def test_wgrad_refusals(ckl, over, code):
    assert status(ckl, wgrad, ckl, **over) == getattr(ckl, "ERR_" + code)


def lora(ckl, **over):
    a = dict(ab_dtype=ckl.F16, x=P, w=P, lora_a=P, lora_b=P, scales=None, y=P, y_dtype=ckl.F16, offsets=P, rows=P,
             adapters=4, m=32, n=64, k=64, rank=16, workspace=P, workspace_bytes=1 << 20)
    a.update(over)
    return ckl.gemm_lora(**a)


def lora_backward(ckl, **over):
    a = dict(ab_dtype=ckl.F16, dy=P, x=P, w=P, lora_a=P, lora_b=P, scales=None, dx=P, dx_dtype=ckl.F16, da=P, db=P,
             dab_dtype=ckl.F32, offsets=P, rows=P, adapters=4, m=32, n=64, k=64, rank=16, workspace=P,
             workspace_bytes=1 << 20)
    a.update(over)
    return ckl.gemm_lora_backward(**a)


@pytest.mark.parametrize("call", [lora, lora_backward], ids=["forward", "backward"])
@pytest.mark.parametrize("over,code", [
    (dict(rank=0), "INVALID_ARG"), (dict(rank=129), "TOO_LARGE"), (dict(adapters=0), "INVALID_ARG"),
    (dict(adapters=1025), "TOO_LARGE"), (dict(w=None), "INVALID_ARG"), (dict(x=P + 2), "UNSUPPORTED"),
    (dict(lora_a=P + 2), "UNSUPPORTED"), (dict(rank=12, ldla=12), "UNSUPPORTED"), (dict(ldla=8), "INVALID_ARG"),
    (dict(ldlb=60), "INVALID_ARG"), (dict(workspace=None), "INVALID_ARG"), (dict(workspace=P + 16), "INVALID_ARG"),
    (dict(workspace_bytes=100), "INVALID_ARG"), (dict(scales=P + 1), "INVALID_ARG"), (dict(rows=P + 2), "INVALID_ARG"),
    (dict(offsets=None), "INVALID_ARG"), (dict(ab_dtype=0), "INVALID_ARG"), (dict(stride_b=3), "UNSUPPORTED"),
])
def test_lora_refusals(ckl, call, over, code):
    assert status(ckl, call, ckl, **over) == getattr(ckl, "ERR_" + code)


def test_lora_output_refusals(ckl):
    assert status(ckl, lora, ckl, y=None) == ckl.ERR_INVALID_ARG
    assert status(ckl, lora, ckl, ldy=63) == ckl.ERR_INVALID_ARG
    assert status(ckl, lora, ckl, k=0, ldx=8) == ckl.ERR_INVALID_ARG
    for over in (dict(lddx=63), dict(ldda=15), dict(lddb=63), dict(dx=P + 1), dict(da=P + 1), dict(db=P + 2),
                 dict(stride_da=-8), dict(dab_dtype=9), dict(dy=None)):
        assert status(ckl, lora_backward, ckl, **over) == ckl.ERR_INVALID_ARG


def test_lora_workspace_size(ckl):
    size = ckl.gemm_lora_workspace_bytes
    assert size(0, 16) == 0 and size(5, 0) == 0 and size(5, 129) == 0
    for m, rank in ((1, 1), (7, 16), (1000, 100), (1 << 24, 128)):
        one = (m * 2 * ((rank + 15) // 16 * 16) * 2 + 255) // 256 * 256
        assert size(m, rank) == 4096 + one
        assert size(m, rank, True) == 4096 + 2 * one


def route(ckl, **over):
    a = dict(logit_dtype=ckl.F32, logits=P, weights=P, experts=P, tokens=4, n_experts=64, top_k=6)
    a.update(over)
    return ckl.moe_route(**a)


@pytest.mark.parametrize("over,code", [
    (dict(logit_dtype=4), "INVALID_ARG"), (dict(logits=None), "INVALID_ARG"), (dict(ldl=63), "INVALID_ARG"),
    (dict(top_k=0), "INVALID_ARG"), (dict(top_k=65), "INVALID_ARG"), (dict(top_k=33), "TOO_LARGE"),
    (dict(n_experts=0), "INVALID_ARG"), (dict(n_experts=1025), "TOO_LARGE"), (dict(score=2), "INVALID_ARG"),
    (dict(groups=0), "INVALID_ARG"), (dict(groups=5), "INVALID_ARG"), (dict(groups=8, top_groups=9), "INVALID_ARG"),
    (dict(groups=64, top_groups=2), "TOO_LARGE"), (dict(weights=None), "INVALID_ARG"), (dict(experts=None), "INVALID_ARG"),
    (dict(bias=P + 2), "INVALID_ARG"), (dict(logits=P + 2), "INVALID_ARG"),
])
def test_route_refusals(ckl, over, code):
    assert status(ckl, route, ckl, **over) == getattr(ckl, "ERR_" + code)


def test_other_refusals(ckl):
    bad = ckl.ERR_INVALID_ARG
    assert status(ckl, ckl.moe_route_backward, ckl.F32, P, P, None, P, 4, 64, 6) == bad
    assert status(ckl, ckl.moe_route_backward, ckl.F32, P, P, P, P, 4, 64, 6, ldd=60) == bad
    assert status(ckl, ckl.group_rows, P, 4, 0, P, P, P) == bad
    assert status(ckl, ckl.group_rows, P, -1, 3, P, P, P) == bad
    assert status(ckl, ckl.group_rows, P, 4, 3, P, None, P) == bad
    assert status(ckl, ckl.group_rows, P, 4, 3, P, P, P, slots_per_row=0) == bad
    assert status(ckl, ckl.group_rows, P, 4, 1025, P, P, P) == ckl.ERR_TOO_LARGE
    assert status(ckl, ckl.moe_combine, ckl.F32, P, P, P, P, 5, 4, 2, 64, 8) == bad
    assert status(ckl, ckl.moe_combine, ckl.F32, P, P, P, P, ckl.F32, 4, 0, 64, 8) == bad
    assert status(ckl, ckl.moe_combine, ckl.F32, P, None, P, P, ckl.F32, 4, 2, 64, 8) == bad
    assert status(ckl, ckl.moe_combine, ckl.F32, P, P, P, P, ckl.F32, 4, 2, 64, 8, ldy=60) == bad
    assert status(ckl, ckl.moe_combine_backward, ckl.F32, P, P, P, P, ckl.F32, None, P, 4, 2, 64, 8) == bad
    assert status(ckl, ckl.moe_combine_backward, ckl.F32, P, P, P, P, ckl.F32, P, P, 4, 2, 64, 8, lddy=3) == bad


def test_degenerate_sizes_are_no_ops(ckl):
    grouped(ckl, rows=0, a=None)
    grouped(ckl, n=0)
    wgrad(ckl, m=0)
    wgrad(ckl, n=0)
    lora(ckl, m=0)
    lora(ckl, n=0)
    lora_backward(ckl, n=0)
    route(ckl, tokens=0)
    ckl.moe_combine(ckl.F32, None, None, None, None, ckl.F32, 0, 2, 64, 8)
    ckl.moe_combine_backward(ckl.F32, None, None, None, None, ckl.F32, None, None, 4, 2, 0, 8)


def test_no_cpu_fallback(ckl):
    """Valid arguments on a machine without the GPU fail with a status, never with a crash."""
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("this machine has a GPU")
    for call in (grouped, wgrad, lora, lora_backward, route):
        assert status(ckl, call, ckl) in (ckl.ERR_CUDA, ckl.ERR_UNSUPPORTED)


def test_exported_from_the_library(ckl):
    lib = ctypes.CDLL(ckl.LIB_PATH)
    for name in ("ckl_group_rows", "ckl_moe_route", "ckl_moe_route_backward", "ckl_gemm_grouped",
                 "ckl_gemm_grouped_wgrad", "ckl_moe_combine", "ckl_moe_combine_backward", "ckl_gemm_lora",
                 "ckl_gemm_lora_backward", "ckl_gemm_lora_workspace_bytes"):
        assert hasattr(lib, name)


def test_counts_that_32_bit_steps_would_pass(ckl):
    big = 2 ** 31 - 1
    for f in (lambda: grouped(ckl, rows=big), lambda: grouped(ckl, n=big, ldb=big - 7, ldc=big, trans_b=True),
              lambda: grouped(ckl, k=big), lambda: wgrad(ckl, rows=big), lambda: wgrad(ckl, m=big),
              lambda: lora(ckl, m=big), lambda: ckl.group_rows(P, big, 4, P, P, P),
              lambda: ckl.moe_route(ckl.F32, P, P, P, big, 8, 2),
              lambda: ckl.moe_combine(ckl.F32, P, P, P, P, ckl.F32, 4, 2, big, 8)):
        assert status(ckl, f) == ckl.ERR_TOO_LARGE


def test_cpp_header_compiles(tmp_path, ckl):
    """include/ckl/grouped.hpp compiles as C++17 and links against the library."""
    import os
    import shutil
    import subprocess
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc here")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "use_grouped.cu"
    src.write_text("""
#include "ckl/grouped.hpp"
int main(int argc, char**) {
    if (argc < 100) return ckl::gemm_lora_workspace_bytes(1, 16) == 0;
    __half* h = nullptr; __nv_bfloat16* b = nullptr; float* f = nullptr; int* i = nullptr;
    ckl::group_rows(i, 1, 1, 1, i, i, i);
    ckl::moe_route(f, f, i, 1, 8, 2);
    ckl::moe_route(h, f, i, 1, 8, 2, ckl::RouteOptions{});
    ckl::moe_route_backward(b, i, f, b, 1, 8, 2);
    ckl::gemm_grouped(h, i, 1, h, f, i, 1, 1, 8, 8);
    ckl::gemm_grouped_wgrad(b, i, 1, b, b, i, 1, 1, 8, 8);
    ckl::moe_combine(h, i, f, f, 1, 1, 8, 1);
    ckl::moe_combine_backward(h, i, f, f, h, f, 1, 1, 8, 1);
    ckl::gemm_lora(h, h, h, h, f, f, i, i, 1, 1, 8, 8, 8, f, 4096);
    ckl::gemm_lora_backward(h, h, h, h, h, f, f, f, f, i, i, 1, 1, 8, 8, 8, f, 4096);
}
""")
    exe = tmp_path / "use_grouped"
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I",
                    os.path.join(root, "include"), "-o", str(exe), str(src), ckl.LIB_PATH,
                    "-Xlinker", f"-rpath={os.path.dirname(ckl.LIB_PATH)}"], check=True)
    assert subprocess.run([str(exe)]).returncode == 0


def test_steps_at_the_largest_extent(tmp_path):
    """The walks of the adapters' kernels at the largest row count that is accepted: compiled for the host,
    no step may come back below the limit after it has passed it."""
    from test_moe_host import run_host
    run_host(tmp_path, """
#include <cstdio>
#include "gemm_grouped.cuh"
#include "ckl_internal.h"
int main() {
    const int limit = ckl::kMaxExtent, step = ckl::kExtChecks * ckl::kExtCheckThreads;
    for (int units : {1, 2, 3, 16, 17, 520, step, step + 1, 1 << 20}) {
        for (int first : {0, 1, 37, step - 1}) {
            for (int rows : {1, 5, 4096, limit - 1, limit}) {
                ckl::detail::UnitWalk at(first, step, units);
                if (rows > 1 << 20) {  // straight to the last rows
                    const unsigned long long steps = (static_cast<unsigned long long>(rows - 1) * units) / step;
                    const unsigned long long unit = first + steps * step;
                    at.r = static_cast<unsigned int>(unit / units);
                    at.u = static_cast<int>(unit % units);
                }
                unsigned long long unit = static_cast<unsigned long long>(at.r) * units + at.u;
                for (int i = 0; i < 12; ++i, unit += step) {  // inside a batch of four, and as far again behind it
                    const bool inside = unit / units < static_cast<unsigned long long>(rows);
                    if (at.inside(rows) != inside || (inside && (at.r != unit / units || at.u != int(unit % units)))) {
                        std::printf("rows %d, units %d, first %d, step %d\\n", rows, units, first, i);
                        return 1;
                    }
                    at.advance();
                }
            }
        }
    }
    for (int s : {128, 256, 1024}) {
        for (int k = limit - 9 * s; k < limit; ++k) {
            const bool inside = k + 7ll * s < limit;
            if (ckl::detail::eight_steps_inside(k, s, limit) != inside || (inside && k + 8ll * s > 0x7fffffffll)) return 2;
        }
        for (int k = 0; k < 9 * s; ++k) {
            for (int n : {1, 7, s, 8 * s}) if (ckl::detail::eight_steps_inside(k, s, n) != (k + 7 * s < n)) return 3;
        }
    }
    return 0;
}
""")
