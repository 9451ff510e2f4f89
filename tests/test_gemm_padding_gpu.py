"""C inside a wider matrix: columns that end inside a 16-byte unit leave their neighbours alone, in every
kernel of the dense GEMM, with and without C_in."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(autouse=True)
def device_healthy(ckl):
    if not torch.cuda.is_available():
        pytest.fail("tests marked gpu need a CUDA device")
    yield
    ckl.device_status()


def run(ckl, out, m, n, k, beta, call):
    """`call(a, b, c, m, n, k, ldb, ldc, beta)` into the middle columns of a matrix of sevens.  The tensor
    cores truncate: k additions of 2^-23 of the sum of absolute values, one rounding of the result."""
    g = torch.Generator(device="cuda").manual_seed(n)
    ldb, ldc = (n + 7) // 8 * 8, (n + 7) // 8 * 8 + 16
    a = torch.randn(m, k, generator=g, device="cuda").half()
    b = (torch.randn(k, ldb, generator=g, device="cuda") * k ** -0.5).half()
    wide = torch.full((m, ldc), 7.0, dtype=DT[out], device="cuda")
    c = wide.view(-1)[8:]  # 16 bytes on, or 32: the pitch decides
    call(a, b, c, m, n, k, ldb, ldc, beta)
    torch.cuda.synchronize()
    assert (wide[:, :8] == 7.0).all() and (wide[:, 8 + n:] == 7.0).all()
    x, w = a.double(), b[:, :n].double()
    ref, mag = x @ w + 7.0 * beta, x.abs() @ w.abs() + 7.0 * abs(beta)
    tol = (k + 4) * 2.0 ** -23 * mag + (HALF_STEP[out] + 2.0 ** -22) * ref.abs() + 2.0 ** -25
    assert ((wide[:, 8:8 + n].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("algo", ["AUTO", "UMMA_1CTA", "UMMA_2CTA", "UMMA_2CTA_WIDE", "UMMA_SK", "UMMA_2CTA_SK",
                                  "UMMA_2CTA_WIDE_SK", "UMMA_1CTA_N128", "UMMA_1CTA_N128_SK", "SIMT"])
@pytest.mark.parametrize("m,n,k,beta", [(300, 611, 264, 0.0), (130, 57, 520, 0.5), (700, 1025, 512, 1.0)])
def test_columns_behind_c_stay(ckl, out, algo, m, n, k, beta):
    if not hasattr(ckl, "ALGO_" + algo):
        pytest.skip("no such kernel")
    which = getattr(ckl, "ALGO_" + algo)

    def call(a, b, c, m, n, k, ldb, ldc, beta):
        ckl.gemm_ex(ckl.F16, a, b, c, {"f32": ckl.F32, "f16": ckl.F16, "bf16": ckl.BF16}[out], m, n, k, k, ldb, ldc, 1.0,
                    beta, which)

    run(ckl, out, m, n, k, beta, call)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_columns_behind_c_stay_without_allocation(ckl, out, beta):
    def call(a, b, c, m, n, k, ldb, ldc, beta):
        ckl.gemm_streamk_noalloc(ckl.F16, a, b, c, {"f32": ckl.F32, "bf16": ckl.BF16}[out], m, n, k, k, ldb, ldc, 1.0, beta)

    run(ckl, out, 300, 611, 1032, beta, call)


def test_columns_behind_c_stay_with_bias(ckl):
    g = torch.Generator(device="cuda").manual_seed(1)
    m, n, k, ldb, ldc = 300, 611, 264, 616, 632
    a, b = (torch.randn(*s, generator=g, device="cuda").half() for s in ((m, k), (k, ldb)))
    wide = torch.full((m, ldc), 7.0, device="cuda")
    bias = torch.full((n,), 1000.0, device="cuda")
    ckl.gemm_bias_relu_ex(ckl.F16, a, b, wide, ckl.F32, bias, m, n, k, k, ldb, ldc, 1.0)
    torch.cuda.synchronize()
    assert (wide[:, n:] == 7.0).all()
    x, w = a.double(), b[:, :n].double()
    ref, mag = (x @ w + 1000.0).clamp(min=0.0), x.abs() @ w.abs() + 1000.0
    assert ((wide[:, :n].double() - ref).abs() <= (k + 4) * 2.0 ** -23 * mag + 2.0 ** -22 * ref).all()
