"""Products whose weight is chosen per row (ckl_gemm_grouped, its weight gradient, low-rank
adapters) against plain 64-bit sums on the same inputs.

Tolerances, element by element.  The tensor cores add products into an FP32 accumulator that is
truncated, so each of at most k additions is off by at most 2^-23 of the partial sum, which
sum |a||b| bounds: ACC = k * 2^-23 * (|A| |B|).  The result is rounded once, by at most half a
step: eps/2 of its value.  beta * C and alpha each add one FP32 rounding, covered by a further 2^-22.
The intermediate of the adapters is kept as two operand-type values: off by 2^-16 (BF16) or 2^-22
(FP16, plus its smallest step) of its value.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TWO_PART = {"f16": 2.0 ** -22, "bf16": 2.0 ** -16}


def code(ckl, name):
    return {"f16": ckl.F16, "bf16": ckl.BF16, "f32": ckl.F32}[name]


@pytest.fixture(autouse=True)
def device_healthy(ckl):
    if not torch.cuda.is_available():
        pytest.fail("tests marked gpu need a CUDA device")
    yield
    ckl.device_status()


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def offsets_of(sizes, start=0):
    o = [start]
    for s in sizes:
        o.append(o[-1] + s)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def check(got, ref, absolute, steps, out, extra=0.0):
    """absolute = sum |a||b| of the element, steps = additions behind it."""
    tol = steps * 2.0 ** -23 * absolute + (HALF_STEP[out] + 2.0 ** -22) * ref.abs() + extra
    if out == "f16":
        tol = tol + 2.0 ** -25  # half the smallest step of a subnormal result
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.3g} times the tolerance"


SIZES = {
    "ragged": [0, 1, 5, 127, 128, 129, 300, 0],
    "single_rows": [1] * 9,
    "one": [77],
    "empty": [0, 0, 0],
    "long": [700, 3],
}


@pytest.mark.parametrize("sizes", SIZES, ids=list(SIZES))
@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
def test_grouped_sizes(ckl, sizes, trans, gather):
    sizes = SIZES[sizes]
    n, k, tail, tokens = 200, 328, 3, 50
    offs = offsets_of(sizes)
    kept = int(offs[-1])
    rows = kept + tail
    a = rand((tokens if gather else rows, k), torch.bfloat16, 1)
    idx = torch.randint(0, tokens, (rows,), device="cuda", dtype=torch.int32) if gather else None
    b = rand((len(sizes), n, k) if trans else (len(sizes), k, n), torch.bfloat16, 2, k ** -0.5)
    c = torch.full((rows, n), 7.25, dtype=torch.bfloat16, device="cuda")
    ckl.gemm_grouped(ckl.BF16, a, b, c, ckl.BF16, offs, len(sizes), rows, n, k, a_rows=idx,
                     a_count=tokens if gather else None, trans_b=trans)
    torch.cuda.synchronize()
    assert (c[kept:] == 7.25).all()  # rows behind the last group stay as they were
    src = a[idx.long()] if gather else a
    o = offs.tolist()
    for g in range(len(sizes)):
        x = src[o[g]:o[g + 1]].double()
        w = (b[g].t() if trans else b[g]).double()
        check(c[o[g]:o[g + 1]], x @ w, x.abs() @ w.abs(), k, "bf16")


@pytest.mark.parametrize("ab,out", [("f16", "f16"), ("f16", "f32"), ("bf16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("n,k", [(1, 8), (17, 8), (64, 64), (65, 130), (257, 1), (1000, 72), (520, 1500)])
def test_grouped_types_and_odd_sizes(ckl, ab, out, n, k):
    sizes = [130, 0, 6]
    offs, rows = offsets_of(sizes), 136
    lda, ldb, ldc = (k + 7) // 8 * 8 + 8, (n + 7) // 8 * 8, n + 3
    a = rand((rows, lda), DT[ab], 3)
    b = rand((3, k, ldb), DT[ab], 4, k ** -0.5)
    c = rand((rows, ldc), DT[out], 5)
    c0 = c.clone()
    alpha, beta = 1.25, 0.5
    ckl.gemm_grouped(code(ckl, ab), a, b, c, code(ckl, out), offs, 3, rows, n, k, lda=lda, ldb=ldb, ldc=ldc,
                     stride_b=k * ldb, alpha=alpha, beta=beta)
    torch.cuda.synchronize()
    assert torch.equal(c[:, n:], c0[:, n:])
    o = offs.tolist()
    for g in range(3):
        x, w = a[o[g]:o[g + 1], :k].double(), b[g, :, :n].double()
        old = beta * c0[o[g]:o[g + 1], :n].double()
        check(c[o[g]:o[g + 1], :n], alpha * (x @ w) + old, alpha * (x.abs() @ w.abs()) + old.abs(), k + 2, out)


def test_grouped_wide_tiles_and_many_groups(ckl):
    """Enough tiles for 256 columns, and more groups than lanes in a warp."""
    g = torch.Generator(device="cuda").manual_seed(11)
    counts = torch.randint(0, 260, (100,), generator=g, device="cuda")
    offs = torch.zeros(101, dtype=torch.int32, device="cuda")
    offs[1:] = torch.cumsum(counts, 0)
    rows, n, k = int(offs[-1]), 640, 192
    a, b = rand((rows, k), torch.float16, 12), rand((100, k, n), torch.float16, 13, k ** -0.5)
    c = torch.empty(rows, n, dtype=torch.float32, device="cuda")
    ckl.gemm_grouped(ckl.F16, a, b, c, ckl.F32, offs, 100, rows, n, k)
    torch.cuda.synchronize()
    w = b.double()[torch.repeat_interleave(torch.arange(100, device="cuda"), counts)]
    ref = torch.einsum("rk,rkn->rn", a.double(), w)
    check(c, ref, torch.einsum("rk,rkn->rn", a.double().abs(), w.abs()), k, "f32")


def test_grouped_masked_rows_and_neighbours(ckl):
    """An index outside A reads zeros; NaN in rows of one group does not reach the others."""
    offs = offsets_of([3, 4])
    a = rand((6, 64), torch.bfloat16, 1)
    a[5] = float("nan")
    idx = torch.tensor([0, -1, 6, 5, 1, 2, 2147483647], dtype=torch.int32, device="cuda")
    b = rand((2, 64, 64), torch.bfloat16, 2, 0.125)
    c = torch.full((7, 64), float("nan"), device="cuda")
    ckl.gemm_grouped(ckl.BF16, a, b, c, ckl.F32, offs, 2, 7, 64, 64, a_rows=idx, a_count=6)
    torch.cuda.synchronize()
    assert (c[[1, 2, 6]] == 0).all() and torch.isnan(c[3]).all()
    for row, src, g in ((0, 0, 0), (4, 1, 1), (5, 2, 1)):
        x, w = a[src:src + 1].double(), b[g].double()
        check(c[row:row + 1], x @ w, x.abs() @ w.abs(), 64, "f32")


def test_grouped_without_k_and_partial_cover(ckl):
    """k = 0 scales C; one group that starts and ends inside the rows leaves the others alone."""
    offs = torch.tensor([2, 5], dtype=torch.int32, device="cuda")
    c = rand((9, 40), torch.float32, 1)
    c0 = c.clone()
    ckl.gemm_grouped(ckl.F16, None, None, c, ckl.F32, offs, 1, 9, 40, 0, beta=0.5)
    assert torch.equal(c[2:5], 0.5 * c0[2:5])
    assert torch.equal(c[:2], c0[:2]) and torch.equal(c[5:], c0[5:])
    a, b = rand((9, 72), torch.float16, 2), rand((1, 72, 40), torch.float16, 3)
    ckl.gemm_grouped(ckl.F16, a, b, c, ckl.F32, offs, 1, 9, 40, 72)
    assert torch.equal(c[:2], c0[:2]) and torch.equal(c[5:], c0[5:])
    x, w = a[2:5].double(), b[0].double()
    check(c[2:5], x @ w, x.abs() @ w.abs(), 72, "f32")


@pytest.mark.parametrize("sizes", SIZES, ids=list(SIZES))
@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_weight_gradient(ckl, sizes, gather, out):
    sizes = SIZES[sizes]
    m, n, tokens = 136, 328, 40
    offs = offsets_of(sizes)
    rows = int(offs[-1]) + 2
    a = rand((tokens if gather else rows, m), torch.bfloat16, 1)
    idx = torch.randint(0, tokens, (rows,), device="cuda", dtype=torch.int32) if gather else None
    d = rand((rows, n), torch.bfloat16, 2)
    d[rows - 2:] = float("nan")  # behind the last group: never read into a sum
    w = rand((len(sizes), m, n), DT[out], 3)
    w0 = w.clone()
    ckl.gemm_grouped_wgrad(ckl.BF16, a, d, w, code(ckl, out), offs, len(sizes), rows, m, n, a_rows=idx,
                           a_count=tokens if gather else None, beta=0.25)
    torch.cuda.synchronize()
    src = a[idx.long()] if gather else a
    o = offs.tolist()
    for g in range(len(sizes)):
        x, y = src[o[g]:o[g + 1]].double(), d[o[g]:o[g + 1]].double()
        old = 0.25 * w0[g].double()
        check(w[g], x.t() @ y + old, x.abs().t() @ y.abs() + old.abs(), sizes[g] + 2, out)


def test_weight_gradient_odd_shapes(ckl):
    sizes, m, n = [65, 64, 0, 1], 37, 9
    offs, rows = offsets_of(sizes), 130
    a, d = rand((rows, 40), torch.float16, 1), rand((rows, 16), torch.float16, 2)
    w = torch.full((4, m, n + 1), 3.0, device="cuda")
    ckl.gemm_grouped_wgrad(ckl.F16, a, d, w, ckl.F32, offs, 4, rows, m, n, lda=40, ldg=16, lddw=n + 1, alpha=0.5)
    torch.cuda.synchronize()
    assert (w[:, :, n] == 3.0).all()
    o = offs.tolist()
    for g in range(4):
        x, y = a[o[g]:o[g + 1], :m].double(), d[o[g]:o[g + 1], :n].double()
        check(w[g, :, :n], 0.5 * (x.t() @ y), 0.5 * (x.abs().t() @ y.abs()), sizes[g], "f32")


def plan(ckl, ids, groups, per_row=1):
    slots = ids.numel()
    offs = torch.empty(groups + 1, dtype=torch.int32, device="cuda")
    rows = torch.empty(slots, dtype=torch.int32, device="cuda")
    pos = torch.empty(slots, dtype=torch.int32, device="cuda")
    ckl.group_rows(ids, slots, groups, offs, rows, pos, slots_per_row=per_row)
    return offs, rows, pos


def lora_case(ckl, ids, g, k, n, r, dt, seed=0):
    m = ids.numel()
    x = rand((m, k), DT[dt], seed + 1)
    w = rand((k, n), DT[dt], seed + 2, k ** -0.5)
    a = rand((g, k, r), DT[dt], seed + 3, k ** -0.5)
    b = rand((g, r, n), DT[dt], seed + 4, r ** -0.5)
    s = 0.5 + torch.rand(g, device="cuda")
    offs, rows, _ = plan(ckl, ids, g)
    return m, x, w, a, b, s, offs, rows


def adapter_ids(kind, g):
    gen = torch.Generator().manual_seed(3)
    if kind == "one_row":
        ids = [0]
    elif kind == "none":
        ids = [-1] * 5
    elif kind == "each_its_own":
        ids = list(range(g))
    elif kind == "one_adapter":
        ids = [g - 1] * 300
    else:
        ids = torch.randint(-1, g, (333,), generator=gen).tolist()
    return torch.tensor(ids, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", ["one_row", "none", "each_its_own", "one_adapter", "mixed"])
@pytest.mark.parametrize("dt,out,r", [("bf16", "bf16", 16), ("f16", "f32", 8), ("bf16", "f32", 72), ("f16", "f16", 128)])
def test_lora(ckl, kind, dt, out, r):
    g, k, n = 7, 264, 328
    ids = adapter_ids(kind, g)
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, dt)
    y = rand((m, n + 8), DT[out], 9)
    y0 = y.clone()
    size = ckl.gemm_lora_workspace_bytes(m, r)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    beta = 0.5
    ckl.gemm_lora(code(ckl, dt), x, w, a, b, s, y, code(ckl, out), offs, rows, g, m, n, k, r, ws, size, ldy=n + 8,
                  beta=beta)
    torch.cuda.synchronize()
    assert torch.equal(y[:, n:], y0[:, n:])
    for i in range(-1, g):
        sel = ids == i
        xs, old = x[sel].double(), beta * y0[sel][:, :n].double()
        ref, mag = xs @ w.double() + old, xs.abs() @ w.double().abs() + old.abs()
        steps, extra = k + 2, 0.0
        if i >= 0:
            f = s[i].double()
            t, ta = f * (xs @ a[i].double()), f * (xs.abs() @ a[i].double().abs())
            ref, mag = ref + t @ b[i].double(), mag + ta @ b[i].double().abs()
            floor = 2.0 ** -25 * r * b[i].double().abs().max() if dt == "f16" else 0.0
            extra = TWO_PART[dt] * (t.abs() @ b[i].double().abs()) + floor
            steps += k + 2 * r
        check(y[sel][:, :n], ref, mag, steps, out, extra)


@pytest.mark.parametrize("kind", ["one_row", "none", "each_its_own", "mixed"])
@pytest.mark.parametrize("dt,out,r", [("bf16", "f32", 16), ("f16", "f16", 40), ("bf16", "bf16", 128)])
def test_lora_gradients(ckl, kind, dt, out, r):
    g, k, n = 5, 264, 200
    ids = adapter_ids(kind, g)
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, dt, 20)
    dy = rand((m, n), DT[dt], 30)
    dx = torch.full((m, k), float("nan"), dtype=DT[out], device="cuda")
    da, db = rand((g, k, r), DT[out], 31), rand((g, r, n), DT[out], 32)
    da0, db0 = da.clone(), db.clone()
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    ckl.gemm_lora_backward(code(ckl, dt), dy, x, w, a, b, s, dx, code(ckl, out), da, db, code(ckl, out), offs, rows, g,
                           m, n, k, r, ws, size, beta=1.0)
    torch.cuda.synchronize()
    for i in range(-1, g):
        sel = ids == i
        ys, xs = dy[sel].double(), x[sel].double()
        ref, mag, steps, extra = ys @ w.double().t(), ys.abs() @ w.double().abs().t(), n, 0.0
        if i >= 0:
            f, aa, bb = s[i].double(), a[i].double(), b[i].double()
            two = TWO_PART[dt]
            tiny = 2.0 ** -25 if dt == "f16" else 0.0
            u, um = f * (ys @ bb.t()), f * (ys.abs() @ bb.abs().t())
            t, tm = f * (xs @ aa), f * (xs.abs() @ aa.abs())
            ref, mag, steps = ref + u @ aa.t(), mag + um @ aa.abs().t(), 2 * n + 2 * r
            extra = two * (u.abs() @ aa.abs().t()) + tiny * r * aa.abs().max()
            count = int(sel.sum())
            check(da[i], xs.t() @ u + da0[i].double(), xs.abs().t() @ um + da0[i].double().abs(),
                  n + 2 * count + 2, out, two * (xs.abs().t() @ u.abs()) + tiny * xs.abs().sum(0).unsqueeze(1))
            check(db[i], t.t() @ ys + db0[i].double(), tm.t() @ ys.abs() + db0[i].double().abs(),
                  k + 2 * count + 2, out, two * (t.abs().t() @ ys.abs()) + tiny * ys.abs().sum(0).unsqueeze(0))
        check(dx[sel], ref, mag, steps, out, extra)


def test_lora_gradients_against_differences(ckl):
    """The loss <y, r> is linear in each of x, A and B: a central difference along a direction is the
    gradient's product with it, up to the FP32 outputs' own error."""
    g, k, n, r = 3, 64, 72, 16
    ids = torch.tensor([0, 2, 2, -1, 0, 2], dtype=torch.int32, device="cuda")
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "f16", 40)
    dy = rand((m, n), torch.float16, 44)
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def loss(x, a, b):
        y = torch.empty(m, n, device="cuda")
        ckl.gemm_lora(ckl.F16, x, w, a, b, s, y, ckl.F32, offs, rows, g, m, n, k, r, ws, size)
        return (y.double() * dy.double()).sum().item()

    dx, da, db = (torch.empty(t.shape, device="cuda") for t in (x, a, b))
    ckl.gemm_lora_backward(ckl.F16, dy, x, w, a, b, s, dx, ckl.F32, da, db, ckl.F32, offs, rows, g, m, n, k, r, ws,
                           size)
    for which, grad in ((0, dx), (1, da), (2, db)):
        args = [x, a, b]
        step = (torch.randint(0, 2, args[which].shape, device="cuda") * 2 - 1).half() * 0.25
        hi, lo = list(args), list(args)
        hi[which], lo[which] = args[which] + step, args[which] - step
        moved = (hi[which].double() - lo[which].double())  # the step after FP16 rounding
        want = (grad.double() * moved).sum().item()
        scale = (grad.double().abs() * moved.abs()).sum().item()
        assert abs(loss(*hi) - loss(*lo) - want) <= 1e-4 * scale


def test_lora_optional_outputs_and_defaults(ckl):
    g, k, n, r, m = 2, 64, 64, 16, 4
    ids = torch.tensor([1, 1, 0, -1], dtype=torch.int32, device="cuda")
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "bf16", 50)
    dy = rand((m, n), torch.bfloat16, 51)
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    args = (offs, rows, g, m, n, k, r, ws, size)
    whole = [torch.empty(t.shape, device="cuda") for t in (x, a, b)]
    ckl.gemm_lora_backward(ckl.BF16, dy, x, w, a, b, None, whole[0], ckl.F32, whole[1], whole[2], ckl.F32, *args)
    for i in range(3):
        part = [None, None, None]
        part[i] = torch.empty_like(whole[i])
        ckl.gemm_lora_backward(ckl.BF16, dy, x, w, a, b, None, part[0], ckl.F32, part[1], part[2], ckl.F32, *args)
        assert torch.equal(part[i], whole[i])
    # rows in adapter order need no permutation
    order = rows.long()
    y = [torch.empty(m, n, device="cuda") for _ in range(2)]
    ckl.gemm_lora(ckl.BF16, x, w, a, b, None, y[0], ckl.F32, *args)
    ckl.gemm_lora(ckl.BF16, x[order].contiguous(), w, a, b, None, y[1], ckl.F32, offs, None, *args[2:])
    assert torch.equal(y[0][order], y[1])


def test_wait_that_runs_out_is_reported(ckl):
    offs = offsets_of([5])
    a, b = rand((5, 128), torch.bfloat16, 1), rand((1, 128, 64), torch.bfloat16, 2)
    c = torch.zeros(5, 64, device="cuda")
    ckl.arm_wait_fault(1, 50_000_000)
    ckl.gemm_grouped(ckl.BF16, a, b, c, ckl.F32, offs, 1, 5, 64, 128)
    with pytest.raises(ckl.CklError) as e:
        ckl.device_status()
    assert e.value.status == ckl.ERR_DEVICE
    ckl.gemm_grouped(ckl.BF16, a, b, c, ckl.F32, offs, 1, 5, 64, 128)
    torch.cuda.synchronize()
    check(c, a.double() @ b[0].double(), a.double().abs() @ b[0].double().abs(), 128, "f32")


@pytest.mark.parametrize("n,k", [(200, 1000), (64, 4096), (24, 2056)])
@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
def test_grouped_few_tiles_share_the_sum(ckl, n, k, trans, gather):
    """Few tiles and a long sum: clusters of CTAs divide the sum, and the parts meet."""
    for sizes in ([1, 0, 3, 40], [140], [2]):
        offs = offsets_of(sizes)
        rows = int(offs[-1])
        a = rand((rows, k), DT["f16"], 1)
        idx = torch.randperm(rows, device="cuda").int() if gather else None
        b = rand((len(sizes), n, k) if trans else (len(sizes), k, n), DT["f16"], 2, k ** -0.5)
        c = rand((rows + 1, n), torch.float32, 3)
        c0 = c.clone()
        ckl.gemm_grouped(ckl.F16, a, b, c, ckl.F32, offs, len(sizes), rows, n, k, a_rows=idx,
                         a_count=rows if gather else None, trans_b=trans, alpha=0.5, beta=2.0)
        torch.cuda.synchronize()
        assert torch.equal(c[rows:], c0[rows:])
        src = a[idx.long()] if gather else a
        o = offs.tolist()
        for g in range(len(sizes)):
            x, w = src[o[g]:o[g + 1]].double(), (b[g].t() if trans else b[g]).double()
            old = 2.0 * c0[o[g]:o[g + 1]].double()
            check(c[o[g]:o[g + 1]], 0.5 * (x @ w) + old, 0.5 * (x.abs() @ w.abs()) + old.abs(), k + 10, "f32")


@pytest.mark.parametrize("m,n", [(37, 9), (128, 200)])
def test_weight_gradient_few_tiles_share_the_sum(ckl, m, n):
    sizes = [1500, 0, 701]
    offs, rows = offsets_of(sizes), 2201
    lda, ldd = (m + 7) // 8 * 8, (n + 7) // 8 * 8
    a, d = rand((rows, lda), torch.bfloat16, 1), rand((rows, ldd), torch.bfloat16, 2)
    w = rand((3, m, n), torch.float32, 3)
    w0 = w.clone()
    ckl.gemm_grouped_wgrad(ckl.BF16, a, d, w, ckl.F32, offs, 3, rows, m, n, lda=lda, ldg=ldd, beta=1.0)
    torch.cuda.synchronize()
    o = offs.tolist()
    for g in range(3):
        x, y = a[o[g]:o[g + 1], :m].double(), d[o[g]:o[g + 1], :n].double()
        check(w[g], x.t() @ y + w0[g].double(), x.abs().t() @ y.abs() + w0[g].double().abs(), sizes[g] + 10, "f32")


@pytest.mark.parametrize("m,g", [(1, 1), (48, 24), (200, 3)])
def test_lora_few_rows(ckl, m, g):
    """Serving sizes: a long k, so that both products are divided over clusters."""
    k, n, r = 2048, 520, 16
    gen = torch.Generator(device="cuda").manual_seed(m)
    ids = torch.randint(-1, g, (m,), generator=gen, device="cuda", dtype=torch.int32)
    ids[0] = 0
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "bf16", 60)
    size = ckl.gemm_lora_workspace_bytes(m, r)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN in every 16-bit type
    y = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    ckl.gemm_lora(ckl.BF16, x, w, a, b, s, y, ckl.BF16, offs, rows, g, m, n, k, r, ws, size)
    torch.cuda.synchronize()
    for i in range(-1, g):
        sel = ids == i
        xs = x[sel].double()
        ref, mag, extra = xs @ w.double(), xs.abs() @ w.double().abs(), 0.0
        if i >= 0:
            t, ta = s[i].double() * (xs @ a[i].double()), s[i].double() * (xs.abs() @ a[i].double().abs())
            ref, mag = ref + t @ b[i].double(), mag + ta @ b[i].double().abs()
            extra = TWO_PART["bf16"] * (t.abs() @ b[i].double().abs())
        check(y[sel], ref, mag, 2 * k + 2 * r + 10, "bf16", extra)


def many_groups(seed, count, most):
    g = torch.Generator().manual_seed(seed)
    sizes = torch.randint(0, most, (count,), generator=g)
    sizes[::7] = 0
    sizes[1], sizes[2], sizes[3] = 1, 256, 257
    return sizes.tolist()


@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
@pytest.mark.parametrize("out,beta,ldc,k", [("bf16", 0.0, 264, 136), ("f32", 0.0, 264, 72), ("f32", 0.5, 265, 72),
                                            ("f16", 0.0, 267, 13)])
def test_grouped_pairs(ckl, trans, gather, out, beta, ldc, k):
    """Tiles enough for CTA pairs: ragged groups from none to two tiles, edges in every direction."""
    sizes, n = many_groups(5, 60, 600), 264
    offs = offsets_of(sizes)
    kept, tokens = int(offs[-1]), 333
    rows, lda, ldb = kept + 5, (k + 7) // 8 * 8, (k + 7) // 8 * 8 if trans else n
    a = rand((tokens if gather else rows, lda), torch.bfloat16, 1)
    if not gather:
        a[kept:] = float("nan")
    idx = torch.randint(-1, tokens, (rows,), device="cuda", dtype=torch.int32) if gather else None
    b = rand((60, n, ldb) if trans else (60, k, ldb), torch.bfloat16, 2, k ** -0.5)
    c = rand((rows, ldc), DT[out], 3)
    c0 = c.clone()
    ckl.gemm_grouped(ckl.BF16, a, b, c, code(ckl, out), offs, 60, rows, n, k, lda=lda, ldb=ldb, ldc=ldc,
                     stride_b=b.stride(0), a_rows=idx, a_count=tokens if gather else None, trans_b=trans, alpha=1.5,
                     beta=beta)
    torch.cuda.synchronize()
    assert torch.equal(c[kept:], c0[kept:]) and torch.equal(c[:, n:], c0[:, n:])
    src = a[:, :k].double()
    if gather:
        src = torch.where((idx >= 0).unsqueeze(1), src[idx.long().clamp(min=0)], 0.0)
    o = offs.tolist()
    for g in range(60):
        x, w = src[o[g]:o[g + 1]], (b[g, :, :k].t() if trans else b[g]).double()
        old = beta * c0[o[g]:o[g + 1], :n].double()
        check(c[o[g]:o[g + 1], :n], 1.5 * (x @ w) + old, 1.5 * (x.abs() @ w.abs()) + old.abs(), k + 2, out)


@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
@pytest.mark.parametrize("out,beta,m,n", [("bf16", 0.0, 264, 264), ("f32", 0.0, 133, 520), ("f32", 1.0, 392, 131),
                                          ("f16", 0.0, 600, 200)])
def test_weight_gradient_pairs(ckl, gather, out, beta, m, n):
    sizes = many_groups(6, 50, 200)
    offs = offsets_of(sizes)
    kept, tokens = int(offs[-1]), 300
    rows, lda, ldg = kept + 3, (m + 7) // 8 * 8, (n + 7) // 8 * 8
    a = rand((tokens if gather else rows, lda), torch.float16, 1)
    idx = torch.randint(-1, tokens, (rows,), device="cuda", dtype=torch.int32) if gather else None
    d = rand((rows, ldg), torch.float16, 2)
    d[kept:] = float("nan")
    w = rand((50, m, n), DT[out], 3)
    w0 = w.clone()
    ckl.gemm_grouped_wgrad(ckl.F16, a, d, w, code(ckl, out), offs, 50, rows, m, n, lda=lda, ldg=ldg, a_rows=idx,
                           a_count=tokens if gather else None, alpha=0.5, beta=beta)
    torch.cuda.synchronize()
    src = a[:, :m].double()
    if gather:
        src = torch.where((idx >= 0).unsqueeze(1), src[idx.long().clamp(min=0)], 0.0)
    o = offs.tolist()
    for g in range(50):
        x, y, old = src[o[g]:o[g + 1]], d[o[g]:o[g + 1], :n].double(), beta * w0[g].double()
        check(w[g], 0.5 * (x.t() @ y) + old, 0.5 * (x.abs().t() @ y.abs()) + old.abs(), sizes[g] + 2, out)


@pytest.mark.parametrize("trans", [False, True], ids=["forward", "dx"])
@pytest.mark.parametrize("r", [8, 72])
def test_lora_pairs(ckl, trans, r):
    """A prefill batch: adapters begin and end inside the tiles, and one tile holds many of them."""
    m, g, k, n = 2701, 90, 200, 1032
    if trans:
        k, n = n, k
    gen = torch.Generator(device="cuda").manual_seed(r)
    ids = torch.randint(-1, g, (m,), generator=gen, device="cuda", dtype=torch.int32)
    ids[:900] = 3
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "f16", 70)
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    dy = rand((m, n), torch.float16, 80)
    out = torch.full((m, k if trans else n), float("nan"), device="cuda")
    if trans:
        ckl.gemm_lora_backward(ckl.F16, dy, x, w, a, b, s, out, ckl.F32, None, None, ckl.F32, offs, rows, g, m, n, k, r,
                               ws, size)
    else:
        ckl.gemm_lora(ckl.F16, x, w, a, b, s, out, ckl.F32, offs, rows, g, m, n, k, r, ws, size)
    torch.cuda.synchronize()
    for i in range(-1, g):
        sel = ids == i
        v, ww = (dy[sel], w.t()) if trans else (x[sel], w)
        v, ww = v.double(), ww.double()
        ref, mag, extra = v @ ww, v.abs() @ ww.abs(), 0.0
        if i >= 0:
            p1, p2 = (b[i].t(), a[i].t()) if trans else (a[i], b[i])
            t = s[i].double() * (v @ p1.double())
            ta = s[i].double() * (v.abs() @ p1.double().abs())
            ref, mag = ref + t @ p2.double(), mag + ta @ p2.double().abs()
            extra = TWO_PART["f16"] * (t.abs() @ p2.double().abs()) + 2.0 ** -25 * r * p2.double().abs().max()
        check(out[sel], ref, mag, 2 * max(k, n) + 2 * r, "f32", extra)


@pytest.mark.parametrize("r", [8, 24, 100])
@pytest.mark.parametrize("dt,out", [("f16", "f32"), ("bf16", "bf16")])
def test_lora_few_rows_ranks_and_gradients(ckl, r, dt, out):
    """As above for odd ranks, an odd n, and the gradient of x, whose adapters are read the other way."""
    m, g, k, n = 37, 9, 1032, 1041
    gen = torch.Generator(device="cuda").manual_seed(r)
    ids = torch.randint(-1, g, (m,), generator=gen, device="cuda", dtype=torch.int32)
    ldn, ldr = (n + 7) // 8 * 8, (r + 7) // 8 * 8
    x, dy = rand((m, k), DT[dt], 91), rand((m, ldn), DT[dt], 92)
    w = rand((k, ldn), DT[dt], 93, k ** -0.5)
    a, b = rand((g, k, ldr), DT[dt], 94, k ** -0.5), rand((g, r, ldn), DT[dt], 95, r ** -0.5)
    s = 0.5 + torch.rand(g, device="cuda")
    offs, rows, _ = plan(ckl, ids, g)
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    y = torch.full((m, n), float("nan"), dtype=DT[out], device="cuda")
    dx = torch.full((m, k), float("nan"), dtype=DT[out], device="cuda")
    ld = dict(ldw=ldn, ldla=ldr, ldlb=ldn)
    ckl.gemm_lora(code(ckl, dt), x, w, a, b, s, y, code(ckl, out), offs, rows, g, m, n, k, r, ws, size, **ld)
    ckl.gemm_lora_backward(code(ckl, dt), dy, x, w, a, b, s, dx, code(ckl, out), None, None, ckl.F32, offs, rows, g, m, n,
                           k, r, ws, size, lddy=ldn, **ld)
    torch.cuda.synchronize()
    tiny = 2.0 ** -25 if dt == "f16" else 0.0
    for i in range(-1, g):
        sel = ids == i
        aa, bb = a[i, :, :r].double(), b[i, :, :n].double()
        for v, ww, p1, p2, got in ((x[sel].double(), w[:, :n].double(), aa, bb, y[sel]),
                                   (dy[sel][:, :n].double(), w[:, :n].double().t(), bb.t(), aa.t(), dx[sel])):
            ref, mag, extra = v @ ww, v.abs() @ ww.abs(), 0.0
            if i >= 0:
                t, ta = s[i].double() * (v @ p1), s[i].double() * (v.abs() @ p1.abs())
                ref, mag = ref + t @ p2, mag + ta @ p2.abs()
                extra = TWO_PART[dt] * (t.abs() @ p2.abs()) + tiny * r * p2.abs().max()
            check(got, ref, mag, 2 * max(k, n) + 2 * r + 10, out, extra)


@pytest.mark.parametrize("m,g,n,k", [(40, 6, 520, 2048), (900, 5, 200, 64), (3000, 9, 1040, 72), (2000, 200, 1040, 72)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_lora_adapters_do_not_reach_each_other(ckl, m, g, n, k, bad):
    """An adapter that holds NaN or infinities, or a row of x that does, spoils its own rows only."""
    r = 16
    gen = torch.Generator(device="cuda").manual_seed(m)
    ids = torch.randint(-1, g, (m,), generator=gen, device="cuda", dtype=torch.int32)
    ids[0], ids[1], ids[2], ids[3] = 0, 1, 2, -1
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "bf16", 96)
    dy = rand((m, n), torch.bfloat16, 97)
    a[0, 3, 5], b[1, 7, 11] = bad, bad
    x[2, 4] = bad
    dy[2, 4] = bad
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    y = torch.empty(m, n, device="cuda")
    dx, da, db = torch.empty(m, k, device="cuda"), torch.empty(g, k, r, device="cuda"), torch.empty(g, r, n, device="cuda")
    ckl.gemm_lora(ckl.BF16, x, w, a, b, s, y, ckl.F32, offs, rows, g, m, n, k, r, ws, size)
    ckl.gemm_lora_backward(ckl.BF16, dy, x, w, a, b, s, dx, ckl.F32, da, db, ckl.F32, offs, rows, g, m, n, k, r, ws, size)
    torch.cuda.synchronize()
    clean = (ids != 0) & (ids != 1)
    clean[2] = False
    assert torch.isfinite(y[clean]).all() and torch.isfinite(dx[clean]).all()
    assert not torch.isfinite(y[ids == 0]).any() and not torch.isfinite(y[ids == 1][:, 11]).any()
    fine = [i for i in range(3, g)]
    assert torch.isfinite(da[fine]).all() and torch.isfinite(db[fine]).all()
    v, ww = x[clean].double(), w.double()
    t = torch.zeros(m, r, dtype=torch.float64, device="cuda")
    ref, mag = v @ ww, v.abs() @ ww.abs()
    which = ids[clean]
    for i in range(2, g):
        sel = which == i
        t = s[i].double() * (v[sel] @ a[i].double())
        ta = s[i].double() * (v[sel].abs() @ a[i].double().abs())
        ref[sel] += t @ b[i].double()
        mag[sel] += ta @ b[i].double().abs()
    check(y[clean], ref, mag, 2 * k + 2 * r + 10, "f32", TWO_PART["bf16"] * mag)


def test_gradients_without_rows(ckl):
    """An empty batch: gradients become beta times their old values, an empty workspace will do."""
    g, k, n, r = 3, 64, 520, 24
    offs = torch.zeros(g + 1, dtype=torch.int32, device="cuda")
    w, a, b = (rand(s, torch.bfloat16, 60 + i) for i, s in enumerate([(k, n), (g, k, r), (g, r, n)]))
    da, db = rand((g, k, r), torch.float32, 63), rand((g, r, n), torch.float32, 64)
    want = 0.5 * da, 0.5 * db
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    assert ckl.gemm_lora_workspace_bytes(0, r, True) == 0
    ckl.gemm_lora_backward(ckl.BF16, None, None, w, a, b, None, None, ckl.F32, da, db, ckl.F32, offs, None, g, 0, n,
                           k, r, none, 0, beta=0.5)
    assert torch.equal(da, want[0]) and torch.equal(db, want[1])
    for m in (72, 520):  # one CTA and a pair per tile
        dw = rand((40, m, n), torch.float32, 65)
        want = 0.5 * dw
        ckl.gemm_grouped_wgrad(ckl.BF16, None, None, dw, ckl.F32, torch.zeros(41, dtype=torch.int32, device="cuda"),
                               40, 0, m, n, beta=0.5)
        assert torch.equal(dw, want)
        ckl.gemm_grouped_wgrad(ckl.BF16, None, None, dw, ckl.F32, torch.zeros(41, dtype=torch.int32, device="cuda"),
                               40, 0, m, n)
        assert not dw.any()


@pytest.mark.parametrize("sizes", [(3, 0, 40), (300, 0, 2000)], ids=["few", "many"])
def test_offsets_that_pass_32_bits(ckl, sizes):
    """Matrices of a stack 2^31 + 8 elements apart, rows of A and C 2^20 and 2^21 apart."""
    n, k, far = 264, 136, 2 ** 31 + 8
    rows = sum(sizes)
    offs = offsets_of(sizes)
    stack = torch.empty(2 * far + n * k, dtype=torch.bfloat16, device="cuda")
    small = rand((3, k, n), torch.bfloat16, 70)
    for g in range(3):
        stack[g * far:g * far + k * n] = small[g].reshape(-1)
    pitch = 2 ** 21 if rows > 1000 else 2 ** 26
    a_far = torch.empty(rows * pitch, dtype=torch.bfloat16, device="cuda").view(rows, pitch)
    a = rand((rows, k), torch.bfloat16, 71)
    a_far[:, :k] = a
    back = torch.arange(rows - 1, -1, -1, dtype=torch.int32, device="cuda")
    c_far = torch.empty(rows * pitch, dtype=torch.bfloat16, device="cuda").view(rows, pitch)
    ref = torch.cat([x.double() @ w.double() for x, w in zip(a.split(sizes), small)])
    mag = torch.cat([x.double().abs() @ w.double().abs() for x, w in zip(a.split(sizes), small)])
    for idx, src in ((None, a), (back, a.flip(0))):
        a_far[:, :k] = src
        c_far[:, :n] = float("nan")
        ckl.gemm_grouped(ckl.BF16, a_far, stack, c_far, ckl.BF16, offs, 3, rows, n, k, a_rows=idx, a_count=rows,
                         lda=pitch, stride_b=far, ldc=pitch)
        check(c_far[:, :n].float(), ref, mag, k, "bf16")
    # the gradient of the weights into the same stack
    gr = rand((rows, n), torch.bfloat16, 72)
    ckl.gemm_grouped_wgrad(ckl.BF16, a_far, gr, stack, ckl.BF16, offs, 3, rows, k, n, a_rows=back, a_count=rows,
                           lda=pitch, stride_dw=far)
    at = 0
    for g, size in enumerate(sizes):
        x, d = a[at:at + size].double(), gr[at:at + size].double()
        check(stack[g * far:g * far + k * n].view(k, n).float(), x.T @ d, x.T.abs() @ d.abs(), max(size, 1), "bf16")
        at += size


def test_lora_weights_written_just_before_the_call(ckl):
    """The check for adapters that are not finite reads beside the kernel before it: it must see what the
    stream wrote last.  One adapter's weights change between finite and NaN before every call."""
    g, m, n, k, r = 9, 900, 1040, 72, 24
    ids = torch.randint(0, g, (m,), device="cuda", dtype=torch.int32,
                        generator=torch.Generator(device="cuda").manual_seed(80))
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "bf16", 81)
    size = ckl.gemm_lora_workspace_bytes(m, r)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    y = torch.empty(24, m, n, device="cuda", dtype=torch.bfloat16)
    good, bad = b[4].clone(), torch.full_like(b[4], float("nan"))
    for i in range(24):
        b[4].copy_(bad if i % 3 == 1 else good)
        ckl.gemm_lora(ckl.BF16, x, w, a, b, s, y[i], ckl.BF16, offs, rows, g, m, n, k, r, ws, size,
                      stream=torch.cuda.current_stream())
    mine = ids == 4
    for i in range(24):
        assert torch.equal(y[i][~mine], y[0][~mine])
        if i % 3 == 1:
            assert y[i][mine].isnan().all()
        else:
            assert torch.equal(y[i][mine], y[0][mine])


@pytest.mark.parametrize("trans", [False, True], ids=["nn", "nt"])
@pytest.mark.parametrize("k", [1000, 2069])
def test_grouped_pairs_long_sums(ckl, trans, k):
    """Gathered rows on CTA pairs with sums that go round the ring of stages many times and end inside a
    block; every repetition gives the same bits."""
    sizes, n, tokens = many_groups(8, 40, 500), 264, 900
    offs, rows = offsets_of(sizes), sum(sizes)
    ldk = (k + 7) // 8 * 8
    a = rand((tokens, ldk), torch.bfloat16, 1)
    idx = torch.randint(0, tokens, (rows,), device="cuda", dtype=torch.int32)
    b = rand((40, n, ldk) if trans else (40, k, n), torch.bfloat16, 2, k ** -0.5)
    c = torch.empty(20, rows, n, device="cuda")
    for out in c:
        ckl.gemm_grouped(ckl.BF16, a, b, out, ckl.F32, offs, 40, rows, n, k, lda=ldk, ldb=ldk if trans else n,
                         stride_b=b.stride(0), a_rows=idx, a_count=tokens, trans_b=trans)
    torch.cuda.synchronize()
    assert all(torch.equal(out, c[0]) for out in c)
    o = offs.tolist()
    for g in range(40):
        x, w = a[idx[o[g]:o[g + 1]].long(), :k].double(), (b[g, :, :k].t() if trans else b[g]).double()
        check(c[0, o[g]:o[g + 1]], x @ w, x.abs() @ w.abs(), k, "f32")


@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
def test_weight_gradient_pairs_long_sums(ckl, gather):
    sizes, m, n, tokens = [1500, 0, 701, 64, 3001, 2048, 63, 833] * 3, 1032, 264, 700
    offs, rows = offsets_of(sizes), sum(sizes)
    a, d = rand((tokens if gather else rows, m), torch.float16, 1), rand((rows, n), torch.float16, 2)
    idx = torch.randint(0, tokens, (rows,), device="cuda", dtype=torch.int32) if gather else None
    w = torch.empty(20, len(sizes), m, n, device="cuda")
    for out in w:
        ckl.gemm_grouped_wgrad(ckl.F16, a, d, out, ckl.F32, offs, len(sizes), rows, m, n, a_rows=idx,
                               a_count=tokens if gather else None)
    torch.cuda.synchronize()
    assert all(torch.equal(out, w[0]) for out in w)
    src, o = a[idx.long()] if gather else a, offs.tolist()
    for g, size in enumerate(sizes):
        x, y = src[o[g]:o[g + 1]].double(), d[o[g]:o[g + 1]].double()
        check(w[0, g], x.t() @ y, x.abs().t() @ y.abs(), size, "f32")


def test_lora_pairs_long_sums(ckl):
    """A prefill batch over a long k, its rows scattered, adapters of rank 72: forward and the gradient of x."""
    m, g, k, n, r = 2100, 7, 2056, 1032, 72
    gen = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(-1, g, (m,), generator=gen, device="cuda", dtype=torch.int32)
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "bf16", 130)
    dy = rand((m, n), torch.bfloat16, 135)
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    y, dx = torch.empty(10, m, n, device="cuda"), torch.empty(10, m, k, device="cuda")
    for i in range(10):
        ckl.gemm_lora(ckl.BF16, x, w, a, b, s, y[i], ckl.F32, offs, rows, g, m, n, k, r, ws, size)
        ckl.gemm_lora_backward(ckl.BF16, dy, x, w, a, b, s, dx[i], ckl.F32, None, None, ckl.F32, offs, rows, g, m, n, k,
                               r, ws, size)
    torch.cuda.synchronize()
    for i in range(10):
        assert torch.equal(y[i], y[0]) and torch.equal(dx[i], dx[0])
    for i in range(-1, g):
        sel = ids == i
        for v, ww, p1, p2, got in ((x, w, a, b, y[0]), (dy, w.t(), b.transpose(1, 2), a.transpose(1, 2), dx[0])):
            v, ww = v[sel].double(), ww.double()
            ref, mag, extra = v @ ww, v.abs() @ ww.abs(), 0.0
            if i >= 0:
                q1, q2 = p1[i].double(), p2[i].double()
                t, ta = s[i].double() * (v @ q1), s[i].double() * (v.abs() @ q1.abs())
                ref, mag = ref + t @ q2, mag + ta @ q2.abs()
                extra = TWO_PART["bf16"] * (t.abs() @ q2.abs())
            check(got[sel], ref, mag, 2 * max(k, n) + 2 * r, "f32", extra)



@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("r", [16, 24, 72])
@pytest.mark.parametrize("m,k,n", [(3, 1032, 520), (40, 2048, 520), (900, 64, 200), (3000, 72, 1040)])
def test_lora_infinite_row(ckl, dt, r, m, k, n):
    """An infinity in a row of x (of dy) under positive weights gives that row infinities, whatever the rank:
    columns that only fill up the rank to a tile's width take no part."""
    g = 3
    ids = torch.arange(m, device="cuda", dtype=torch.int32) % g
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, dt, 120)
    dy = rand((m, n), DT[dt], 125)
    x[2], dy[2] = 1.0, 1.0
    x[2, 4], dy[2, 7] = float("inf"), float("inf")
    w.abs_(), a[2].abs_(), b[2].abs_()
    for t in (w, a, b):
        t[t == 0] = 1.0
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    y, dx = torch.empty(m, n, device="cuda"), torch.empty(m, k, device="cuda")
    ckl.gemm_lora(code(ckl, dt), x, w, a, b, s, y, ckl.F32, offs, rows, g, m, n, k, r, ws, size)
    ckl.gemm_lora_backward(code(ckl, dt), dy, x, w, a, b, s, dx, ckl.F32, None, None, ckl.F32, offs, rows, g, m, n, k, r,
                           ws, size)
    torch.cuda.synchronize()
    assert (y[2] == float("inf")).all() and (dx[2] == float("inf")).all()
    others = torch.arange(m, device="cuda") != 2
    assert torch.isfinite(y[others]).all() and torch.isfinite(dx[others]).all()


@pytest.mark.parametrize("m,n", [(37, 9), (128, 200), (264, 520)])
def test_weight_gradient_ends_found_in_time(ckl, m, n):
    """Rows in place: only the last block of a group needs the loader warps, which must find it however late
    they come.  Many launches, each the same bits, none that gives up a wait."""
    sizes = [1500, 0, 701, 3001] if m < 200 else [1500, 0, 701, 1] * 12
    offs, rows = offsets_of(sizes), sum(sizes)
    lda, ldd = (m + 7) // 8 * 8, (n + 7) // 8 * 8
    a, d = rand((rows, lda), torch.bfloat16, 1), rand((rows, ldd), torch.bfloat16, 2)
    first, w = (torch.empty(len(sizes), m, n, device="cuda") for _ in range(2))
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for i in range(400):
        out = w if i else first
        ckl.gemm_grouped_wgrad(ckl.BF16, a, d, out, ckl.F32, offs, len(sizes), rows, m, n, lda=lda, ldg=ldd)
        same &= (out == first).all()
    assert bool(same)
    o = offs.tolist()
    for g in range(len(sizes)):
        x, y = a[o[g]:o[g + 1], :m].double(), d[o[g]:o[g + 1], :n].double()
        check(first[g], x.t() @ y, x.abs().t() @ y.abs(), sizes[g] + 10, "f32")


def test_grouped_pairs_half_a_tile_of_columns(ckl):
    """The last tile has columns for one CTA of the pair only, and gathered rows: the other copies nothing.
    Many launches, each the same bits, none that gives up a wait."""
    sizes, n, k, tokens = [300, 5, 256, 1000] * 10, 296, 1032, 500
    offs, rows = offsets_of(sizes), sum(sizes)
    a = rand((tokens, k), torch.float16, 1)
    idx = torch.randint(0, tokens, (rows,), device="cuda", dtype=torch.int32)
    b = rand((40, k, n), torch.float16, 2, k ** -0.5)
    first, c = (torch.empty(rows, n, device="cuda") for _ in range(2))
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for i in range(200):
        out = c if i else first
        ckl.gemm_grouped(ckl.F16, a, b, out, ckl.F32, offs, 40, rows, n, k, a_rows=idx, a_count=tokens)
        same &= (out == first).all()
    assert bool(same)
    o = offs.tolist()
    for g in range(40):
        x, w = a[idx[o[g]:o[g + 1]].long()].double(), b[g].double()
        check(first[o[g]:o[g + 1]], x @ w, x.abs() @ w.abs(), k, "f32")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_lora_rows_in_place_many_times(ckl, dt):
    """Rows already in adapter order: only the adapters' blocks pass through the loader warps.  The gradients
    have the bits that an explicit order gives."""
    g, r = 5, 24
    for m, k, n in ((300, 1032, 328), (3000, 1032, 1040)):
        ids = torch.sort(torch.randint(0, g, (m,), device="cuda", dtype=torch.int32)).values.int()
        m, x, w, a, b, s, offs, order = lora_case(ckl, ids, g, k, n, r, dt, 140)
        assert torch.equal(order, torch.arange(m, dtype=torch.int32, device="cuda"))
        size = ckl.gemm_lora_workspace_bytes(m, r, True)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        first, y = (torch.empty(m, n, device="cuda") for _ in range(2))
        same = torch.ones((), dtype=torch.bool, device="cuda")
        for i in range(200):
            out = y if i else first
            ckl.gemm_lora(code(ckl, dt), x, w, a, b, s, out, ckl.F32, offs, None, g, m, n, k, r, ws, size)
            same &= (out == first).all()
        assert bool(same)
        dy = rand((m, n), DT[dt], 145)
        grads = [[torch.empty(t.shape, device="cuda") for t in (x, a, b)] for _ in range(2)]
        for (dx, da, db), rows in zip(grads, (None, order)):
            ckl.gemm_lora_backward(code(ckl, dt), dy, x, w, a, b, s, dx, ckl.F32, da, db, ckl.F32, offs, rows, g, m, n, k,
                                   r, ws, size)
        assert all(torch.equal(p, q) for p, q in zip(*grads))
        f = s[ids.long()].double().unsqueeze(1)
        t, ta = torch.zeros(m, r, dtype=torch.float64, device="cuda"), torch.zeros(m, r, dtype=torch.float64, device="cuda")
        ref, mag = x.double() @ w.double(), x.double().abs() @ w.double().abs()
        extra = torch.zeros_like(ref)
        for i in range(g):
            sel = ids == i
            t, ta = f[sel] * (x[sel].double() @ a[i].double()), f[sel] * (x[sel].double().abs() @ a[i].double().abs())
            ref[sel] += t @ b[i].double()
            mag[sel] += ta @ b[i].double().abs()
            extra[sel] = TWO_PART[dt] * (t.abs() @ b[i].double().abs())
        check(first, ref, mag, 2 * k + 2 * r + 10, "f32", extra)



@pytest.mark.parametrize("m,g,k,n,r", [(5, 3, 40, 24, 8), (300, 4, 40, 24, 24), (3000, 6, 72, 1032, 16)],
                         ids=["few", "single", "pairs"])
@pytest.mark.parametrize("size", [1e-4, 1e-5])
def test_lora_small_values(ckl, m, g, k, n, r, size):
    """FP16 adapters early in training: the second factor is almost zero and so is what passes through it,
    far below FP16's smallest normal number, while FP32 gradients hold it.  The intermediate is two FP16
    words: the first leaves 2^-11 of a value, the second, whose last bit says in which unit the words
    are, 2^-10 of that: 2^-21 = 4 * 2^-23, which the 10 steps on top count.  The last unit is 2^-22, FP16's
    smallest step 2^-24: 2^-46 at most is left of a value that both words are too coarse for.

    Operands that are themselves subnormal: the tensor core multiplies significands as they stand and
    aligns the products by their exponent fields, and a subnormal's field is 2^-14's.  An addition is
    then off by up to 2^-23 of the sum that the same operands raised to 2^-14 would have, so that is the
    sum of absolute values that counts (zeros stay zeros)."""

    def raised(v):
        return torch.where(v == 0, 0.0, v.abs().clamp(min=2.0 ** -14))
    gen = torch.Generator(device="cuda").manual_seed(m)
    ids = torch.randint(-1, g, (m,), generator=gen, device="cuda", dtype=torch.int32)
    ids[0], ids[1] = 0, 1
    m, x, w, a, b, s, offs, rows = lora_case(ckl, ids, g, k, n, r, "f16", 110)
    w = (w * 2.0 ** -10).contiguous()
    b = rand((g, r, n), torch.float16, 111, 1e-4)
    dy = rand((m, n), torch.float16, 112, size)
    xs_small = (x.float() * size).half()  # and forward: a small T under a second factor of ordinary size
    b_big = rand((g, r, n), torch.float16, 113, 1.0)
    bytes_ = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.full((bytes_,), 255, dtype=torch.uint8, device="cuda")
    y, dx = torch.empty(m, n, device="cuda"), torch.empty(m, k, device="cuda")
    da, db = torch.empty(g, k, r, device="cuda"), torch.empty(g, r, n, device="cuda")
    small_a = rand((g, k, r), torch.float16, 114, 1e-3)
    ckl.gemm_lora(ckl.F16, xs_small, w, small_a, b_big, s, y, ckl.F32, offs, rows, g, m, n, k, r, ws, bytes_)
    ckl.gemm_lora_backward(ckl.F16, dy, xs_small, w, small_a, b, s, dx, ckl.F32, da, db, ckl.F32, offs, rows, g, m, n,
                           k, r, ws, bytes_)
    torch.cuda.synchronize()
    tiny = 2.0 ** -46
    for i in range(-1, g):
        sel = ids == i
        v, d, ww = xs_small[sel].double(), dy[sel].double(), w.double()
        ref, mag, extra = v @ ww, raised(v) @ raised(ww), 0.0
        dref, dmag, dextra = d @ ww.t(), raised(d) @ raised(ww).t(), 0.0
        if i >= 0:
            f, aa, b0, b1 = s[i].double(), small_a[i].double(), b[i].double(), b_big[i].double()
            t, ta = f * (v @ aa), f * (raised(v) @ raised(aa))
            u, ua = f * (d @ b0.t()), f * (raised(d) @ raised(b0).t())
            ref, mag, extra = ref + t @ b1, mag + ta @ raised(b1), tiny * b1.abs().sum(0)
            dref, dmag, dextra = dref + u @ aa.t(), dmag + ua @ raised(aa).t(), tiny * aa.abs().sum(1)
            count = int(sel.sum())
            check(da[i], v.t() @ u, raised(v).t() @ ua, n + 3 * count + 10, "f32", tiny * v.abs().sum(0).unsqueeze(1))
            check(db[i], t.t() @ d, ta.t() @ raised(d), k + 3 * count + 10, "f32", tiny * d.abs().sum(0).unsqueeze(0))
        check(y[sel], ref, mag, 2 * k + 3 * r + 10, "f32", extra)
        check(dx[sel], dref, dmag, 2 * n + 3 * r + 10, "f32", dextra)


@pytest.mark.parametrize("m,n", [(600, 200), (3000, 1040)], ids=["single", "pairs"])
@pytest.mark.parametrize("trans", [False, True], ids=["forward", "dx"])
def test_lora_intermediate_holds_its_digits(ckl, m, n, trans):
    """Nothing but the intermediate, in every binary order of magnitude from 2^-45 to 2^15: one rank with a 1
    behind it and no shared weights.  Left of it: 2^-21 of its value (two words, the second one with a bit
    less), 2^-46 (the last word's step), the FP32 result's own rounding, and 2^-23 of 2^-25, the least that
    the tensor core takes a word in the middle unit for: 2^-48."""
    k, r, g = 64, 24, 2
    if trans:
        k, n = n, k
    x = torch.zeros(m, n if trans else k, dtype=torch.float16, device="cuda")
    e = torch.randint(-24, 16, (m,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[:, 0] = (rand((m,), torch.float32, 2) * 2.0 ** e).clamp(-65504, 65504).half()
    x[5, 0], x[6, 0] = 0.0, 2.0 ** -14
    w = torch.zeros(k, n, dtype=torch.float16, device="cuda")
    a, b = (torch.zeros(g, *s, dtype=torch.float16, device="cuda") for s in ((k, r), (r, n)))
    small = torch.tensor([1.0, 1.375 * 2.0 ** -21], dtype=torch.float64)
    s = torch.tensor([1.0, 2.0 ** -10], device="cuda")
    first, second = (b, a) if trans else (a, b)
    second.fill_(0.0)
    for i in range(g):
        first[i, 0, 0] = small[i] * 2.0 ** 10 if i else small[i]
        if trans:
            second[i, :, 0] = 1.0
        else:
            second[i, 0] = 1.0
    ids = torch.arange(m, device="cuda", dtype=torch.int32) % g
    offs, rows, _ = plan(ckl, ids, g)
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((m, k if trans else n), float("nan"), device="cuda")
    if trans:
        ckl.gemm_lora_backward(ckl.F16, x, None, w, a, b, s, out, ckl.F32, None, None, ckl.F32, offs, rows, g, m, n, k, r,
                               ws, size)
    else:
        ckl.gemm_lora(ckl.F16, x, w, a, b, s, out, ckl.F32, offs, rows, g, m, n, k, r, ws, size)
    t = x[:, 0].double() * torch.stack([first[i, 0, 0].double() * s[i].double() for i in range(g)])[ids.long()]
    err = (out.double() - t.unsqueeze(1)).abs()
    assert (err <= (t.abs() * (2.0 ** -21 + 2.0 ** -23) + 2.0 ** -46 + 2.0 ** -48).unsqueeze(1)).all()
    assert (out[5] == 0).all()


@pytest.mark.parametrize("gather", [False, True], ids=["rows", "gather"])
def test_wait_that_runs_out_is_reported_by_pairs(ckl, gather):
    """A stage that never fills: both CTAs of every pair leave, the status says so, and the next call is right."""
    sizes, n, k = [300, 5, 256, 1000] * 10, 296, 264
    offs, rows = offsets_of(sizes), sum(sizes)
    a, b = rand((rows, k), torch.float16, 1), rand((40, k, n), torch.float16, 2, k ** -0.5)
    idx = torch.arange(rows, dtype=torch.int32, device="cuda") if gather else None
    c = torch.empty(rows, n, device="cuda")
    args = (ckl.F16, a, b, c, ckl.F32, offs, 40, rows, n, k)
    torch.cuda.synchronize()
    ckl.arm_wait_fault(1, 50_000_000)
    ckl.gemm_grouped(*args, a_rows=idx, a_count=rows)
    with pytest.raises(ckl.CklError) as e:
        ckl.device_status()
    assert e.value.status == ckl.ERR_DEVICE
    ckl.gemm_grouped(*args, a_rows=idx, a_count=rows)
    torch.cuda.synchronize()
    o = offs.tolist()
    for g in range(40):
        x, w = a[o[g]:o[g + 1]].double(), b[g].double()
        check(c[o[g]:o[g + 1]], x @ w, x.abs() @ w.abs(), k, "f32")


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [57, 62, 257, 611])
def test_columns_that_end_inside_16_bytes(ckl, out, n):
    """Results in a wider matrix whose rows begin on 16-byte boundaries: the columns behind them stay."""
    ldn = (n + 7) // 8 * 8 + 8
    for sizes, k in (([300, 5, 64], 72), ([300, 5, 256, 1000] * 10, 136), ([40], 2048)):
        g, rows, offs = len(sizes), sum(sizes), offsets_of(sizes)
        a, b = rand((rows, k), DT["f16"], 1), rand((g, k, ldn), DT["f16"], 2, k ** -0.5)
        c = torch.full((rows, ldn), 7.0, dtype=DT[out], device="cuda")
        ckl.gemm_grouped(ckl.F16, a, b, c, code(ckl, out), offs, g, rows, n, k, ldb=ldn, ldc=ldn)
        assert (c[:, n:] == 7.0).all()
        o = offs.tolist()
        for i in range(g):
            x, w = a[o[i]:o[i + 1]].double(), b[i, :, :n].double()
            check(c[o[i]:o[i + 1], :n], x @ w, x.abs() @ w.abs(), k + 10, out)
        for m in (72, 520):
            x, d = rand((rows, m), DT["f16"], 3), rand((rows, ldn), DT["f16"], 4)
            dw = torch.full((g, m, ldn), 7.0, dtype=DT[out], device="cuda")
            ckl.gemm_grouped_wgrad(ckl.F16, x, d, dw, code(ckl, out), offs, g, rows, m, n, ldg=ldn, lddw=ldn)
            assert (dw[:, :, n:] == 7.0).all()
            for i in range(g):
                u, v = x[o[i]:o[i + 1]].double(), d[o[i]:o[i + 1], :n].double()
                check(dw[i, :, :n], u.t() @ v, u.abs().t() @ v.abs(), sizes[i] + 10, out)


@pytest.mark.parametrize("m", [5, 300, 3000])
def test_adapters_that_end_inside_16_bytes(ckl, m):
    """The same of the adapters' outputs: y, the gradient of x, and gradients of rank 13."""
    g, k, n, r = 4, 131, 611, 13
    ids = torch.arange(m, device="cuda", dtype=torch.int32) % g
    offs, rows, _ = plan(ckl, ids, g)
    ldk, ldn, ldr = 136, 616, 16
    x, w, dy = rand((m, ldk), DT["bf16"], 1), rand((k, ldn), DT["bf16"], 2), rand((m, ldn), DT["bf16"], 3)
    a, b = rand((g, k, ldr), DT["bf16"], 4), rand((g, r, ldn), DT["bf16"], 5)
    y, dx = torch.full((m, ldn), 7.0, device="cuda"), torch.full((m, ldk), 7.0, device="cuda")
    da, db = torch.full((g, k, ldr), 7.0, device="cuda"), torch.full((g, r, ldn), 7.0, device="cuda")
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    ld = dict(ldx=ldk, ldw=ldn, ldla=ldr, ldlb=ldn)
    for order in (rows, None):
        ckl.gemm_lora(ckl.BF16, x, w, a, b, None, y, ckl.F32, offs, order, g, m, n, k, r, ws, size, ldy=ldn, **ld)
        ckl.gemm_lora_backward(ckl.BF16, dy, x, w, a, b, None, dx, ckl.F32, da, db, ckl.F32, offs, order, g, m, n, k, r, ws,
                               size, lddy=ldn, lddx=ldk, ldda=ldr, lddb=ldn, **ld)
        assert (y[:, n:] == 7.0).all() and (dx[:, k:] == 7.0).all()
        assert (da[:, :, r:] == 7.0).all() and (db[:, :, n:] == 7.0).all()
        for t, end in ((y, n), (dx, k), (da, r), (db, n)):
            assert torch.isfinite(t[..., :end]).all() and not (t[..., :end] == 7.0).all()
