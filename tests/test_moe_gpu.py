"""Routing to experts, the order of rows by group and the weighted sum back, against plain 64-bit
forms.  Whole numbers are compared exactly.  Weights and gradients are FP32 sums of a few hundred
terms with exp of CUDA's stated 2-ulp error: 1e-5 of the row's largest value holds them all
(1024 terms * 2^-24 < 1e-4 of a sum of positive terms is reached only if every rounding points
the same way; the tests use at most 256 terms, 256 * 2^-24 = 1.5e-5, halved by the tree sum)."""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def code(ckl, name):
    return {"f16": ckl.F16, "bf16": ckl.BF16, "f32": ckl.F32}[name]


@pytest.fixture(autouse=True)
def device_healthy(ckl):
    if not torch.cuda.is_available():
        pytest.fail("tests marked gpu need a CUDA device")
    yield
    ckl.device_status()


def plain_route(logits, bias, k, score, groups, top_groups, renorm, scale):
    """Row by row in Python floats of 64 bits."""
    weights, experts = [], []
    for row in logits.double().cpu().tolist():
        e = len(row)
        row = [-math.inf if math.isnan(v) else min(v, 3.4028234663852886e38) for v in row]
        if score == "sigmoid":
            s = [0.0 if v < -700 else 1 / (1 + math.exp(-v)) for v in row]
        else:
            top = max(row)
            s = [0.0 if v == -math.inf else math.exp(v - top) for v in row]
            total = sum(s)
            s = [v / total if total else 0.0 for v in s]
        key = list(s) if bias is not None or groups > 1 else list(row)
        if bias is not None:
            key = [a + b for a, b in zip(key, bias)]
        key = [-math.inf if r == -math.inf or math.isnan(v) else v for v, r in zip(key, row)]
        if groups > 1:
            size = e // groups
            best = []
            for g in range(groups):
                two = sorted(key[g * size:(g + 1) * size], reverse=True)[:2]
                two = [v for v in two if v > -math.inf]
                best.append(sum(two) if two else -math.inf)
            keep = sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups]
            key = [v if i // size in keep else -math.inf for i, v in enumerate(key)]
        order = sorted(range(e), key=lambda i: (-key[i], i))[:k]
        chosen = [i if key[i] > -math.inf else -1 for i in order]
        w = [s[i] if i >= 0 else 0.0 for i in chosen]
        if renorm and score == "sigmoid":
            # s_i / sum s through log s = l - log(1 + e^l): the quotient exists where s itself is
            # below the smallest 64-bit number
            logs = [row[i] - math.log1p(math.exp(row[i])) if row[i] < 0 else -math.log1p(math.exp(-row[i]))
                    for i in chosen if i >= 0]
            w = [math.exp(v - max(logs)) for v in logs] + [0.0] * (len(chosen) - len(logs))
        if renorm:
            total = sum(w)
            w = [v / total if total else 0.0 for v in w]
        weights.append([v * scale for v in w])
        experts.append(chosen)
    return torch.tensor(weights, dtype=torch.float64), torch.tensor(experts, dtype=torch.int32)


def route(ckl, logits, k, score, bias=None, groups=1, top_groups=1, renorm=False, scale=1.0, ldl=None, e=None):
    t = logits.shape[0]
    e = logits.shape[1] if e is None else e
    w = torch.full((t, k), 99.0, device="cuda")
    x = torch.full((t, k), -7, dtype=torch.int32, device="cuda")
    name = {v: n for n, v in DT.items()}[logits.dtype]
    ckl.moe_route(code(ckl, name), logits, w, x, t, e, k, ldl=ldl, bias=bias,
                  score=ckl.SCORE_SOFTMAX if score == "softmax" else ckl.SCORE_SIGMOID, groups=groups,
                  top_groups=top_groups, renormalise=renorm, scale=scale)
    return w, x


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("t,e,k,groups,top_groups,bias,dt", [
    (1, 8, 2, 1, 1, False, "bf16"), (5, 1, 1, 1, 1, False, "f32"), (7, 33, 4, 1, 1, True, "f32"),
    (6, 64, 6, 8, 3, False, "f16"), (9, 160, 6, 8, 3, True, "bf16"), (3, 256, 8, 8, 4, True, "f32"),
    (4, 40, 5, 5, 2, False, "f32"), (3, 1024, 32, 32, 9, True, "f32"), (2, 1000, 32, 1, 1, False, "f16"),
    (3, 24, 3, 24, 2, True, "f32"),
])
def test_route(ckl, score, renorm, t, e, k, groups, top_groups, bias, dt):
    g = torch.Generator(device="cuda").manual_seed(e)
    logits = (torch.randn(t, e, generator=g, device="cuda") * 2).to(DT[dt])
    values = torch.randn(e, generator=g, device="cuda") * 0.1 if bias else None
    w, x = route(ckl, logits, k, score, values, groups, top_groups, renorm, 2.5)
    rw, rx = plain_route(logits, values.double().tolist() if bias else None, k, score, groups, top_groups, renorm, 2.5)
    assert torch.equal(x.cpu(), rx)
    assert ((w.cpu().double() - rw).abs() <= 1e-5 * rw.abs().amax(1, keepdim=True)).all()


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_masks_and_special_values(ckl, score, groups, top_groups):
    inf, nan = math.inf, math.nan
    low = torch.finfo(torch.float32).min
    rows = [
        [0.0] * 16,                                    # all equal: lowest indices
        [0.0, -0.0] * 8,                               # both zeros are one value
        [-inf] * 16,                                   # nothing may be chosen
        [-inf] * 13 + [1.0, -inf, 2.0],                # fewer than top_k may be
        [nan, 1.0, nan, 2.0] + [-1.0] * 12,
        [inf, 0.0, inf, 1.0] + [0.5] * 12,
        [low] * 16,
        [low] * 8 + [0.0] * 8,
        [-90.0 - i for i in range(16)],                # sigmoid scores that FP32 cannot hold apart
        [200.0 if i == 3 else -float(i) for i in range(16)],
        [float(i % 4) for i in range(16)],
    ]
    logits = torch.tensor(rows, device="cuda")
    for renorm in (False, True):
        w, x = route(ckl, logits, 4, score, None, groups, top_groups, renorm)
        rw, rx = plain_route(logits, None, 4, score, groups, top_groups, renorm, 1.0)
        assert torch.equal(x.cpu(), rx)
        assert torch.isfinite(w).all()
        assert ((w.cpu().double() - rw).abs() <= 1e-5 * rw.abs().amax(1, keepdim=True) + 1e-37).all()


def test_route_bias_masks_and_strides(ckl):
    """A bias of -inf or NaN takes an expert out; logits may be a column block of a wider matrix."""
    wide = torch.randn(6, 50, device="cuda")
    bias = torch.zeros(20, device="cuda")
    bias[3], bias[7] = -math.inf, math.nan
    logits = wide[:, 5:25]
    w = torch.empty(6, 18, device="cuda")
    x = torch.empty(6, 18, dtype=torch.int32, device="cuda")
    ckl.moe_route(ckl.F32, logits.data_ptr(), w, x, 6, 20, 18, ldl=50, bias=bias)
    rw, rx = plain_route(logits, bias.double().tolist(), 18, "softmax", 1, 1, False, 1.0)
    assert torch.equal(x.cpu(), rx) and not ((x == 3) | (x == 7)).any()
    assert ((w.cpu().double() - rw).abs() <= 1e-5).all()


def plain_weights(logits, chosen, score, renorm, scale):
    """The weights as a function of the logits, the choice held."""
    s = torch.sigmoid(logits) if score == "sigmoid" else torch.softmax(logits, 1)
    some = chosen >= 0
    w = torch.where(some, s.gather(1, chosen.long().clamp(min=0)), torch.zeros((), dtype=s.dtype, device=s.device))
    return scale * (w / w.sum(1, keepdim=True) if renorm else w)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("t,e,k,dt", [(1, 4, 1, "f32"), (5, 37, 6, "f32"), (3, 160, 8, "bf16"), (4, 250, 32, "f16")])
def test_route_backward(ckl, score, renorm, t, e, k, dt):
    g = torch.Generator(device="cuda").manual_seed(e + k)
    logits = (torch.randn(t, e, generator=g, device="cuda") * 2).to(DT[dt])
    _, chosen = route(ckl, logits, k, score)
    if k > 1:
        chosen[0, k - 1] = -1  # a place that was not filled
    dw = torch.randn(t, k, generator=g, device="cuda")
    dl = torch.full((t, e + 3), 5.0, dtype=DT[dt], device="cuda")
    ckl.moe_route_backward(code(ckl, dt), logits, chosen, dw, dl, t, e, k, ldd=e + 3,
                           score=ckl.SCORE_SOFTMAX if score == "softmax" else ckl.SCORE_SIGMOID, renormalise=renorm,
                           scale=1.5)
    x = logits.double().requires_grad_(True)
    plain_weights(x, chosen, score, renorm, 1.5).backward(dw.double())
    tol = 1e-5 * dw.double().abs().amax(1, keepdim=True) * 1.5 + (HALF_STEP[dt] + 1e-6) * x.grad.abs()
    if dt == "f16":
        tol = tol + 2.0 ** -25
    assert ((dl[:, :e].double() - x.grad).abs() <= tol).all()
    assert (dl[:, e:] == 5.0).all()
    # and against differences of the weights themselves
    step = torch.randn(t, e, generator=g, device="cuda", dtype=torch.float64)
    h = 1e-5
    up = plain_weights(logits.double() + h * step, chosen, score, renorm, 1.5)
    down = plain_weights(logits.double() - h * step, chosen, score, renorm, 1.5)
    slope = ((up - down) / (2 * h) * dw.double()).sum()
    have = (dl[:, :e].double() * step).sum()
    assert abs(slope - have) <= (tol * step.abs()).sum() + 1e-7


def test_route_backward_masked_rows(ckl):
    logits = torch.full((3, 8), -math.inf, device="cuda")
    logits[1, 2], logits[2, 5], logits[2, 6] = 1.0, math.nan, 0.5
    for score in (ckl.SCORE_SOFTMAX, ckl.SCORE_SIGMOID):
        for renorm in (False, True):
            w, x = torch.empty(3, 2, device="cuda"), torch.empty(3, 2, dtype=torch.int32, device="cuda")
            ckl.moe_route(ckl.F32, logits, w, x, 3, 8, 2, score=score, renormalise=renorm)
            assert x.tolist() == [[-1, -1], [2, -1], [6, -1]] and (w[0] == 0).all()
            dl = torch.full((3, 8), math.nan, device="cuda")
            ckl.moe_route_backward(ckl.F32, logits, x, torch.ones(3, 2, device="cuda"), dl, 3, 8, 2, score=score,
                                   renormalise=renorm)
            assert torch.isfinite(dl).all() and (dl[0] == 0).all()
            one = torch.sigmoid(torch.tensor(1.0)).item()
            want = one * (1 - one) if score == ckl.SCORE_SIGMOID and not renorm else 0.0
            assert abs(dl[1, 2].item() - want) < 1e-6


@pytest.mark.parametrize("slots,groups,per_row", [
    (0, 3, 1), (1, 1, 1), (6, 64, 6), (31, 5, 1), (1023, 1024, 3), (8192, 7, 8), (8193, 256, 8), (40000, 256, 8),
    (70001, 1, 1), (262147, 130, 4),
])
def test_group_rows(ckl, slots, groups, per_row):
    g = torch.Generator(device="cuda").manual_seed(slots)
    ids = torch.randint(-2, groups + 2, (slots,), generator=g, device="cuda", dtype=torch.int32)
    if slots > 1000:
        ids[100:900] = 0  # a run of one group
    offs = torch.full((groups + 1,), -5, dtype=torch.int32, device="cuda")
    rows = torch.full((slots + 1,), -5, dtype=torch.int32, device="cuda")
    pos = torch.full((slots + 1,), -5, dtype=torch.int32, device="cuda")
    ckl.group_rows(ids, slots, groups, offs, rows, pos, slots_per_row=per_row)
    key = torch.where((ids < 0) | (ids >= groups), groups, ids).long().cpu()
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=groups + 1)[:groups]
    want = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)])
    assert torch.equal(offs.cpu().long(), want)
    assert torch.equal(rows[:slots].cpu().long(), order // per_row)
    back = torch.empty_like(order)
    back[order] = torch.arange(slots)
    assert torch.equal(pos[:slots].cpu().long(), back)
    assert rows[slots] == -5 and pos[slots] == -5


@pytest.mark.parametrize("t,k,n,dt,out", [
    (1, 1, 1, "f32", "f32"), (3, 6, 64, "bf16", "bf16"), (5, 9, 2050, "f16", "f32"), (300, 8, 136, "f16", "f16"),
    (4, 33, 24, "f32", "bf16"), (7, 2, 7, "bf16", "f16"),
])
def test_combine_and_gradient(ckl, t, k, n, dt, out):
    g = torch.Generator(device="cuda").manual_seed(t * k + n)
    rows = t * k + 2
    y = torch.randn(rows, n, generator=g, device="cuda").to(DT[dt])
    perm = torch.randperm(rows, generator=g, device="cuda")[:t * k].int().view(t, k).contiguous()
    if k > 1:
        perm[0, 0], perm[t - 1, k - 1] = -1, rows  # two places that name no row
    w = torch.randn(t, k, generator=g, device="cuda")
    res = torch.full((t, n + 1), 3.0, dtype=DT[out], device="cuda")
    ckl.moe_combine(code(ckl, dt), y, perm, w, res, code(ckl, out), t, k, n, rows, ldo=n + 1)
    ok = (perm >= 0) & (perm < rows)
    picked = torch.where(ok.unsqueeze(2), y[perm.long().clamp(0, rows - 1)].double(), 0.0)
    terms = w.double().unsqueeze(2) * picked
    ref = terms.sum(1)
    tol = HALF_STEP[out] * ref.abs() + (k + 1) * 2.0 ** -24 * terms.abs().sum(1) + (2.0 ** -25 if out == "f16" else 0)
    assert ((res[:, :n].double() - ref).abs() <= tol).all()
    assert (res[:, n] == 3.0).all()
    dout = torch.randn(t, n, generator=g, device="cuda").to(DT[out])
    dy = torch.full((rows, n), 9.0, dtype=DT[dt], device="cuda")
    dw = torch.full((t, k), math.nan, device="cuda")
    ckl.moe_combine_backward(code(ckl, dt), y, perm, w, dout, code(ckl, out), dy, dw, t, k, n, rows)
    want = (picked * dout.double().unsqueeze(1)).sum(2)
    mag = (picked * dout.double().unsqueeze(1)).abs().sum(2)
    assert ((dw.double() - want).abs() <= (n + 2) * 2.0 ** -24 * mag).all()
    ref = torch.full((rows, n), 9.0, dtype=torch.float64, device="cuda")
    ref[perm[ok].long()] = (w.double().unsqueeze(2) * dout.double().unsqueeze(1))[ok]
    assert ((dy.double() - ref).abs() <= (HALF_STEP[dt] + 2.0 ** -23) * ref.abs() + (2.0 ** -25 if dt == "f16" else 0)).all()


@pytest.mark.parametrize("slots,per_row", [(2 ** 24 + 3001, 1), (2 ** 25 + 11, 2), (2 ** 27 + 4103, 8)])
def test_group_rows_past_row_2_24(ckl, slots, per_row):
    """Rows from 2^24 on.  Five slots of group 1 come first and end up last, so every place is known."""
    ids = torch.zeros(slots, dtype=torch.int32, device="cuda")
    ids[:5] = 1
    offs = torch.empty(3, dtype=torch.int32, device="cuda")
    rows, pos = (torch.full((slots,), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    ckl.group_rows(ids, slots, 2, offs, rows, pos, slots_per_row=per_row)
    assert offs.tolist() == [0, slots - 5, slots]
    step = 1 << 24
    for at in range(0, slots, step):
        s = torch.arange(at, min(at + step, slots), device="cuda")
        want = torch.where(s < 5, s + slots - 5, s - 5)
        assert torch.equal(pos[at:at + step].long(), want)
        slot = torch.where(s < slots - 5, s + 5, s - (slots - 5))  # the slot at position s
        assert torch.equal(rows[at:at + step].long(), slot // per_row)



@pytest.mark.parametrize("t,k,n,dt,out", [(5, 3, 64, "bf16", "bf16"), (9, 4, 7, "f32", "f16"), (300, 8, 136, "f16", "f32")])
@pytest.mark.parametrize("known", [False, True], ids=["weight_0", "kept"])
def test_combine_leaves_out_rows_that_no_group_holds(ckl, t, k, n, dt, out, known):
    """Slots of no group stand behind the groups, where y was never written.  A weight of 0 adds nothing
    there; with `kept` a weight of any size does not, and the gradients know it too."""
    g = torch.Generator(device="cuda").manual_seed(t + n)
    slots, groups = t * k, 4
    ids = torch.randint(-1, groups, (t, k), generator=g, device="cuda", dtype=torch.int32)
    ids[0] = -1  # a token of no group at all
    offs = torch.empty(groups + 1, dtype=torch.int32, device="cuda")
    rows, pos = (torch.empty(slots, dtype=torch.int32, device="cuda") for _ in range(2))
    ckl.group_rows(ids, slots, groups, offs, rows, pos, slots_per_row=k)
    kept = int(offs[-1])
    y = torch.full((slots, n), math.nan, device="cuda").to(DT[dt])
    y[:kept] = torch.randn(kept, n, generator=g, device="cuda").to(DT[dt])
    some = ids >= 0
    w = torch.randn(t, k, generator=g, device="cuda")
    if not known:
        w = torch.where(some, w, 0.0)
    end = dict(kept=offs[groups:]) if known else {}
    res = torch.full((t, n), 3.0, dtype=DT[out], device="cuda")
    ckl.moe_combine(code(ckl, dt), y, pos, w, res, code(ckl, out), t, k, n, slots, **end)
    at = pos.view(t, k).long()
    picked = torch.where(some.unsqueeze(2), y[at].double(), 0.0)
    terms = w.double().unsqueeze(2) * picked
    ref = terms.sum(1)
    tiny = 2.0 ** -25 if out == "f16" else 0.0
    assert ((res.double() - ref).abs() <= HALF_STEP[out] * ref.abs() + (k + 1) * 2.0 ** -24 * terms.abs().sum(1) + tiny).all()
    assert (res[0] == 0).all()
    if not known:
        return
    dout = torch.randn(t, n, generator=g, device="cuda").to(DT[out])
    dy = torch.full((slots, n), 9.0, dtype=DT[dt], device="cuda")
    dw = torch.full((t, k), math.nan, device="cuda")
    ckl.moe_combine_backward(code(ckl, dt), y, pos, w, dout, code(ckl, out), dy, dw, t, k, n, slots, **end)
    prod = picked * dout.double().unsqueeze(1)
    assert ((dw.double() - prod.sum(2)).abs() <= (n + 2) * 2.0 ** -24 * prod.abs().sum(2)).all()
    assert (dw[~some] == 0).all() and (dy[kept:] == 9.0).all()
    want = (w.double().unsqueeze(2) * dout.double().unsqueeze(1))[some]
    tiny = 2.0 ** -25 if dt == "f16" else 0.0
    assert ((dy[at[some]].double() - want).abs() <= (HALF_STEP[dt] + 2.0 ** -23) * want.abs() + tiny).all()
