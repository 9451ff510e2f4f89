"""The operators together as a layer of experts uses them, forward and backward, eager, captured into
graphs and on several streams."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

T, E, K, D, H = 301, 12, 3, 264, 392


@pytest.fixture(autouse=True)
def device_healthy(ckl):
    if not torch.cuda.is_available():
        pytest.fail("tests marked gpu need a CUDA device")
    yield
    ckl.device_status()


def rand(shape, seed, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


class Layer:
    """Buffers of one layer: x -> route -> first products -> relu -> second products -> combine."""

    def __init__(self, ckl, seed):
        self.ckl = ckl
        self.x, self.logits = rand((T, D), seed), rand((T, E), seed + 1, 1.5, torch.float32)
        self.w1, self.w2 = rand((E, D, H), 1, D ** -0.5), rand((E, H, D), 2, H ** -0.5)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.weights, self.experts = torch.empty(T, K, device="cuda"), torch.empty(T, K, **i32)
        self.offsets = torch.empty(E + 1, **i32)
        self.rows, self.positions = torch.empty(T * K, **i32), torch.empty(T * K, **i32)
        bf = dict(dtype=torch.bfloat16, device="cuda")
        self.h, self.y, self.out = torch.empty(T * K, H, **bf), torch.empty(T * K, D, **bf), torch.empty(T, D, **bf)
        self.dout = rand((T, D), 3)
        self.dy, self.dh, self.dxr = torch.empty_like(self.y), torch.empty_like(self.h), torch.empty(T * K, D, **bf)
        self.dweights, self.dlogits = torch.empty_like(self.weights), torch.empty_like(self.logits)
        self.dw1, self.dw2 = torch.empty(E, D, H, device="cuda"), torch.empty(E, H, D, device="cuda")

    def forward(self, stream):
        c, s = self.ckl, stream
        c.moe_route(c.F32, self.logits, self.weights, self.experts, T, E, K, renormalise=True, stream=s)
        c.group_rows(self.experts, T * K, E, self.offsets, self.rows, self.positions, slots_per_row=K, stream=s)
        c.gemm_grouped(c.BF16, self.x, self.w1, self.h, c.BF16, self.offsets, E, T * K, H, D, a_rows=self.rows,
                       a_count=T, stream=s)
        self.h.relu_()
        c.gemm_grouped(c.BF16, self.h, self.w2, self.y, c.BF16, self.offsets, E, T * K, D, H, stream=s)
        c.moe_combine(c.BF16, self.y, self.positions, self.weights, self.out, c.BF16, T, K, D, T * K, stream=s)

    def backward(self, stream):
        c, s = self.ckl, stream
        c.moe_combine_backward(c.BF16, self.y, self.positions, self.weights, self.dout, c.BF16, self.dy, self.dweights,
                               T, K, D, T * K, stream=s)
        c.gemm_grouped(c.BF16, self.dy, self.w2, self.dh, c.BF16, self.offsets, E, T * K, H, D, trans_b=True, stream=s)
        c.gemm_grouped_wgrad(c.BF16, self.h, self.dy, self.dw2, c.F32, self.offsets, E, T * K, H, D, stream=s)
        self.dh.mul_(self.h > 0)
        c.gemm_grouped(c.BF16, self.dh, self.w1, self.dxr, c.BF16, self.offsets, E, T * K, D, H, trans_b=True,
                       stream=s)
        c.gemm_grouped_wgrad(c.BF16, self.x, self.dh, self.dw1, c.F32, self.offsets, E, T * K, D, H, a_rows=self.rows,
                             a_count=T, stream=s)
        c.moe_route_backward(c.F32, self.logits, self.experts, self.dweights, self.dlogits, T, E, K, renormalise=True,
                             stream=s)

    def results(self):
        return [t.clone() for t in (self.out, self.weights, self.experts, self.positions, self.dxr, self.dw1, self.dw2,
                                    self.dlogits)]


def test_layer_against_64_bits(ckl):
    """Output and gradients against 64-bit autograd of the same choice.  Bounds, with H1 = |x||W1| and so
    on for the sums of absolute values: a bf16 rounding is 2^-8 of a value, an accumulator loses
    2^-23 per addition; the forward chain rounds h, y and out, the backward one dy, dh and dx besides,
    and a relu that flips because of a rounding moves a value by no more than that rounding."""
    s = Layer(ckl, 10)
    stream = torch.cuda.current_stream()
    s.forward(stream)
    s.backward(stream)
    torch.cuda.synchronize()
    x, w1, w2 = (t.double().requires_grad_(True) for t in (s.x, s.w1, s.w2))
    logits = s.logits.double().requires_grad_(True)
    score = torch.softmax(logits, 1).gather(1, s.experts.long())
    weight = score / score.sum(1, keepdim=True)
    e = s.experts.long().reshape(-1)
    token = torch.arange(T, device="cuda").repeat_interleave(K)
    order = torch.argsort(e, stable=True)
    assert torch.equal(s.rows.long(), token[order])
    pre = torch.zeros(T * K, H, dtype=torch.float64, device="cuda")
    y = torch.zeros(T * K, D, dtype=torch.float64, device="cuda")
    h_mag, y_mag = torch.zeros_like(pre), torch.zeros_like(y)
    for i in range(E):
        sel = (e == i).nonzero().flatten()
        pre = pre.index_add(0, sel, x[token[sel]] @ w1[i])
        h_mag.index_add_(0, sel, (x[token[sel]].abs() @ w1[i].abs()).detach())
    h = torch.relu(pre)
    for i in range(E):
        sel = (e == i).nonzero().flatten()
        y = y.index_add(0, sel, h[sel] @ w2[i])
        y_mag.index_add_(0, sel, (h_mag[sel] @ w2[i].abs()).detach())
    out = (weight.unsqueeze(2) * y.view(T, K, D)).sum(1)
    out.backward(s.dout.double())
    step = 2.0 ** -8
    mag = (weight.detach().unsqueeze(2) * y_mag.view(T, K, D)).sum(1)
    assert ((s.out.double() - out).abs() <= 3.1 * step * mag).all()
    # gradients: the same sums of absolute values, one rounding per tensor on the way
    g_mag = weight.detach().view(T * K, 1) * s.dout.double().abs()[token]
    dh_mag, dx_mag = torch.zeros_like(pre), torch.zeros(T, D, dtype=torch.float64, device="cuda")
    for i in range(E):
        sel = (e == i).nonzero().flatten()
        dh_mag[sel] = g_mag[sel] @ w2[i].detach().abs().t()
        w1_mag, w2_mag = s.x.double().abs()[token[sel]].t() @ dh_mag[sel], h_mag[sel].t() @ g_mag[sel]
        flips = 4.0  # a flipped relu takes a whole term, at most a rounding of h's magnitude away from 0
        near = (pre[sel].detach().abs() <= 2 * step * h_mag[sel]).double()
        extra = s.x.double().abs()[token[sel]].t() @ (dh_mag[sel] * near)
        assert ((s.dw2[i].double() - w2.grad[i]).abs() <= flips * step * w2_mag).all()
        assert ((s.dw1[i].double() - w1.grad[i]).abs() <= 4 * step * w1_mag + extra).all()
        dx_mag.index_add_(0, token[sel], (dh_mag[sel] * (4 * step + near)) @ w1[i].detach().abs().t())
    dx = torch.zeros(T, D, dtype=torch.float64, device="cuda")
    dx.index_add_(0, s.rows.long(), s.dxr.double())
    assert ((dx - x.grad).abs() <= dx_mag + step * dx.abs()).all()
    dw_mag = (y_mag.view(T, K, D) * s.dout.double().abs().unsqueeze(1)).sum(2)
    p = weight.detach()
    tol = 3 * step * p * (dw_mag + (dw_mag * p).sum(1, keepdim=True))
    got, want = s.dlogits.double().gather(1, s.experts.long()), logits.grad.gather(1, s.experts.long())
    assert ((got - want).abs() <= tol + 1e-6 * want.abs()).all()


def test_layer_is_deterministic_and_replays(ckl):
    """The same bits again, from a captured graph with new inputs in the same buffers too."""
    s = Layer(ckl, 20)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(2):  # first use outside the capture
            s.forward(stream)
            s.backward(stream)
    stream.synchronize()
    first = s.results()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s.forward(stream)
        s.backward(stream)
    other = Layer(ckl, 30)
    with torch.cuda.stream(stream):
        other.forward(stream)
        other.backward(stream)
    stream.synchronize()
    for seed, want in ((30, other.results()), (20, first)):
        s.x.copy_(rand((T, D), seed))
        s.logits.copy_(rand((T, E), seed + 1, 1.5, torch.float32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(s.results(), want):
            assert torch.equal(a, b)


def test_layers_on_two_streams(ckl):
    """Two layers in flight at once share nothing but the library."""
    alone = []
    for seed in (40, 50):
        s = Layer(ckl, seed)
        s.forward(torch.cuda.current_stream())
        s.backward(torch.cuda.current_stream())
        torch.cuda.synchronize()
        alone.append(s.results())
    both = [Layer(ckl, 40), Layer(ckl, 50)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, q in zip(both, streams):
            with torch.cuda.stream(q):
                s.forward(q)
                s.backward(q)
    torch.cuda.synchronize()
    for s, want in zip(both, alone):
        for a, b in zip(s.results(), want):
            assert torch.equal(a, b)


def test_adapters_in_a_graph_beside_the_dense_kernel(ckl):
    """Capture of both adapter calls between dense products of the same stream; replays with new rows
    per adapter (the order is made on the GPU, so the graph follows it)."""
    m, g, k, n, r = 300, 5, 264, 328, 16
    x, w, dy = rand((m, k), 1), rand((k, n), 2, k ** -0.5), rand((m, n), 3)
    a, b = rand((g, k, r), 4, k ** -0.5), rand((g, r, n), 5, r ** -0.5)
    scales = torch.linspace(0.5, 1.5, g, device="cuda")
    ids = torch.empty(m, dtype=torch.int32, device="cuda")
    offs = torch.empty(g + 1, dtype=torch.int32, device="cuda")
    rows, pos = (torch.empty(m, dtype=torch.int32, device="cuda") for _ in range(2))
    y, dx = torch.empty(m, n, device="cuda"), torch.empty(m, k, device="cuda")
    da, db = torch.empty(g, k, r, device="cuda"), torch.empty(g, r, n, device="cuda")
    dense = torch.empty(m, n, device="cuda")
    size = ckl.gemm_lora_workspace_bytes(m, r, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def step(s):
        ckl.gemm_ex(ckl.BF16, x, w, dense, ckl.F32, m, n, k, k, n, n, 1.0, 0.0, stream=s)
        ckl.group_rows(ids, m, g, offs, rows, pos, stream=s)
        ckl.gemm_lora(ckl.BF16, x, w, a, b, scales, y, ckl.F32, offs, rows, g, m, n, k, r, ws, size, stream=s)
        ckl.gemm_ex(ckl.BF16, x, w, dense, ckl.F32, m, n, k, k, n, n, 1.0, 1.0, stream=s)
        ckl.gemm_lora_backward(ckl.BF16, dy, x, w, a, b, scales, dx, ckl.F32, da, db, ckl.F32, offs, rows, g, m, n, k,
                               r, ws, size, stream=s)

    stream = torch.cuda.Stream()
    ids.fill_(0)
    torch.cuda.synchronize()
    step(stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(stream)
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        ids.copy_(torch.randint(-1, g, (m,), generator=gen, device="cuda", dtype=torch.int32))
        torch.cuda.synchronize()
        step(stream)
        stream.synchronize()
        want = [t.clone() for t in (y, dx, da, db, dense)]
        for t in (y, dx, da, db, dense):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for t, u in zip((y, dx, da, db, dense), want):
            assert torch.equal(t, u)



def test_layer_with_tokens_that_route_nowhere(ckl):
    """Padded tokens (every logit -inf) and tokens with fewer experts than places, in buffers that hold NaN
    from before: the same bits as in zeroed buffers, and nothing from a place that holds no expert."""
    got = []
    for old in (0.0, float("nan")):
        s = Layer(ckl, 60)
        s.logits[T - 7:] = -float("inf")
        s.logits[11, 2:] = -float("inf")  # two experts for three places
        for buf in (s.h, s.y, s.out, s.dy, s.dh, s.dxr, s.dw1, s.dw2, s.dlogits, s.weights):
            buf.fill_(old)
        s.forward(torch.cuda.current_stream())
        s.backward(torch.cuda.current_stream())
        torch.cuda.synchronize()
        kept = int(s.offsets[-1])
        assert kept == T * K - 7 * K - 1 and (s.experts[T - 7:] == -1).all() and (s.experts[11, 2:] == -1).all()
        assert (s.out[T - 7:] == 0).all() and (s.dlogits[T - 7:] == 0).all()
        got.append([s.out, s.weights, s.experts, s.positions, s.dxr[:kept], s.dw1, s.dw2, s.dlogits])
    for a, b in zip(*got):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_every_kernel_reads_what_the_one_before_it_wrote(ckl):
    """Each launch may be set up while its predecessor runs.  Ids, scores and rows change in every step of a
    long chain without a pause; each step must give what it gives alone."""
    t, k, e, n, steps = 64, 4, 8, 64, 40
    gen = torch.Generator(device="cuda").manual_seed(70)
    logits = torch.randn(steps, t, e, generator=gen, device="cuda")
    y = torch.randn(t * k, n, generator=gen, device="cuda")
    dout = torch.randn(t, n, generator=gen, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    w, experts = torch.empty(t, k, device="cuda"), torch.empty(t, k, **i32)
    offs, rows, pos = torch.empty(e + 1, **i32), torch.empty(t * k, **i32), torch.empty(t * k, **i32)
    x = torch.randn(t, n, generator=gen, device="cuda").bfloat16()
    b = torch.randn(e, n, n, generator=gen, device="cuda").bfloat16()

    def chain(pause):
        got = []
        for i in range(steps):
            out, dy, dw = torch.empty(t, n, device="cuda"), torch.empty(t * k, n, device="cuda"), torch.empty(t, k, device="cuda")
            c = torch.empty(t * k, n, device="cuda")
            s = torch.cuda.current_stream()
            ckl.moe_route(ckl.F32, logits[i], w, experts, t, e, k, stream=s)
            pause()
            ckl.group_rows(experts, t * k, e, offs, rows, pos, slots_per_row=k, stream=s)
            pause()
            ckl.moe_combine(ckl.F32, y, pos, w, out, ckl.F32, t, k, n, t * k, stream=s, kept=offs[e:])
            pause()
            ckl.moe_combine_backward(ckl.F32, y, pos, w, dout, ckl.F32, dy, dw, t, k, n, t * k, stream=s)
            pause()
            ckl.gemm_grouped(ckl.BF16, x, b, c, ckl.F32, offs, e, t * k, n, n, a_rows=rows, a_count=t, stream=s)
            pause()
            got += [out, dy, dw, c]
        torch.cuda.synchronize()
        return got

    alone = chain(torch.cuda.synchronize)
    for _ in range(3):
        for a, b_ in zip(chain(lambda: None), alone):
            assert torch.equal(a, b_)
