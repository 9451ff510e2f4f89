"""Cases for the operators that choose a weight per row: routing to experts, the experts' products,
the weighted sum that brings their rows back, and low-rank adapters beside a shared projection.

`run` computes a case either from elementary torch operations in 32 bits (the plain form) or, with
`own` set, through this repository's entry points.
"""

import importlib.util
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of one request through the router of a served model: latency alone counts
        dict(name="route_one_token", op="route", tokens=1, experts=64, top_k=6, score="softmax", bias=False,
             groups=1, top_groups=1, renorm=False, dtype="bf16", padded=0),
        # a prefill batch: sigmoid scores, balance bias, limited groups, a few padded rows at the end
        dict(name="route_prefill", op="route", tokens=8192, experts=256, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, renorm=True, dtype="f32", padded=37),
        # the router's part of a training step, odd sizes
        dict(name="route_backward", op="route_bwd", tokens=4099, experts=160, top_k=6, score="softmax", bias=False,
             groups=8, top_groups=3, renorm=False, dtype="bf16", padded=0),
        # a decode step of a small batch: few rows, each reads a whole expert
        dict(name="experts_decode", op="experts", tokens=5, experts=64, top_k=6, k=2048, n=1408, dtype="bf16"),
        # an ordinary prefill chunk
        dict(name="experts_prefill", op="experts", tokens=4096, experts=64, top_k=6, k=2048, n=1408, dtype="bf16"),
        # the largest: a full batch over many experts
        dict(name="experts_large", op="experts", tokens=8192, experts=128, top_k=8, k=4096, n=2048, dtype="f16"),
        # gradients of one expert layer in a training step
        dict(name="experts_backward", op="experts_bwd", tokens=4097, experts=32, top_k=4, k=2048, n=1536, dtype="bf16"),
        # rows back to their tokens after a prefill chunk
        dict(name="combine_prefill", op="combine", tokens=4096, experts=64, top_k=6, n=4096, dtype="bf16"),
        # and its gradient, odd token count
        dict(name="combine_backward", op="combine_bwd", tokens=2047, experts=128, top_k=8, n=2048, dtype="f16"),
        # a decode step of many requests: every row may name another adapter, some name none
        dict(name="lora_decode", op="lora", rows=48, adapters=24, rank=16, k=4096, n=4096, dtype="bf16"),
        # ragged prompts of a few requests in one prefill batch
        dict(name="lora_prefill", op="lora", rows=4100, adapters=8, rank=64, k=4096, n=4096, dtype="bf16"),
        # several adapters trained in one batch over a frozen projection
        dict(name="lora_backward", op="lora_bwd", rows=2050, adapters=4, rank=32, k=2048, n=2048, dtype="f16"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route", "route_bwd", "experts", "experts", "experts_bwd", "combine", "combine_bwd",
                     "lora", "lora", "lora_bwd"])
    half = rng.choice(["bf16", "f16"])
    if op in ("route", "route_bwd"):
        groups = rng.choice([1, 1, 4, 8])
        experts = rng.randint(2, 32) * groups if groups > 1 else rng.randint(9, 256)
        top_groups = rng.randint(max(1, groups // 2), groups)
        top_k = rng.randint(1, min(8, top_groups * (experts // groups)))
        tokens = _spread(rng, 1, 8192)
        return dict(op=op, tokens=tokens, experts=experts, top_k=top_k, score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, renorm=rng.random() < 0.5,
                    dtype=rng.choice(["f32", "bf16", "f16"]), padded=rng.choice([0, min(3, tokens - 1)]))
    if op in ("experts", "experts_bwd"):
        tokens, experts = _spread(rng, 1, 4096), _spread(rng, 8, 128)
        return dict(op=op, tokens=tokens, experts=experts, top_k=rng.randint(1, 8),
                    k=8 * _spread(rng, 32, 320), n=8 * _spread(rng, 32, 256), dtype=half)
    if op in ("combine", "combine_bwd"):
        return dict(op=op, tokens=_spread(rng, 1, 8192), experts=_spread(rng, 8, 256), top_k=rng.randint(1, 8),
                    n=8 * _spread(rng, 32, 512), dtype=half)
    rows = _spread(rng, 1, 4096)
    return dict(op=op, rows=rows, adapters=_spread(rng, 1, 32), rank=rng.choice([8, 16, 24, 32, 64, 128]),
                k=8 * _spread(rng, 64, 512), n=8 * _spread(rng, 64, 512), dtype=half)


# ---- inputs -----------------------------------------------------------------------------------


def _plan(ids, groups, per_row):
    """Positions of all slots ordered by group (slots of no group last): what a program keeps per batch."""
    slots = ids.numel()
    key = torch.where((ids < 0) | (ids >= groups), groups, ids).long()
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(groups + 1, dtype=torch.int64, device=ids.device).index_add_(
        0, key, torch.ones_like(key))
    offsets = torch.zeros(groups + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum(counts[:groups], 0)
    positions = torch.empty(slots, dtype=torch.int64, device=ids.device)
    positions[order] = torch.arange(slots, device=ids.device)
    return offsets.int(), (order // per_row).int(), positions.int(), key[order], max(1, int(counts[:groups].max()))


def _choose(gen, tokens, experts, top_k, dev):
    """top_k distinct experts per token, some asked for more often than others."""
    lean = 0.5 * torch.randn(experts, generator=gen, device=dev)
    noise = -torch.log(-torch.log(torch.rand(tokens, experts, generator=gen, device=dev).clamp(1e-9, 1 - 1e-7)))
    return torch.topk(lean + noise, top_k, dim=1).indices.int()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    s = dict(case)
    op = case["op"]
    if op in ("route", "route_bwd"):
        t, e, dt = case["tokens"], case["experts"], _DTYPES[case["dtype"]]
        s["logits"] = normal(t, e, std=1.5, dtype=dt)
        if case["padded"]:
            s["logits"][t - case["padded"]:] = -math.inf
        s["bias_values"] = normal(e, std=0.1) if case["bias"] else None
        slots = t * case["top_k"]
        s["weights"] = torch.empty(t, case["top_k"], device=dev)
        s["chosen"] = torch.empty(t, case["top_k"], dtype=torch.int32, device=dev)
        if op == "route":
            s["offsets"] = torch.empty(e + 1, dtype=torch.int32, device=dev)
            s["rows"] = torch.empty(slots, dtype=torch.int32, device=dev)
            s["positions"] = torch.empty(slots, dtype=torch.int32, device=dev)
        else:
            _, s["chosen"] = _route_plain(s)
            s["dweights"] = normal(t, case["top_k"])
            s["dlogits"] = torch.empty(t, e, dtype=dt, device=dev)
        return s
    dt = _DTYPES[case["dtype"]]
    if op in ("lora", "lora_bwd"):
        m, g, k, n, r = case["rows"], case["adapters"], case["k"], case["n"], case["rank"]
        ids = torch.randint(-1, g, (m,), generator=gen, device=dev, dtype=torch.int32)
        s["offsets"], s["order"], s["positions"], s["group"], s["cap"] = _plan(ids, g, 1)
        s["kept"] = int(s["offsets"][-1])
        s["x"] = normal(m, k, dtype=dt)
        s["w"] = normal(k, n, std=k ** -0.5, dtype=dt)
        s["a"] = normal(g, k, r, std=k ** -0.5, dtype=dt)
        s["b"] = normal(g, r, n, std=r ** -0.5, dtype=dt)
        s["scales"] = 0.5 + torch.rand(g, generator=gen, device=dev)
        words = 8 * m * (2 * r + 64) + 4096  # bytes that hold every workspace of this family
        s["workspace"] = torch.empty(words, dtype=torch.uint8, device=dev)
        if op == "lora":
            s["y"] = torch.empty(m, n, dtype=dt, device=dev)
        else:
            s["dy"] = normal(m, n, dtype=dt)
            s["dx"] = torch.empty(m, k, dtype=dt, device=dev)
            s["da"] = torch.empty(g, k, r, dtype=dt, device=dev)
            s["db"] = torch.empty(g, r, n, dtype=dt, device=dev)
        return s
    t, e, j, n = case["tokens"], case["experts"], case["top_k"], case["n"]
    rows = t * j
    ids = _choose(gen, t, e, j, dev)
    s["offsets"], s["token"], s["positions"], s["group"], s["cap"] = _plan(ids.reshape(-1), e, j)
    if op in ("experts", "experts_bwd"):
        k = case["k"]
        s["x"] = normal(t, k, dtype=dt)
        s["w"] = torch.empty(e, k, n, dtype=dt, device=dev)
        for i in range(e):
            s["w"][i] = normal(k, n, std=k ** -0.5)
        if op == "experts":
            s["y"] = torch.empty(rows, n, dtype=dt, device=dev)
        else:
            s["dy"] = normal(rows, n, dtype=dt)
            s["dx"] = torch.empty(rows, k, dtype=dt, device=dev)
            s["dw"] = torch.empty(e, k, n, dtype=dt, device=dev)
        return s
    s["y"] = normal(rows, n, dtype=dt)
    s["weights"] = torch.softmax(normal(t, j), dim=1)
    if op == "combine":
        s["out"] = torch.empty(t, n, dtype=dt, device=dev)
    else:
        s["dout"] = normal(t, n, dtype=dt)
        s["dy"] = torch.empty(rows, n, dtype=dt, device=dev)
        s["dweights"] = torch.empty(t, j, device=dev)
    return s


# ---- the plain form ---------------------------------------------------------------------------


def _scores(logits, score):
    """Scores in 64 bits: which of two nearly equal ones is larger decides whole numbers."""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    if score == "sigmoid":
        return x, 1 / (1 + torch.exp(-x))
    top = x.amax(1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(1, keepdim=True)
    return x, p / torch.where(total == 0, 1.0, total)


def _route_plain(s):
    t, e, k, groups = s["tokens"], s["experts"], s["top_k"], s["groups"]
    x, score = _scores(s["logits"], s["score"])
    if s["bias_values"] is None and groups == 1:
        key = x
    else:
        key = score if s["bias_values"] is None else score + s["bias_values"].double()
        key = torch.where(x == -math.inf, -math.inf, key)
    if groups > 1:
        best = torch.sort(key.view(t, groups, e // groups), dim=2, descending=True).values[:, :, :2]
        none = best[:, :, 0] == -math.inf
        best = torch.where(best == -math.inf, 0.0, best).sum(2)
        best = torch.where(none, -math.inf, best)
        chosen = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        keep = torch.zeros(t, groups, dtype=torch.bool, device=x.device).scatter_(1, chosen, True)
        key = torch.where(keep.repeat_interleave(e // groups, dim=1), key, -math.inf)
    value, index = torch.sort(key, dim=1, descending=True, stable=True)
    value, index = value[:, :k], index[:, :k]
    none = value == -math.inf
    w = torch.where(none, 0.0, score.gather(1, index))
    if s["renorm"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total == 0, 1.0, total)
    return w.float(), torch.where(none, -1, index).int()


def _route_backward_plain(s):
    logits = s["logits"].float()
    if s["score"] == "sigmoid":
        score = torch.sigmoid(logits)
        slope = score * torch.sigmoid(-logits)
    else:
        top = logits.amax(1, keepdim=True)
        score = torch.exp(logits - torch.where(torch.isinf(top), 0.0, top))
        total = score.sum(1, keepdim=True)
        score = score / torch.where(total == 0, 1.0, total)
    some = s["chosen"] >= 0
    index = s["chosen"].long().clamp(min=0)
    w = torch.where(some, score.gather(1, index), 0.0)
    d = torch.where(some, s["dweights"], 0.0)
    if s["renorm"]:
        total = w.sum(1, keepdim=True)
        total = torch.where(total == 0, math.inf, total)
        d = torch.where(some, (d - (d * w).sum(1, keepdim=True) / total) / total, 0.0)
    dscore = torch.zeros_like(score).scatter_add_(1, index, d)
    if s["score"] == "sigmoid":
        out = dscore * slope
    else:
        out = score * (dscore - (dscore * score).sum(1, keepdim=True))
    return out.to(s["logits"].dtype)


def _padded(values, slot, groups, cap):
    out = torch.zeros(groups * cap, values.shape[1], device=values.device)
    out[slot] = values
    return out.view(groups, cap, -1)


def _slots(s, count):
    group = s["group"][:count]
    return group * s["cap"] + torch.arange(count, device=group.device) - s["offsets"].long()[group]


def _plain(s):
    op = s["op"]
    if op == "route":
        w, chosen = _route_plain(s)
        e = s["experts"]
        flat = chosen.reshape(-1).long()
        key = torch.where(flat < 0, e, flat)
        order = torch.argsort(key, stable=True)
        offsets = torch.searchsorted(key[order].contiguous(), torch.arange(e + 1, device=key.device))
        positions = torch.empty_like(order)
        positions[order] = torch.arange(order.numel(), device=key.device)
        return [w, chosen, offsets.int(), (order // s["top_k"]).int(), positions.int()]
    if op == "route_bwd":
        return [_route_backward_plain(s)]
    if op in ("lora", "lora_bwd"):
        g, kept, cap = s["adapters"], s["kept"], s["cap"]
        rows = s["order"][:kept].long()
        slot = _slots(s, kept)
        x, a, b = s["x"].float(), s["a"].float(), s["b"].float()
        scale = s["scales"].view(g, 1, 1)
        px = _padded(x[rows], slot, g, cap)
        t = torch.bmm(px, a) * scale
        if op == "lora":
            y = x @ s["w"].float()
            y[rows] += torch.bmm(t, b).view(g * cap, -1)[slot]
            return [y.to(s["y"].dtype)]
        dy = s["dy"].float()
        pdy = _padded(dy[rows], slot, g, cap)
        u = torch.bmm(pdy, b.transpose(1, 2)) * scale
        dx = dy @ s["w"].float().t()
        dx[rows] += torch.bmm(u, a.transpose(1, 2)).view(g * cap, -1)[slot]
        da = torch.bmm(px.transpose(1, 2), u)
        db = torch.bmm(t.transpose(1, 2), pdy)
        return [dx.to(s["dx"].dtype), da.to(s["da"].dtype), db.to(s["db"].dtype)]
    rows = s["positions"].numel()
    if op in ("experts", "experts_bwd"):
        e, cap, w = s["experts"], s["cap"], s["w"].float()
        slot = _slots(s, rows)
        px = _padded(s["x"].float()[s["token"].long()], slot, e, cap)
        if op == "experts":
            return [torch.bmm(px, w).view(e * cap, -1)[slot].to(s["y"].dtype)]
        pdy = _padded(s["dy"].float(), slot, e, cap)
        dx = torch.bmm(pdy, w.transpose(1, 2)).view(e * cap, -1)[slot]
        dw = torch.bmm(px.transpose(1, 2), pdy)
        return [dx.to(s["dx"].dtype), dw.to(s["dw"].dtype)]
    t, j = s["tokens"], s["top_k"]
    y = s["y"].float()[s["positions"].long()].view(t, j, -1)
    if op == "combine":
        return [(s["weights"].unsqueeze(2) * y).sum(1).to(s["out"].dtype)]
    dout = s["dout"].float()
    dy = torch.empty(t * j, dout.shape[1], device=dout.device)
    dy[s["positions"].long()] = (s["weights"].unsqueeze(2) * dout.unsqueeze(1)).view(t * j, -1)
    return [dy.to(s["dy"].dtype), (y * dout.unsqueeze(1)).sum(2)]


# ---- through the entry points ------------------------------------------------------------------


def _package():
    """The package directory's name has a hyphen: it is imported under the name ckl_b200."""
    if "ckl_b200" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        pkg = os.path.join(root, "cuda-kernel-library_b200")
        spec = importlib.util.spec_from_file_location(
            "ckl_b200", os.path.join(pkg, "__init__.py"), submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["ckl_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["ckl_b200"]


def _own(s):
    ckl = _package()
    op = s["op"]
    code = {torch.float32: ckl.F32, torch.float16: ckl.F16, torch.bfloat16: ckl.BF16}
    stream = torch.cuda.current_stream()
    if op in ("route", "route_bwd"):
        t, e, k = s["tokens"], s["experts"], s["top_k"]
        how = dict(score=ckl.SCORE_SOFTMAX if s["score"] == "softmax" else ckl.SCORE_SIGMOID, renormalise=s["renorm"],
                   stream=stream)
        dt = code[s["logits"].dtype]
        if op == "route":
            ckl.moe_route(dt, s["logits"], s["weights"], s["chosen"], t, e, k, bias=s["bias_values"],
                          groups=s["groups"], top_groups=s["top_groups"], **how)
            ckl.group_rows(s["chosen"], t * k, e, s["offsets"], s["rows"], s["positions"], slots_per_row=k,
                           stream=stream)
            return [s["weights"], s["chosen"], s["offsets"], s["rows"], s["positions"]]
        ckl.moe_route_backward(dt, s["logits"], s["chosen"], s["dweights"], s["dlogits"], t, e, k, **how)
        return [s["dlogits"]]
    dt = code[_DTYPES[s["dtype"]]]
    if op == "lora":
        m, n, k = s["rows"], s["n"], s["k"]
        ckl.gemm_lora(dt, s["x"], s["w"], s["a"], s["b"], s["scales"], s["y"], code[s["y"].dtype], s["offsets"],
                      s["order"], s["adapters"], m, n, k, s["rank"], s["workspace"],
                      s["workspace"].numel(), stream=stream)
        return [s["y"]]
    if op == "lora_bwd":
        m, n, k = s["rows"], s["n"], s["k"]
        ckl.gemm_lora_backward(dt, s["dy"], s["x"], s["w"], s["a"], s["b"], s["scales"], s["dx"], dt, s["da"], s["db"],
                               code[s["da"].dtype], s["offsets"], s["order"], s["adapters"], m, n, k,
                               s["rank"], s["workspace"], s["workspace"].numel(), stream=stream)
        return [s["dx"], s["da"], s["db"]]
    t, e, j, n = s["tokens"], s["experts"], s["top_k"], s["n"]
    rows = t * j
    if op == "experts":
        ckl.gemm_grouped(dt, s["x"], s["w"], s["y"], code[s["y"].dtype], s["offsets"], e, rows, n, s["k"],
                         a_rows=s["token"], a_count=t, stream=stream)
        return [s["y"]]
    if op == "experts_bwd":
        k = s["k"]
        ckl.gemm_grouped(dt, s["dy"], s["w"], s["dx"], dt, s["offsets"], e, rows, k, n, trans_b=True, stream=stream)
        ckl.gemm_grouped_wgrad(dt, s["x"], s["dy"], s["dw"], code[s["dw"].dtype], s["offsets"], e, rows, k, n,
                               a_rows=s["token"], a_count=t, stream=stream)
        return [s["dx"], s["dw"]]
    if op == "combine":
        ckl.moe_combine(dt, s["y"], s["positions"], s["weights"], s["out"], dt, t, j, n, rows, stream=stream)
        return [s["out"]]
    ckl.moe_combine_backward(dt, s["y"], s["positions"], s["weights"], s["dout"], dt, s["dy"], s["dweights"], t, j, n,
                             rows, stream=stream)
    return [s["dy"], s["dweights"]]


def run(state):
    return _own(state) if own else _plain(state)


# ---- 64 bits, row by row or group by group ------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("route", "route_bwd"):
        x = s["logits"].double()
        if case["score"] == "sigmoid":
            score = torch.exp(-torch.logaddexp(torch.zeros_like(x), -x))
        else:
            score = torch.nan_to_num(torch.exp(x - torch.logsumexp(x, 1, keepdim=True)), nan=0.0)
        if op == "route":
            chosen = _route_plain(s)[1].long()
            w = torch.where(chosen < 0, 0.0, torch.take_along_dim(score, chosen.clamp(min=0), 1))
            if case["renorm"]:
                w = torch.nan_to_num(w / w.sum(1, keepdim=True), nan=0.0)
            return [w, None, None, None, None]
        chosen, e = s["chosen"].long(), case["experts"]
        pick = torch.nn.functional.one_hot(chosen.clamp(min=0), e).double() * (chosen >= 0).unsqueeze(2)
        w = torch.einsum("tke,te->tk", pick, score)
        d = s["dweights"].double()
        if case["renorm"]:
            total = w.sum(1, keepdim=True)
            d = torch.nan_to_num(d / total - (d * w).sum(1, keepdim=True) / total ** 2, nan=0.0, posinf=0.0, neginf=0.0)
        d = torch.einsum("tke,tk->te", pick, d)
        if case["score"] == "sigmoid":
            return [d * score * torch.exp(-torch.logaddexp(torch.zeros_like(x), x))]
        return [score * d - score * (score * d).sum(1, keepdim=True)]
    if op in ("lora", "lora_bwd"):
        x, w = s["x"].double(), s["w"].double()
        bounds = s["offsets"].tolist()
        y = x @ w if op == "lora" else None
        dx = s["dy"].double() @ w.t() if op == "lora_bwd" else None
        da = torch.zeros(s["a"].shape, dtype=torch.float64, device=x.device)
        db = torch.zeros(s["b"].shape, dtype=torch.float64, device=x.device)
        for g in range(case["adapters"]):
            rows = s["order"][bounds[g]:bounds[g + 1]].long()
            a, b, f = s["a"][g].double(), s["b"][g].double(), s["scales"][g].double()
            if op == "lora":
                y[rows] += f * (x[rows] @ a) @ b
            else:
                dy = s["dy"][rows].double()
                u = f * dy @ b.t()
                dx[rows] += u @ a.t()
                da[g] = x[rows].t() @ u
                db[g] = f * (x[rows] @ a).t() @ dy
        return [y] if op == "lora" else [dx, da, db]
    if op in ("experts", "experts_bwd"):
        if case["tokens"] * case["top_k"] * case["k"] * case["n"] > 1 << 40:
            return None
        bounds = s["offsets"].tolist()
        rows, k, n = bounds[-1], case["k"], case["n"]
        if op == "experts":
            y = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
        else:
            dx = torch.zeros(rows, k, dtype=torch.float64, device="cuda")
            dw = torch.zeros(case["experts"], k, n, dtype=torch.float64, device="cuda")
        for g in range(case["experts"]):
            p, q = bounds[g], bounds[g + 1]
            if p == q:
                continue
            x, w = s["x"][s["token"][p:q].long()].double(), s["w"][g].double()
            if op == "experts":
                y[p:q] = x @ w
            else:
                dy = s["dy"][p:q].double()
                dx[p:q] = dy @ w.t()
                dw[g] = x.t() @ dy
        return [y] if op == "experts" else [dx, dw]
    t, j, n = case["tokens"], case["top_k"], case["n"]
    at = s["positions"].view(t, j).long()
    if op == "combine":
        out = torch.zeros(t, n, dtype=torch.float64, device="cuda")
        for i in range(j):
            out += s["weights"][:, i:i + 1].double() * s["y"][at[:, i]].double()
        return [out]
    dout = s["dout"].double()
    dy = torch.zeros(t * j, n, dtype=torch.float64, device="cuda")
    dw = torch.zeros(t, j, dtype=torch.float64, device="cuda")
    for i in range(j):
        dy[at[:, i]] = s["weights"][:, i:i + 1].double() * dout
        dw[:, i] = torch.einsum("tn,tn->t", s["y"][at[:, i]].double(), dout)
    return [dy, dw]


def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if op in ("route", "route_bwd"):
        t, e, k, b = case["tokens"], case["experts"], case["top_k"], size[case["dtype"]]
        if op == "route":
            # logits and bias in; weights, experts, rows, positions and offsets out
            return {"bytes": t * e * b + 4 * e * case["bias"] + 16 * t * k + 4 * (e + 1), "flops": 4 * t * e}
        return {"bytes": 2 * t * e * b + 8 * t * k, "flops": 6 * t * e}
    b = size[case["dtype"]]
    if op in ("lora", "lora_bwd"):
        m, k, n, r, o = case["rows"], case["k"], case["n"], case["rank"], b
        g = min(case["adapters"], m)
        with_adapter = m * case["adapters"] / (case["adapters"] + 1)
        weights = b * (k * n + g * r * (k + n))
        if op == "lora":
            return {"bytes": weights + b * m * k + o * m * n + 8 * m,
                    "flops": 2 * m * k * n + 2 * with_adapter * r * (k + n)}
        return {"bytes": weights + b * m * (2 * k + n) + o * g * r * (k + n) + 8 * m,
                "flops": 2 * m * k * n + with_adapter * r * (6 * k + 4 * n)}
    t, e, j, n = case["tokens"], case["experts"], case["top_k"], case["n"]
    rows = t * j
    if op in ("experts", "experts_bwd"):
        k, o = case["k"], b
        used = e * (1 - (1 - min(1.0, j / e)) ** t)  # experts that at least one token asks for
        weights = b * used * k * n
        if op == "experts":
            return {"bytes": weights + b * t * k + o * rows * n + 4 * rows, "flops": 2 * rows * k * n}
        return {"bytes": weights + b * t * k + b * rows * (n + k) + o * e * k * n + 4 * rows, "flops": 4 * rows * k * n}
    if op == "combine":
        return {"bytes": b * (rows + t) * n + 8 * rows, "flops": 2 * rows * n}
    return {"bytes": b * (2 * rows + t) * n + 12 * rows, "flops": 3 * rows * n}
