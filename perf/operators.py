"""What a program that serves a model in microscaled 4-bit floating point (MXFP4) asks of this framework, as
measurable cases.

  linear   one linear layer, bf16 in and out: ``MxLinearMethod.apply`` of MXFP4 weights (dynamic MXFP4
           activations: quantisation and product)
  down     SwiGLU -> MXFP4 -> down projection of an MLP: ``linear.swiglu_mxfp4_down``
  experts  the routed experts of a mixture: ``Mxfp4Experts`` from hidden states, route weights and ids
  router   scores, groups, top-k and the sort of the routes by expert: ``ops.moe_router_grouped``

Where ``own`` is false ``run`` computes the same from the checkpoint tensors by elementary torch
operations.  Decode cases with ``"graph"`` replay one captured call of the framework, as a serving loop
does after its warmup; the others are plain calls.
"""
from __future__ import annotations

import math

import torch

own = False

SOFTMAX, SIGMOID = 0, 1
_capture_stream = None


def listed():
    return [
        # decode of one sequence through an attention-sized projection: the smallest call, latency and little else
        dict(name="linear_decode_1", kind="linear", m=1, n=2048, k=2048, bias=False, graph=True),
        # decode of an odd batch through the widest layer: its weights and little else
        dict(name="linear_decode_27", kind="linear", m=27, n=17408, k=5120, bias=False, graph=True),
        # a ragged prompt through a layer whose K is an odd number of 128-blocks, with a bias, called eagerly
        dict(name="linear_prefill_333", kind="linear", m=333, n=5120, k=2688, bias=True, graph=False),
        # the largest call: a long prefill chunk through the widest layer
        dict(name="linear_prefill_4096", kind="linear", m=4096, n=17408, k=5120, bias=False, graph=False),
        # a short prompt through the second half of an MLP block
        dict(name="down_512", kind="down", m=512, n=2560, k=9216, graph=False),
        # one sequence through a mixture's experts: the smallest step
        dict(name="experts_decode_1", kind="experts", m=1, h=2048, i=512, e=256, topk=8, graph=True),
        # a decode batch: nearly every expert's weights for a few rows each
        dict(name="experts_decode_64", kind="experts", m=64, h=2048, i=512, e=256, topk=8, graph=True),
        # a ragged prompt through few experts whose sizes are odd numbers of 128-blocks
        dict(name="experts_prefill_777", kind="experts", m=777, h=1920, i=640, e=48, topk=6, graph=False),
        # a prefill chunk through the mixture
        dict(name="experts_prefill_2048", kind="experts", m=2048, h=2048, i=512, e=256, topk=8, graph=False),
        # routing of one decode batch: sigmoid scores with a balance bias, half of eight groups
        dict(name="router_decode_17", kind="router", m=17, e=256, topk=8, scoring=SIGMOID, bias=True, groups=8,
             keep=4, renorm=True, scale=2.5, bf16=False, graph=True),
        # routing of a ragged prefill chunk: softmax scores from bf16 logits, an expert count that is no power of two
        dict(name="router_softmax_1000", kind="router", m=1000, e=160, topk=6, scoring=SOFTMAX, bias=False, groups=8,
             keep=3, renorm=False, scale=16.0, bf16=True, graph=False),
        # routing of the longest prefill chunk
        dict(name="router_prefill_16384", kind="router", m=16384, e=256, topk=8, scoring=SIGMOID, bias=True, groups=8,
             keep=4, renorm=True, scale=2.5, bf16=False, graph=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _multiple(rng, lo, hi, q):
    return max(lo, min(hi, _log(rng, lo, hi) // q * q))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "down", "experts", "experts", "router", "router"])
    if kind == "router":
        m, groups = _log(rng, 1, 16384), rng.choice([1, 2, 4, 8])
        e = groups * rng.randint(max(2, 16 // groups), 512 // groups)
        keep = rng.randint(1, groups)
        return dict(kind=kind, m=m, e=e, topk=rng.randint(1, min(10, keep * (e // groups))),
                    scoring=rng.choice([SOFTMAX, SIGMOID]), bias=rng.random() < 0.5, groups=groups, keep=keep,
                    renorm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5, 16.0]), bf16=rng.random() < 0.4,
                    graph=m <= 64 and rng.random() < 0.7)
    m = _log(rng, 1, 4096)
    graph = m <= 64 and rng.random() < 0.7
    if kind == "experts":
        return dict(kind=kind, m=min(m, 2048), h=_multiple(rng, 1024, 2048, 128), i=_multiple(rng, 256, 512, 128),
                    e=rng.randint(8, 256), topk=rng.randint(1, 8), graph=graph)
    k = _multiple(rng, 1024, 9216, 128)
    n = _multiple(rng, 512, 17408 if k <= 5120 else 9216, 8)
    if kind == "down":
        return dict(kind=kind, m=min(m, 2048), n=min(n, 5120), k=k, graph=graph)
    return dict(kind=kind, m=m, n=n, k=k, bias=rng.random() < 0.3, graph=graph)


# ------------------------------------------------------------------ inputs, from the seed alone


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _activations(g, m, k):
    """bf16 N(0, 1) with one channel in a hundred twenty times larger, as activations have."""
    x = _randn(g, m, k)
    x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 100)]] *= 20
    return x.bfloat16()


def _weight(g, shape, std):
    """Checkpoint tensors of an MXFP4 weight: codes, two per byte (the even column in the low half), and the
    E8M0 byte of every 32 columns, amax's power of two over 4."""
    w = _randn(g, *shape, std=std).view(*shape[:-1], -1, 32)
    e = torch.frexp(w.abs().amax(-1, keepdim=True).clamp_min(1e-20))[1] - 3
    codes = _code(torch.ldexp(w, -e)).view(*shape[:-1], -1, 2)
    return (codes[..., 0] | codes[..., 1] << 4).to(torch.uint8), (e + 127).squeeze(-1).to(torch.uint8)


def _code(v):
    """E2M1 codes of v: to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, sign in bit 3."""
    a = v.abs()
    c = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
         + (a >= 3.5).int() + (a > 5.0).int())
    return c | torch.signbit(v).int() << 3


def _inputs(case, seed):
    g, m, kind = torch.Generator(device="cuda").manual_seed(int(seed)), case["m"], case["kind"]
    if kind == "router":
        x = _randn(g, m, case["e"])
        return dict(x=x.bfloat16() if case["bf16"] else x, bias=_randn(g, case["e"], std=0.05) if case["bias"] else None)
    if kind == "experts":
        e, h, i = case["e"], case["h"], case["i"]
        w1, s1 = _weight(g, (e, 2 * i, h), 0.02)
        w2, s2 = _weight(g, (e, h, i), 0.02)
        p, ids = torch.softmax(_randn(g, m, e), -1).topk(case["topk"], -1)
        return dict(x=_activations(g, m, h), w1=w1, s1=s1, w2=w2, s2=s2, p=p / p.sum(-1, keepdim=True),
                    ids=ids.int(), most=int(torch.bincount(ids.flatten(), minlength=e).max()))
    n, k = case["n"], case["k"]
    w, s = _weight(g, (n, k), 0.02)
    if kind == "down":
        return dict(x=_randn(g, m, 2 * k).bfloat16(), w=w, s=s)
    return dict(x=_activations(g, m, k), w=w, s=s, bias=_randn(g, n).bfloat16() if case["bias"] else None)


# ------------------------------------------------------------------ the framework's calls


def _layer(mx, n, k, w, s):
    method, layer = mx.MxLinearMethod(mx.linear.MXFP4_STATIC), torch.nn.Module()
    method.create_weights(layer, k, [n], k, n, torch.bfloat16, device="cuda")
    layer.weight.weight_loader(layer.weight, w)
    layer.weight_scale.weight_loader(layer.weight_scale, s)
    method.process_weights_after_loading(layer)
    return method, layer


def _program(case, d):
    """The call that a user's program makes on each pass, as a function without arguments."""
    from __graft_entry__ import load_package

    mx = load_package()
    if case["kind"] == "router":
        return lambda: mx.ops.moe_router_grouped(d["x"], d["bias"], case["topk"], case["scoring"], case["groups"],
                                                 case["keep"], case["renorm"], case["scale"])
    if case["kind"] == "experts":
        experts = mx.Mxfp4Experts()
        w1, w2 = experts.process_weights_after_loading(d["w1"], d["s1"], d["w2"], d["s2"])
        return lambda: experts(d["x"], w1, w2, d["p"], d["ids"])
    method, layer = _layer(mx, case["n"], case["k"], d["w"], d["s"])
    if case["kind"] == "down":
        return lambda: mx.linear.swiglu_mxfp4_down(d["x"], layer)
    return lambda: method.apply(layer, d["x"], d["bias"])


def _captured(call):
    """The call in a graph, as a serving loop keeps it for a batch size: (graph, its output)."""
    global _capture_stream
    if _capture_stream is None:  # a program captures on one stream of its own
        _capture_stream = torch.cuda.Stream()
    _capture_stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(_capture_stream):
        call()
    _capture_stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=_capture_stream):
        out = call()
    return graph, out


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:
        # the layer's laid-out weights stand for the checkpoint's, which a program drops; a decode step is captured
        call = _program(case, d)
        for name in ("w", "s", "w1", "s1", "w2", "s2"):
            d.pop(name, None)
        if case["graph"]:
            graph, out = _captured(call)
            return dict(graph=graph, out=out, call=call)
        return dict(call=call)
    return dict(case=case, d=d)


def run(state):
    if own:
        if "graph" in state:
            state["graph"].replay()
            return state["out"]
        return state["call"]()
    return _PLAIN[state["case"]["kind"]](state["case"], state["d"])


# ------------------------------------------------------------------ the plain form


def _values(packed, scale):
    """The values of packed MXFP4 codes, fp32."""
    c = torch.stack([packed & 15, packed >> 4], -1).long()
    t = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=packed.device)
    v = torch.cat([t, -t])[c].view(*scale.shape, 32)
    return torch.ldexp(v, scale.int().unsqueeze(-1) - 127).view(*packed.shape[:-1], -1)


def _quantized(x):
    """The values that the dynamic MXFP4 quantisation of bf16 ``x`` stands for: per 32 the amax's power of two
    over 4, doubled from 1.75 of it on, where the amax would round past 6."""
    b = x.float().view(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    f, e = torch.frexp(amax)
    s = torch.where(amax > 0, (e - 1 + (f >= 0.875).int() - 2 + 127).clamp_min(0), 0)
    c = _code(torch.ldexp(b, 127 - s))
    t = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    v = torch.ldexp(torch.cat([t, -t])[c.long()], s - 127)
    return torch.where(torch.isfinite(amax), v, math.nan).view(x.shape)


def _swiglu(mid):
    g, u = mid.float().chunk(2, -1)
    return ((g / (1 + torch.exp(-g))).bfloat16().float() * u).bfloat16()


def _plain_linear(case, d):
    y = _quantized(d["x"]) @ _values(d["w"], d["s"]).t()
    return (y if d["bias"] is None else y + d["bias"].float()).bfloat16()


def _plain_down(case, d):
    return (_quantized(_swiglu(d["x"])) @ _values(d["w"], d["s"]).t()).bfloat16()


def _plain_experts(case, d):
    m, h, e, topk, cap = case["m"], case["h"], case["e"], case["topk"], d["most"]
    ids, order = torch.sort(d["ids"].flatten().long(), stable=True)
    first = torch.searchsorted(ids, torch.arange(e, device=ids.device))
    slot = ids * cap + torch.arange(m * topk, device=ids.device) - first[ids]  # each expert's rows side by side
    rows = torch.zeros(e * cap, h, device=ids.device)
    rows[slot] = _quantized(d["x"])[order // topk]
    mid = torch.bmm(rows.view(e, cap, h), _values(d["w1"], d["s1"]).transpose(1, 2).contiguous()).bfloat16()
    act = _quantized(_swiglu(mid).view(e * cap, -1)).view(e, cap, -1)
    y = torch.bmm(act, _values(d["w2"], d["s2"]).transpose(1, 2).contiguous()).bfloat16().float().view(e * cap, h)
    routed = torch.empty(m * topk, h, device=ids.device)
    routed[order] = y[slot]
    return (routed.view(m, topk, h) * d["p"].unsqueeze(-1)).sum(1).bfloat16()


def _plain_router(case, d):
    m, e, topk, groups = case["m"], case["e"], case["topk"], case["groups"]
    x = d["x"].double()  # in 64 bits: which experts are chosen hangs on scores next to each other
    s = torch.softmax(x, -1) if case["scoring"] == SOFTMAX else 1 / (1 + torch.exp(-x))
    c = s if d["bias"] is None else s + d["bias"].double()
    per = c.view(m, groups, e // groups)
    of_group = per.amax(-1) if d["bias"] is None else per.topk(min(2, e // groups), -1).values.sum(-1)
    kept = torch.sort(of_group, stable=True, dim=-1, descending=True).indices[:, : case["keep"]]
    allowed = torch.zeros(m, groups, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
    c = torch.where(allowed.unsqueeze(-1), per, -math.inf).view(m, e)
    ids = torch.sort(c, stable=True, dim=-1, descending=True).indices[:, :topk]
    w = s.gather(1, ids)
    w = (w / (w.sum(-1, keepdim=True) + 1e-20) if case["renorm"] else w) * case["scale"]
    in_order, routes = torch.sort(ids.flatten(), stable=True)
    offsets = torch.searchsorted(in_order, torch.arange(e + 1, device=x.device))
    inverse = torch.empty_like(routes).scatter_(0, routes, torch.arange(m * topk, device=x.device))
    return w.float(), ids.int(), routes.int(), offsets, inverse.int()


_PLAIN = dict(linear=_plain_linear, down=_plain_down, experts=_plain_experts, router=_plain_router)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    m = case["m"]
    if case["kind"] == "router":
        # the logits and the bias; weights, ids, sorted routes and their inverse; offsets.  Per score an exp's worth
        return dict(bytes=m * case["e"] * (2 if case["bf16"] else 4) + 16 * m * case["topk"] + 8 * (case["e"] + 1)
                    + 4 * case["e"] * case["bias"], flops=10 * m * case["e"])
    if case["kind"] == "experts":
        # each expert that some token is routed to (uniform routing: the expected share) reads its weights once
        h, i, e = case["h"], case["i"], case["e"]
        hit = e * (1 - (1 - case["topk"] / e) ** m)
        return dict(bytes=int(hit * 3 * i * h * 17 / 32) + 4 * m * h + 8 * m * case["topk"],
                    flops=6 * m * case["topk"] * h * i)
    n, k = case["n"], case["k"]
    wide = 2 if case["kind"] == "down" else 1
    return dict(bytes=n * k * 17 // 32 + 2 * wide * m * k + 2 * m * n + 2 * n * bool(case.get("bias")),
                flops=2 * m * n * k)


# ------------------------------------------------------------------ the same in 64 bits


def _exact_weight(packed, scale):
    sign = 1.0 - 2.0 * torch.stack([packed >> 3 & 1, packed >> 7], -1).double()
    e = torch.stack([packed >> 1 & 3, packed >> 5 & 3], -1).double()
    f = torch.stack([packed & 1, packed >> 4 & 1], -1).double()
    v = sign * torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2(e - 1))
    return (v.view(*scale.shape, 32) * torch.exp2(scale.double() - 127).unsqueeze(-1)).view(*packed.shape[:-1], -1)


def _exact_quantized(x):
    b = x.double().view(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax.clamp_min(2.0 ** -126))[1].double() - 1
    e = e + (amax >= 1.75 * torch.exp2(e)) - 2
    scale = torch.exp2(e.clamp_min(-127))
    v = b.abs() / scale
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    q = (torch.round(v / step) * step).clamp_max(6)  # torch.round takes halves to the even integer
    return (torch.copysign(q, b) * scale).view(x.shape)


def exact(case, seed):
    d, kind = _inputs(case, seed), case["kind"]
    x = d["x"]
    if kind == "router":
        s = torch.sigmoid(x.double()) if case["scoring"] == SIGMOID else torch.exp(torch.log_softmax(x.double(), -1))
        c = s + (0 if d["bias"] is None else d["bias"].double())
        size, taken = case["e"] // case["groups"], []
        best = torch.stack([c[:, j * size:(j + 1) * size].sort(-1, descending=True).values[:, : 2 if case["bias"] else 1]
                            .sum(-1) for j in range(case["groups"])], -1)
        out = torch.ones_like(best, dtype=torch.bool)
        for _ in range(case["keep"]):  # argmax takes the first of equals
            top = torch.where(out, best, -math.inf).max(-1, keepdim=True).values
            out.scatter_(1, (out & (best == top)).int().argmax(-1, keepdim=True), False)
        left = ~out.repeat_interleave(size, 1)
        for _ in range(case["topk"]):
            top = torch.where(left, c, -math.inf).max(-1, keepdim=True).values
            taken.append((left & (c == top)).int().argmax(-1, keepdim=True))
            left.scatter_(1, taken[-1], False)
        w = s.gather(1, torch.cat(taken, 1))
        if case["renorm"]:
            w = w / w.sum(-1, keepdim=True)
        return w * case["scale"], None, None, None, None
    if kind == "down":
        return _exact_quantized(_swiglu(x)) @ _exact_weight(d["w"], d["s"]).t()
    if kind == "linear":
        y = _exact_quantized(x) @ _exact_weight(d["w"], d["s"]).t()
        return y if d["bias"] is None else y + d["bias"].double()
    a, out = _exact_quantized(x), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(case["e"]):
        t, slot = (d["ids"] == e).nonzero(as_tuple=True)
        if len(t):
            mid = (a[t] @ _exact_weight(d["w1"][e], d["s1"][e]).t()).bfloat16()
            y = (_exact_quantized(_swiglu(mid)) @ _exact_weight(d["w2"][e], d["s2"][e]).t()).bfloat16()
            out.index_add_(0, t, y.double() * d["p"][t, slot].double().unsqueeze(-1))
    return out
