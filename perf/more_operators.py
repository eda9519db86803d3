"""What a program that serves or fine-tunes adapters on a quantized model asks of this framework, as measurable cases.

  adapters        one quantized linear layer with the low-rank adapters of many requests beside it:
                  ``MxLinearMethod.apply(..., adapters=, batch=)``
  adapters_train  the same with its gradients: the adapters' and the input's, the layer frozen
  gated           the first half of an MLP block, act(gate) * up of a quantized gate/up layer: ``linear.gated_linear``
  gated_train     the same with the input's gradient, the layer frozen

Where ``own`` is false ``run`` computes the same from the checkpoint tensors by elementary torch
operations.  Decode cases with ``"graph"`` replay one captured call of the framework, as a serving loop
does after its warmup; the others are plain calls.
"""
from __future__ import annotations

import math

import torch

own = False

_capture_stream = None


def listed():
    return [
        # decode of one request with its adapter through an attention-sized projection: the smallest call, latency
        # and little else
        dict(name="adapters_decode_1", kind="adapters", fmt="mxfp8", m=1, k=2048, widths="2048", rank=16, slots=8,
             requests=1, graph=True),
        # decode of 48 requests that share 32 adapters, some without one, through the widest layer
        dict(name="adapters_decode_48", kind="adapters", fmt="mxfp6", m=48, k=5120, widths="17408", rank=16, slots=32,
             requests=48, graph=True),
        # a batch of ragged prompts through a merged projection of three parts, ranks of 8, called eagerly
        dict(name="adapters_prefill_777", kind="adapters", fmt="mxfp4", m=777, k=2688, widths="4096,512,512", rank=8,
             slots=5, requests=6, graph=False),
        # the largest call: a long prefill chunk of several requests through the widest layer, ranks of 64
        dict(name="adapters_prefill_4096", kind="adapters", fmt="mxfp8", m=4096, k=5120, widths="17408", rank=64,
             slots=8, requests=7, graph=False),
        # a small step of training three adapters at once on a merged block-FP8 layer
        dict(name="adapters_train_333", kind="adapters_train", fmt="block", m=333, k=2688, widths="2560,2560", rank=8,
             slots=3, requests=4, graph=False),
        # a step of training one adapter on the widest MLP layer
        dict(name="adapters_train_2048", kind="adapters_train", fmt="mxfp8", m=2048, k=2560, widths="9216,9216",
             rank=16, slots=1, requests=1, graph=False),
        # decode of one sequence through an MLP's first half: its weights and little else
        dict(name="gated_decode_1", kind="gated", fmt="mxfp8", m=1, k=2560, i=9216, act="silu", graph=True),
        # a decode batch through a mixture's small shared expert: latency
        dict(name="gated_decode_16", kind="gated", fmt="mxfp4", m=16, k=2048, i=512, act="silu", graph=True),
        # a ragged prompt through a small MLP with the other activation, odd numbers of 128-blocks
        dict(name="gated_prefill_777", kind="gated", fmt="mxfp6", m=777, k=1920, i=640, act="gelu_tanh", graph=False),
        # a long prefill chunk through an MLP's first half
        dict(name="gated_prefill_4096", kind="gated", fmt="mxfp8", m=4096, k=2560, i=9216, act="silu", graph=False),
        # a small training step, an odd number of tokens
        dict(name="gated_train_513", kind="gated_train", fmt="mxfp8", m=513, k=2688, i=2560, act="gelu_tanh",
             graph=False),
        # a training step through the widest MLP
        dict(name="gated_train_2048", kind="gated_train", fmt="mxfp4", m=2048, k=2560, i=9216, act="silu", graph=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _multiple(rng, lo, hi, q):
    return max(lo, min(hi, _log(rng, lo, hi) // q * q))


def draw(rng):
    kind = rng.choice(["adapters", "adapters", "adapters_train", "gated", "gated", "gated_train"])
    train = kind.endswith("_train")
    m = _log(rng, 16, 2048) if train else _log(rng, 1, 4096)
    graph = not train and m <= 64 and rng.random() < 0.7
    k = _multiple(rng, 1024, 2560 if train else 5120, 128)
    if kind.startswith("gated"):
        return dict(kind=kind, fmt=rng.choice(["mxfp8", "mxfp6", "mxfp4"]), m=m, k=k, i=_multiple(rng, 512, 9216, 64),
                    act=rng.choice(["silu", "gelu_tanh"]), graph=graph)
    parts = rng.choice([1, 1, 2, 3])
    widths = [_multiple(rng, 512, (16384 if train else 17408) // parts, 128) for _ in range(parts)]
    slots = rng.randint(1, 8) if train else rng.randint(1, 32)
    return dict(kind=kind, fmt=rng.choice(["mxfp8", "mxfp6", "mxfp4", "block"]), m=m, k=k,
                widths=",".join(map(str, widths)), rank=rng.choice([8, 16, 24, 32, 64]), slots=slots,
                requests=m if m <= 64 and not train else rng.randint(1, min(m, 2 * slots)), graph=graph)


# ------------------------------------------------------------------ inputs, from the seed alone


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _activations(g, m, k):
    """bf16 N(0, 1) with one channel in a hundred twenty times larger, as activations have."""
    x = _randn(g, m, k)
    x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 100)]] *= 20
    return x.bfloat16()


_FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_FP6 = [i / 8 for i in range(16)] + [(8 + i) / 4 for i in range(8)] + [(8 + i) / 2 for i in range(8)]  # E2M3


def _nearest(v, table):
    """The index into ``table`` (ascending) of the value next to |v|, with v's sign above the index bits."""
    t = torch.tensor(table, device=v.device)
    return torch.bucketize(v.abs(), (t[1:] + t[:-1]) / 2) + torch.signbit(v).long() * len(table)


def _weight(g, fmt, n, k):
    """Checkpoint tensors of a weight N(0, 0.02): E4M3 codes, four 6-bit E2M3 codes to three bytes (a little-endian
    bit stream) or two E2M1 codes to a byte (the even column in the low half), each with the E8M0 bytes of every 32
    columns; block-FP8: E4M3 codes and fp32 scales of 128 x 128."""
    w = _randn(g, n, k, std=0.02)
    if fmt == "block":
        s = w.view(n // 128, 128, k // 128, 128).abs().amax((1, 3)) / 448
        wide = s.repeat_interleave(128, 0).repeat_interleave(128, 1)
        return (w / wide).to(torch.float8_e4m3fn), s
    w = w.view(n, -1, 32)
    e = torch.frexp(w.abs().amax(-1, keepdim=True).clamp_min(1e-20))[1] - 1 - {"mxfp8": 7, "mxfp6": 2, "mxfp4": 2}[fmt]
    scale, v = (e + 127).squeeze(-1).to(torch.uint8), torch.ldexp(w, -e)
    if fmt == "mxfp8":
        return v.view(n, k).to(torch.float8_e4m3fn), scale
    if fmt == "mxfp4":
        c = _nearest(v, _FP4).view(n, -1, 2)
        return (c[..., 0] | c[..., 1] << 4).to(torch.uint8), scale
    c = _nearest(v, _FP6).view(n, -1, 4)
    bits = c[..., 0] | c[..., 1] << 6 | c[..., 2] << 12 | c[..., 3] << 18
    return torch.stack([bits & 255, bits >> 8 & 255, bits >> 16], -1).to(torch.uint8).view(n, -1), scale


def _ids(g, case):
    """The adapter of each token: requests of ragged lengths one after the other, one in eight without an adapter (-1);
    a training batch has none of those."""
    m, many = case["m"], case["requests"]
    cuts = torch.randperm(m - 1, generator=g, device="cuda")[: many - 1] + 1
    request = torch.zeros(m, dtype=torch.long, device="cuda")
    request[cuts] = 1
    of = torch.randint(0, case["slots"], (many,), generator=g, device="cuda")
    if case["kind"] == "adapters" and many > 1:
        of = torch.where(torch.rand(many, generator=g, device="cuda") < 0.125, -1, of)
    return of[request.cumsum(0)].int()


def _parts(case):
    return [int(n) for n in case["widths"].split(",")]


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    m, k, train = case["m"], case["k"], case["kind"].endswith("_train")
    d = dict(x=_activations(g, m, k))
    if case["kind"].startswith("gated"):
        d["w"], d["s"] = _weight(g, case["fmt"], 2 * case["i"], k)
        n = case["i"]
    else:
        n, slots, rank = sum(_parts(case)), case["slots"], case["rank"]
        d["w"], d["s"] = _weight(g, case["fmt"], n, k)
        d["a"] = _randn(g, slots, len(_parts(case)) * rank, k, std=k ** -0.5).bfloat16()
        d["b"] = _randn(g, slots, n, rank, std=0.05).bfloat16()
        d["scaling"] = 0.5 + torch.rand(slots, generator=g, device="cuda")
        d["ids"] = _ids(g, case)
    if train:
        d["dy"] = _randn(g, m, n).bfloat16()
    return d


# ------------------------------------------------------------------ the framework's calls


def _layer(mx, fmt, widths, k, w, s):
    key = dict(mxfp8=mx.linear.MXFP8_STATIC, mxfp6=mx.linear.MXFP6_E2M3_STATIC, mxfp4=mx.linear.MXFP4_STATIC,
               block=mx.linear.FP8_BLOCK128)[fmt]
    method, layer = mx.MxLinearMethod(key), torch.nn.Module()
    method.create_weights(layer, k, widths, k, sum(widths), torch.bfloat16, device="cuda")
    scale = layer.weight_scale_inv if fmt == "block" else layer.weight_scale
    layer.weight.weight_loader(layer.weight, w)
    scale.weight_loader(scale, s)
    method.process_weights_after_loading(layer)
    return method, layer


def _program(case, d):
    """The call that a user's program makes on each pass, as a function without arguments."""
    from __graft_entry__ import load_package

    mx = load_package()
    if case["kind"].startswith("gated"):
        method, layer = _layer(mx, case["fmt"], [case["i"]] * 2, case["k"], d["w"], d["s"])
        call, leaves = (lambda x: mx.linear.gated_linear(x, layer, case["act"])), []
    else:
        method, layer = _layer(mx, case["fmt"], _parts(case), case["k"], d["w"], d["s"])
        adapters = mx.LowRankAdapters(layer, case["slots"], case["rank"])
        adapters.lora_a.data.copy_(d["a"])
        adapters.lora_b.data.copy_(d["b"])
        adapters.scaling.copy_(d["scaling"])
        batch = mx.AdapterBatch(d["ids"], case["slots"])  # one for all layers of a step
        call = lambda x: method.apply(layer, x, None, adapters=adapters, batch=batch)  # noqa: E731
        leaves = [adapters.lora_a, adapters.lora_b]
        for leaf in leaves:
            leaf.requires_grad_(case["kind"].endswith("_train"))
    x = d["x"]
    if not case["kind"].endswith("_train"):
        return lambda: call(x)
    x.requires_grad_()

    def step():
        y = call(x)
        return (y.detach(), *torch.autograd.grad(y, [x, *leaves], d["dy"]))

    return step


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
        for name in ("w", "s", "a", "b"):
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


def _values(fmt, w, s):
    """The weight's values, fp32."""
    if fmt == "block":
        return w.float() * s.repeat_interleave(128, 0).repeat_interleave(128, 1)
    if fmt == "mxfp8":
        v = w.float()
    elif fmt == "mxfp4":
        t = torch.tensor(_FP4, device=w.device)
        v = torch.cat([t, -t])[torch.stack([w & 15, w >> 4], -1).long()]
    else:
        t = torch.tensor(_FP6, device=w.device)
        b = w.view(len(w), -1, 3).int()
        b = b[..., 0] | b[..., 1] << 8 | b[..., 2] << 16
        v = torch.cat([t, -t])[torch.stack([b & 63, b >> 6 & 63, b >> 12 & 63, b >> 18], -1).long()]
    return torch.ldexp(v.view(*s.shape, 32), s.int().unsqueeze(-1) - 127).view(len(w), -1)


def _quantized(fmt, x):
    """The values that the dynamic quantization of bf16 ``x`` stands for.  MXFP8 and MXFP4 (MXFP4 weights): per 32 the
    amax's power of two under the format's largest, doubled from 1.75 of it on; block-FP8: per 128 amax / 448."""
    if fmt == "block":
        b = x.float().view(len(x), -1, 128)
        s = b.abs().amax(-1, keepdim=True).clamp_min(1e-10)
        s = s / torch.full_like(s, 448)  # (by a number torch multiplies with its reciprocal)
        return ((b / s).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s).view(x.shape)
    b = x.float().view(len(x), -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    f, e = torch.frexp(amax)
    s = torch.where(amax > 0, e - 1 + (f >= 0.875).int() - (2 if fmt == "mxfp4" else 8), -127)
    v = torch.ldexp(b, -s)
    if fmt != "mxfp4":
        return torch.ldexp(v.to(torch.float8_e4m3fn).float(), s).view(x.shape)
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return torch.ldexp(torch.round(v / step) * step, s).view(x.shape)


def _low_rank(case, d):
    """For every adapter side by side (the others' columns zero): s x A^T of a token's own, [M, parts, slots rank]."""
    m, parts, slots, rank = case["m"], len(_parts(case)), case["slots"], case["rank"]
    v = (d["x"].detach().float() @ d["a"].float().view(-1, case["k"]).t()).view(m, slots, parts, rank)
    return (v * _mine(case, d)).transpose(1, 2).reshape(m, parts, slots * rank)


def _mine(case, d):
    """[M, slots, 1, 1]: the scaling of a token's adapter, 0 of the others."""
    is_mine = d["ids"].unsqueeze(-1) == torch.arange(case["slots"], device="cuda")
    return (is_mine * d["scaling"])[:, :, None, None]


def _b_parts(case, d):
    """Each part's rows of every adapter's B: [slots rank, N of the part]."""
    return [b.transpose(0, 1).reshape(b.shape[1], -1).t() for b in d["b"].float().split(_parts(case), 1)]


def _plain_adapters(case, d):
    v = _low_rank(case, d)
    delta = torch.cat([v[:, p] @ b for p, b in enumerate(_b_parts(case, d))], -1)
    return (_quantized(case["fmt"], d["x"]) @ _values(case["fmt"], d["w"], d["s"]).t() + delta).bfloat16()


def _plain_adapters_train(case, d):
    m, k, slots, rank, parts = case["m"], case["k"], case["slots"], case["rank"], _parts(case)
    w, v, bs, x = _values(case["fmt"], d["w"], d["s"]), _low_rank(case, d), _b_parts(case, d), d["x"].float()
    y = _quantized(case["fmt"], d["x"]) @ w.t() + torch.cat([v[:, p] @ b for p, b in enumerate(bs)], -1)
    dy = d["dy"].float()
    pieces = dy.split(parts, -1)
    dv = torch.stack([t @ b.t() for t, b in zip(pieces, bs)], 1).view(m, len(parts), slots, rank)
    dv = (dv.transpose(1, 2) * _mine(case, d)).reshape(m, -1)
    db = torch.cat([(t.t() @ v[:, p]).view(-1, slots, rank).transpose(0, 1) for p, t in enumerate(pieces)], 1)
    dx = dy @ w + dv @ d["a"].float().view(-1, k)
    return y.bfloat16(), dx.bfloat16(), (dv.t() @ x).view(slots, -1, k).bfloat16(), db.bfloat16()


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _plain_gated(case, d):
    g, u = (_quantized(case["fmt"], d["x"]) @ _values(case["fmt"], d["w"], d["s"]).t()).chunk(2, -1)
    return (_act(case["act"], g)[0] * u).bfloat16()


def _plain_gated_train(case, d):
    w = _values(case["fmt"], d["w"], d["s"])
    g, u = (_quantized(case["fmt"], d["x"]) @ w.t()).chunk(2, -1)
    (a, slope), dh = _act(case["act"], g), d["dy"].float()
    return (a * u).bfloat16(), (torch.cat([dh * u * slope, dh * a], -1) @ w).bfloat16()


_PLAIN = dict(adapters=_plain_adapters, adapters_train=_plain_adapters_train, gated=_plain_gated,
              gated_train=_plain_gated_train)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    m, k = case["m"], case["k"]
    n = 2 * case["i"] if case["kind"].startswith("gated") else sum(_parts(case))
    out = case["i"] if case["kind"].startswith("gated") else n
    # the weight's codes and scales, the input and the output
    nbytes = n * k * {"mxfp8": 33, "mxfp6": 25, "mxfp4": 17, "block": 32}[case["fmt"]] // 32 + 2 * m * (k + out)
    flops = 2 * m * n * k
    if not case["kind"].startswith("gated"):
        # the adapters that some request has (drawn evenly: the expected share), their two products
        hit = case["slots"] * (1 - (1 - 1 / case["slots"]) ** case["requests"])
        nbytes += int(hit * 2 * case["rank"] * (len(_parts(case)) * k + n)) + 4 * m
        flops += 2 * m * case["rank"] * (len(_parts(case)) * k + n)
    if case["kind"] == "gated_train":
        nbytes, flops = nbytes + 2 * m * (out + k), 2 * flops  # dh, dx; the input's gradient
    if case["kind"] == "adapters_train":
        # dy, dx and both gradients; three products of the low rank, two of each side
        size = 2 * case["slots"] * case["rank"] * (len(_parts(case)) * k + n)
        nbytes, flops = nbytes + 2 * m * (out + k) + size, 2 * flops + 2 * m * case["rank"] * (len(_parts(case)) * k + n)
    return dict(bytes=nbytes, flops=flops)


# ------------------------------------------------------------------ the same in 64 bits


def _exact_weight(fmt, w, s):
    if fmt == "block":
        return (w.double().view(w.shape[0] // 128, 128, -1, 128) * s.double()[:, None, :, None]).view(w.shape)
    if fmt == "mxfp8":
        v = w.double()
    else:
        bits, man = (4, 1) if fmt == "mxfp4" else (6, 3)
        per = 2 if fmt == "mxfp4" else 4
        word = sum(w.view(len(w), -1, per * bits // 8)[..., i].long() << 8 * i for i in range(per * bits // 8))
        c = torch.stack([word >> bits * i & (1 << bits) - 1 for i in range(per)], -1)
        e, f = (c >> man & 3).double(), (c & (1 << man) - 1).double() / (1 << man)
        v = torch.where(e == 0, f, (1 + f) * torch.exp2(e - 1)) * (1 - 2 * (c >> bits - 1).double())
    return (v.view(*s.shape, 32) * torch.exp2(s.double() - 127).unsqueeze(-1)).view(len(w), -1)


def _exact_quantized(fmt, x):
    group, top, man, low = {"block": (128, None, 3, -6), "mxfp4": (32, 2, 1, 0)}.get(fmt, (32, 8, 3, -6))
    b = x.double().view(len(x), -1, group)
    amax = b.abs().amax(-1, keepdim=True)
    if top is None:
        # its scale and quotient are binary32 by definition, correctly rounded
        scale = (amax.clamp_min(1e-10).float() / torch.full_like(amax, 448, dtype=torch.float32)).double()
        v = (b.float() / scale.float()).double().clamp(-448, 448)
    else:
        e = torch.frexp(amax.clamp_min(2.0 ** -100))[1].double() - 1
        scale = torch.exp2(e + (amax >= 1.75 * torch.exp2(e)) - top)
        v = b / scale
    step = torch.exp2((torch.frexp(v.abs().clamp_min(2.0 ** -60))[1].double() - 1).clamp_min(low) - man)
    return (torch.round(v / step) * step * scale).view(x.shape)  # torch.round takes halves to the even integer


def exact(case, seed):
    d, train = _inputs(case, seed), case["kind"].endswith("_train")
    w = _exact_weight(case["fmt"], d["w"], d["s"])
    y = _exact_quantized(case["fmt"], d["x"]) @ w.t()
    if case["kind"].startswith("gated"):
        i = case["i"]
        with torch.enable_grad():
            g, u = y[:, :i].detach().requires_grad_(), y[:, i:].detach().requires_grad_()
            if case["act"] == "silu":
                h = g * torch.sigmoid(g) * u
            else:
                h = g / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
            if not train:
                return h.detach()
            dg, du = torch.autograd.grad(h, [g, u], d["dy"].double())
        return h.detach(), dg @ w[:i] + du @ w[i:]
    x, a, b, rank = d["x"].double(), d["a"].double(), d["b"].double(), case["rank"]
    dy = d["dy"].double() if train else None
    dx, da, db = dy @ w if train else None, torch.zeros_like(a), torch.zeros_like(b)
    for slot in range(case["slots"]):
        t, lo, s = (d["ids"] == slot).nonzero().squeeze(-1), 0, d["scaling"][slot].double()
        for p, n in enumerate(_parts(case)):
            ap, bp = a[slot, p * rank:(p + 1) * rank], b[slot, lo:lo + n]
            v = x[t] @ ap.t()
            y[t, lo:lo + n] += s * (v @ bp.t())
            if train:
                dv = s * (dy[t, lo:lo + n] @ bp)
                dx[t] += dv @ ap
                da[slot, p * rank:(p + 1) * rank] = dv.t() @ x[t]
                db[slot, lo:lo + n] = s * (dy[t, lo:lo + n].t() @ v)
            lo += n
    return (y, dx, da, db) if train else y
