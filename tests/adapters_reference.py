"""The definitions of the quantized layers, their adapters, gated blocks and gradients in 64 bits, and random layers.

Weights are drawn as codes, so their values are known exactly.  ``bound`` is the elementwise error that a kernel may
have: bf16 roundings of half a step (2^-8 relative) and fp32 sums of ``terms`` products, 2^-24 of the products' absolute
sum each.
"""
import torch

U = 2.0 ** -8  # half a step of bf16, relative

_E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
_E2M3 = torch.tensor([i / 8 for i in range(8)] + [(8 + i) / 8 * 2 ** e for e in range(3) for i in range(8)], dtype=torch.float64)
_E3M2 = torch.tensor([i / 16 for i in range(4)] + [(4 + i) / 4 * 2.0 ** (e - 2) for e in range(7) for i in range(4)],
                     dtype=torch.float64)
FORMATS = ("mxfp8", "mxfp6", "mxfp6_e3m2", "mxfp4", "block")


def key_of(pkg, fmt):
    linear = pkg.linear
    return {"mxfp8": linear.MXFP8_STATIC, "mxfp6": linear.MXFP6_E2M3_STATIC, "mxfp6_e3m2": linear.MXFP6_E3M2_STATIC,
            "mxfp4": linear.MXFP4_STATIC, "block": linear.FP8_BLOCK128}[fmt]


def draw_weight(fmt, n, k, g, spread=3):
    """(codes, scales) as a checkpoint holds them and the values [n, k] in 64 bits."""
    if fmt in ("mxfp8", "block"):
        c = torch.randint(0, 0x78, (n, k), generator=g, dtype=torch.uint8) | torch.randint(0, 2, (n, k), generator=g, dtype=torch.uint8) << 7
        codes = c.view(torch.float8_e4m3fn)
        v = codes.float().double() / 64
    elif fmt == "mxfp4":
        c = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
        codes = c[:, 0::2] | c[:, 1::2] << 4
        v = torch.cat([_E2M1, -_E2M1])[c.long()]
    else:
        c = torch.randint(0, 64, (n, k), generator=g, dtype=torch.int32)
        t = _E2M3 if fmt == "mxfp6" else _E3M2
        v = torch.cat([t, -t])[c.long()]
        q = c.view(n, k // 4, 4)
        word = q[..., 0] | q[..., 1] << 6 | q[..., 2] << 12 | q[..., 3] << 18
        codes = torch.stack([word & 255, word >> 8 & 255, word >> 16], -1).to(torch.uint8).view(n, -1)
    if fmt == "block":
        s = torch.rand(((n + 127) // 128, k // 128), generator=g) * 1e-2 + 1e-3
        return codes, s, v * 64 * s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    s = torch.randint(127 - 5 - spread, 127 - 4, (n, k // 32), generator=g, dtype=torch.uint8)
    scale = torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    return codes, s, (v * 64 if fmt == "mxfp8" else v) * scale


def make_layer(pkg, fmt, widths, k, dev, g):
    """(method, prepared layer on dev, the weight's values in 64 bits on dev)."""
    n = sum(widths)
    method, layer = pkg.MxLinearMethod(key_of(pkg, fmt)), torch.nn.Module()
    method.create_weights(layer, k, list(widths), k, n, torch.bfloat16, device=dev)
    codes, s, v = draw_weight(fmt, n, k, g)
    scale = layer.weight_scale_inv if fmt == "block" else layer.weight_scale
    layer.weight.weight_loader(layer.weight, codes.to(dev))
    scale.weight_loader(scale, s.to(dev))
    method.process_weights_after_loading(layer)
    return method, layer, v.to(dev)


def quantized(fmt, x):
    """The values that a layer's dynamic quantization of x (bf16 [M, K], finite) stands for, in 64 bits."""
    group, top, man, low = {"block": (128, None, 3, -6), "mxfp4": (32, 2, 1, 0)}.get(fmt, (32, 8, 3, -6))
    b = x.double().view(x.shape[0], -1, group)
    amax = b.abs().amax(-1, keepdim=True)
    if top is None:
        scale = (amax.clamp_min(1e-10).float() / torch.full_like(amax, 448, dtype=torch.float32)).double()
        v = (b.float() / scale.float()).double().clamp(-448, 448)
    else:
        e = torch.frexp(amax.clamp_min(2.0 ** -100))[1].double() - 1
        scale = torch.exp2(e + (amax >= 1.75 * torch.exp2(e)) - top)
        v = b / scale
    step = torch.exp2((torch.frexp(v.abs().clamp_min(2.0 ** -60))[1].double() - 1).clamp_min(low) - man)
    return (torch.round(v / step) * step * scale).view(x.shape)


def product(a, w, scaled=False):
    """a w^T in 64 bits and the bound of its sum: fp32, or (``scaled``) by the scaled MFMA, which aligns the products of
    eight columns to the largest of them and cuts what lies below 2^-13 of its power of two (measured with products of
    2^8, -2^8 and n times 2^(8 - j): from j = 14 on exactly the seven beside a large one are lost, of 1.875^2 2^(8 - j) the
    bits below 2^(8 - 13)), so that up to seven products lose 2^-13 of the largest each: 7 2^-13 of the absolute sum."""
    return a @ w.t(), (a.abs() @ w.abs().t()) * (a.shape[1] * 2.0 ** -24 + (7 * 2.0 ** -13 if scaled else 0))


def adapters(x, a, b, scaling, ids, widths, rank):
    """(delta, bound of its fp32 part, v [M, parts, rank]) in 64 bits: v reaches B with 2^-16 of itself at most missing
    (two bf16 halves of 2^-8 each)."""
    m, n = x.shape[0], sum(widths)
    delta = torch.zeros(m, n, dtype=torch.float64, device=x.device)
    off = torch.zeros_like(delta)
    v_all = torch.zeros(m, len(widths), rank, dtype=torch.float64, device=x.device)
    x, a, b = x.double(), a.double(), b.double()
    for s in range(a.shape[0]):
        t, lo = (ids == s).nonzero().squeeze(-1), 0
        for p, w in enumerate(widths):
            ap, bp, f = a[s, p * rank:(p + 1) * rank], b[s, lo:lo + w], float(scaling[s])
            v = f * (x[t] @ ap.t())
            v_off = abs(f) * (x[t].abs() @ ap.abs().t()) * ((x.shape[1] + 2) * 2.0 ** -24)
            v_all[t, p] = v
            delta[t, lo:lo + w] = v @ bp.t()
            off[t, lo:lo + w] = (v.abs() * (2.0 ** -16 + 2 * rank * 2.0 ** -24) + v_off) @ bp.abs().t()
            lo += w
    return delta, off, v_all


def check(got, want, bound, what=""):
    bad = (got.double() - want).abs() > bound
    assert not bool(bad.any()), (what, int(bad.sum()), float((got.double() - want).abs().max()), float(want.abs().max()))


def act(name, g):
    """The activation and its derivative in 64 bits."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return g / 2 * (1 + t), (1 + t) / 2 + g / 2 * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
