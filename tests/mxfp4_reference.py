"""MXFP4 and grouped routing by their formulas, in 64 bits, for the tests of the kernels: elementary torch and
numpy on the CPU, without the package."""
import numpy as np
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
FLOOR_CARRY175, FLOOR_OCP = 0, 3


def quantize(x, rule=FLOOR_CARRY175):
    """(codes u8 [M, K/2], scales u8 [M, K/32]) of bf16 x: the nearest grid value, ties to the even code."""
    x = x.cpu().double()
    b = x.view(x.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = torch.frexp(torch.where(bad, torch.zeros_like(amax), amax))[1].double() - 1
    if rule == FLOOR_CARRY175:
        e = e + (amax >= 1.75 * torch.exp2(e)).double()
    s = torch.where(amax > 0, (e - 2 + 127).clamp_min(0), torch.zeros_like(e))
    v = (b * torch.exp2(127 - s).unsqueeze(-1)).abs().nan_to_num()
    d = (v.unsqueeze(-1) - GRID).abs()
    lo = d.argmin(-1)  # the first of equals: of a tie the lower code
    up = (lo + 1).clamp_max(7)
    tie = (d.gather(-1, lo.unsqueeze(-1)) == d.gather(-1, up.unsqueeze(-1))).squeeze(-1) & (v < 6)
    code = torch.where(tie & (lo % 2 == 1), up, lo) + 8 * torch.signbit(b)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).view(x.shape[0], -1, 2)
    packed = (code[..., 0] + 16 * code[..., 1]).to(torch.uint8)
    return packed, torch.where(bad, torch.full_like(s, 255), s).to(torch.uint8)


def dequantize(codes, scales):
    """The values of packed codes and scales, float64 (a NaN scale: NaN)."""
    codes, scales = codes.cpu(), scales.cpu()
    c = torch.stack([codes & 15, codes >> 4], -1).long()
    v = torch.cat([GRID, -GRID])[c].view(*scales.shape, 32)
    f = torch.exp2(scales.double() - 127)
    f = torch.where(scales == 255, torch.full_like(f, float("nan")), f)
    return (v * f.unsqueeze(-1)).view(*codes.shape[:-1], -1)


def random_operand(g, rows, k, spread=3):
    """Codes and scales of every kind: uniform codes, scales within 2^+-spread of one."""
    return (torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8),
            torch.randint(127 - spread, 128 + spread, (rows, k // 32), generator=g, dtype=torch.uint8))


def check_product(got, a, w, bias=None):
    """got (bf16) against A W^T of the float64 operands.  Elementwise: the rounding to bf16 is off by at most half
    a step, 2^-8 of the value (twice with a bias), and the fp32 sum of K exact products by at most K 2^-23 of their
    magnitudes' sum; over the whole the half step alone bounds the relative error, as fp32's part is a thousandth of
    the largest share that a sum of random signs leaves.  Where the magnitudes' sum passes 2^127, an fp32 sum in
    progress may pass the largest fp32 value and be infinite or NaN with it: such elements say nothing."""
    a, w, got = a.cuda(), w.cuda(), got.double()
    ref, most = a @ w.t(), a.abs() @ w.abs().t()
    room = 2.0 ** -8 * ref.abs() + a.shape[1] * 2.0 ** -23 * most + 1e-30
    if bias is not None:
        ref = ref + bias.cuda().double()
        room = room + 2.0 ** -8 * ref.abs() + 2.0 ** -8 * room
    assert got.shape == ref.shape
    nan, over = torch.isnan(ref), most >= 2.0 ** 127
    assert torch.equal(torch.isnan(got)[~over], nan[~over])
    fine = ~nan & ~over
    got, ref, room = got[fine], ref[fine], room[fine]
    off = (got - ref).abs()
    assert bool((off <= room).all()), float((off / room).max())
    if ref.numel() and float(ref.norm()) > 0:
        rel = float((got - ref).norm() / ref.norm())
        assert rel <= 2.0 ** -8 * (1 if bias is None else 2), rel


def silu_activation(gate_up):
    """bf16(bf16(silu(g)) u): the activation ahead of the SwiGLU producer's quantization, from float64 exp."""
    g, u = gate_up.cpu().double().chunk(2, -1)
    return ((g / (1 + torch.exp(-g))).bfloat16().double() * u).bfloat16()


def route(logits, bias, topk, sigmoid, groups, keep, renorm, factor):
    """(weights float64 [T, k], ids [T, k]) token by token in Python's order of tuples: ties to the lower index."""
    x = logits.cpu().double().numpy()
    T, E = x.shape
    b = np.zeros(E) if bias is None else bias.cpu().double().numpy()
    size = E // groups
    with np.errstate(all="ignore"):
        if sigmoid:
            s = 1.0 / (1.0 + np.exp(-x))
        else:
            e = np.exp(x - x.max(-1, keepdims=True))
            s = e / e.sum(-1, keepdims=True)
        c = s + b
    c = np.where(np.isnan(c), -np.inf, c)
    weights, ids = np.zeros((T, topk)), np.zeros((T, topk), dtype=np.int64)
    for t in range(T):
        scores = []
        for k in range(groups):
            best = sorted(c[t, k * size:(k + 1) * size], reverse=True)
            v = best[0] + (best[1] if bias is not None and size > 1 else 0.0)
            scores.append(-np.inf if np.isnan(v) else v)
        kept = sorted(range(groups), key=lambda k: (-scores[k], k))[:keep]
        allowed = [i for k in kept for i in range(k * size, (k + 1) * size)]
        ids[t] = sorted(allowed, key=lambda i: (-c[t, i], i))[:topk]
        w = s[t, ids[t]]
        with np.errstate(all="ignore"):
            weights[t] = (w / (w.sum() + 1e-20) if renorm else w) * factor
    return weights, ids
