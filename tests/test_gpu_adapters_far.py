"""Outputs, gradients and adapters of more than 2^31 values, checked in 64 bits at rows and columns from end to end."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu
M, N, K = 140000, 17408, 256


def _rows(dev):
    return torch.tensor([0, 1, 255, M // 2, 123361, 123362, M - 257, M - 2, M - 1], device=dev)


@pytest.mark.parametrize("slots", [2, 20])
def test_adapters(pkg, dev, slots):
    """M N > 2^31: in one product (2 slots) and apart (20)."""
    rank, eps = 16, 2.0 ** -24
    g = torch.Generator().manual_seed(slots)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [9216, 8192], K, dev, g)
    ad = pkg.LowRankAdapters(layer, slots, rank).requires_grad_()
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) / 16)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.copy_(torch.rand(slots, generator=g) + 0.5)
    x = torch.randn(M, K, generator=g).bfloat16().to(dev).requires_grad_()
    ids = torch.randint(-1, slots, (M,), generator=g).to(dev)
    bias = torch.randn(N, generator=g).bfloat16().to(dev).requires_grad_()
    assert pkg.ops.adapter_linear_supported(M, N, K, 0, False, slots, 2, rank) == (slots == 2)
    y = method.apply(layer, x, bias, adapters=ad, batch=pkg.AdapterBatch(ids, slots))
    dy = torch.randn(M, N, dtype=torch.bfloat16, device=dev)
    dx, da, db, dbias = torch.autograd.grad(y, [x, ad.lora_a, ad.lora_b, bias], dy)
    at = _rows(dev)
    xs, own = x.detach()[at], ids[at]
    base, off = ref.product(ref.quantized("mxfp8", xs), w, scaled=True)
    delta, doff, _ = ref.adapters(xs, ad.lora_a, ad.lora_b, ad.scaling, own, ad.widths, rank)
    b = bias.detach().double()
    size = (base.abs() + delta.abs() + b.abs()) * (1 + ref.U) ** 2
    ref.check(y.detach()[at], base + delta + b, 3 * ref.U * size + (1 + ref.U) ** 3 * (2 * off + doff))
    # dx of those rows, and the gradients of one slot's adapter at a few columns and ranks
    dys = dy[at].double()
    want, boff = ref.product(dys, w.t().contiguous())
    more = torch.zeros_like(want)
    for s in range(slots):
        lo = 0
        for p, width in enumerate(ad.widths):
            t = (own == s).nonzero().squeeze(-1)
            dv = float(ad.scaling[s]) * dys[t, lo:lo + width] @ ad.lora_b[s, lo:lo + width].double()
            ap = ad.lora_a[s, p * rank:(p + 1) * rank].double()
            want[t] += dv @ ap
            more[t] += (dv.abs() * (2.0 ** -16 + 64 * eps) + 2 * width * eps * float(ad.scaling[s])
                        * (dys[t, lo:lo + width].abs() @ ad.lora_b[s, lo:lo + width].double().abs())) @ ap.abs()
            lo += width
    ref.check(dx[at], want, 2 * ref.U * (want.abs() + (dys @ w).abs()) + (1 + ref.U) * (2 * boff + more), "dx")
    s, cols = slots - 1, torch.tensor([0, 9215, 9216, N - 1], device=dev)
    t = (ids == s).nonzero().squeeze(-1)
    xt, f = x.detach()[t].double(), float(ad.scaling[s])
    for c in cols.tolist():
        ap = ad.lora_a[s, (c >= 9216) * rank:(c >= 9216) * rank + rank].double()
        v, d = f * (xt @ ap.t()), dy[t, c].double()
        vo = f * (xt.abs() @ ap.abs().t()) * ((K + 2) * eps) + v.abs() * (2.0 ** -16 + (2 * len(t) + 16) * eps)
        ref.check(db[s, c], d @ v, ref.U * (d @ v).abs() + (1 + ref.U) * (d.abs() @ vo), "db")
        ref.check(dbias[c], dy[:, c].double().sum(), ref.U * dy[:, c].double().sum().abs() + M * eps * dy[:, c].double().abs().sum())
    dv = torch.cat([f * (dy[c, 9216:].double() @ ad.lora_b[s, 9216:].double()) for c in t.split(4096)])
    dvo = torch.cat([f * (dy[c, 9216:].double().abs() @ ad.lora_b[s, 9216:].double().abs()) for c in t.split(4096)])
    want = dv.t() @ xt
    off = (dvo * (8194 * eps) + dv.abs() * (2.0 ** -16 + (2 * len(t) + 16) * eps)).t() @ xt.abs()
    ref.check(da[s, rank:], want, ref.U * want.abs() + (1 + ref.U) * off, "da")


def test_adapters_of_many_values(pkg, dev):
    """Slots whose A and B lie past 2^31 values."""
    slots, rank, n, k = 1100, 256, 7680, 7680
    g = torch.Generator().manual_seed(1)
    method, layer, w = ref.make_layer(pkg, "mxfp4", [n], k, dev, g)
    ad = pkg.LowRankAdapters(layer, slots, rank).requires_grad_()
    assert ad.lora_a.numel() > 1 << 31 and ad.lora_b.numel() > 1 << 31
    used = [0, 1091, 1092, 1099]
    for s in used:
        ad.lora_a.data[s] = (torch.randn(rank, k, generator=g) * k ** -0.5).to(dev)
        ad.lora_b.data[s] = torch.randn(n, rank, generator=g).to(dev)
    ad.scaling.fill_(0.5)
    ids = torch.tensor([1099, 0, -1, 1092, 1091, 1099, 1092], device=dev)
    x = torch.randn(7, k, generator=g).bfloat16().to(dev).requires_grad_()
    y = method.apply(layer, x, None, adapters=ad, batch=pkg.AdapterBatch(ids, slots))
    dy = torch.randn(7, n, generator=g).bfloat16().to(dev)
    dx, da, db = torch.autograd.grad(y, [x, ad.lora_a, ad.lora_b], dy)
    base, off = ref.product(ref.quantized("mxfp4", x.detach()), w, scaled=True)
    eps, gx = 2.0 ** -24, dy.double() @ w
    for s in used:
        t = (ids == s).nonzero().squeeze(-1)
        a, b, xt, dt = ad.lora_a[s].double(), ad.lora_b[s].double(), x.detach()[t].double(), dy[t].double()
        v, dv = 0.5 * xt @ a.t(), 0.5 * dt @ b
        vo = 0.5 * (xt.abs() @ a.abs().t()) * ((k + 2) * eps) + v.abs() * (2.0 ** -16 + 2 * rank * eps)
        dvo = 0.5 * (dt.abs() @ b.abs()) * ((n + 2) * eps) + dv.abs() * (2.0 ** -16 + 2 * rank * eps)
        want = base[t] + v @ b.t()
        ref.check(y.detach()[t], want, ref.U * (want.abs() + base[t].abs() * (1 + ref.U)) + (1 + ref.U) * (2 * off[t] + vo @ b.abs().t()))
        want = gx[t] + dv @ a
        ref.check(dx[t], want, ref.U * (want.abs() + 2 * gx[t].abs()) + (1 + ref.U) * (2 * n * eps * (dt.abs() @ w.abs()) + dvo @ a.abs()), "dx")
        want = dv.t() @ xt
        ref.check(da[s], want, ref.U * want.abs() + (1 + ref.U) * (dvo.t() @ xt.abs()) + 1e-30, "da")
        want = dt.t() @ v
        ref.check(db[s], want, ref.U * want.abs() + (1 + ref.U) * (dt.abs().t() @ vo) + 1e-30, "db")
    for s in (1, 1090, 1093, 1098):
        assert not bool(da[s].any()) and not bool(db[s].any())


def test_gated(pkg, dev):
    i = 9216
    g = torch.Generator().manual_seed(2)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [i, i], K, dev, g)
    x = torch.randn(M, K, generator=g).bfloat16().to(dev)
    dh = torch.randn(M, i, dtype=torch.bfloat16, device=dev)
    h = pkg.gated_linear(x, layer)
    both = pkg.ops.gated_grad(x, dh, layer.weight, layer.weight_scale, i, layer.mxl_format)
    assert both.numel() > 1 << 31
    at = _rows(dev)
    # the same rows alone (other tiles, the same sums): within two roundings of bf16
    few, both_few = pkg.gated_linear(x[at], layer), pkg.ops.gated_grad(x[at], dh[at], layer.weight, layer.weight_scale, i, layer.mxl_format)
    for p, q in ((h[at], few), (both[at], both_few)):
        ref.check(p, q.double(), 4 * ref.U * q.double().abs() + 1e-2)
    dx = pkg.ops.input_grad(both, *pkg.adapters.grad_of(layer))
    d = both[at].double()
    ref.check(dx[at], d @ w, ref.U * (d @ w).abs() + (2 * i * 2.0 ** -24) * (1 + ref.U) * (d.abs() @ w.abs()))
