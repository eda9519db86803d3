"""Gated blocks of MX layers, act(x Wg^T) * (x Wu^T), and their gradients against 64 bits."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu
MX = ref.FORMATS[:4]


def _want(fmt, act, x, w):
    """(h, its bound, gate, up, their bounds): a bf16 rounding, and the sums' errors through the product.  The
    activations' own arithmetic is within 2^-16 of |g| (the hardware's exp2 and reciprocal)."""
    i = w.shape[0] // 2
    y, off = ref.product(ref.quantized(fmt, x), w, scaled=True)
    g, u, go, uo = y[:, :i], y[:, i:], off[:, :i], off[:, i:]
    a, _ = ref.act(act, g)
    ao = 1.13 * go + 2.0 ** -16 * g.abs()  # (both activations' slopes are below 1.13)
    h = a * u
    return h, ref.U * h.abs() + (1 + ref.U) * (ao * (u.abs() + uo) + a.abs() * uo) + 1e-30, g, u, go, uo


@pytest.mark.parametrize("fmt", MX)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,i,k", [(1, 64, 128), (3, 192, 640), (17, 256, 1024), (130, 320, 384), (300, 1088, 2688)])
def test_against_64_bits(pkg, dev, fmt, act, m, i, k):
    g = torch.Generator().manual_seed(m + i + k)
    method, layer, w = ref.make_layer(pkg, fmt, [i, i], k, dev, g)
    x = torch.randn(m, k, generator=g).bfloat16().to(dev)
    h = pkg.gated_linear(x, layer, act)
    assert h.shape == (m, i) and h.dtype == torch.bfloat16
    ref.check(h, *_want(fmt, act, x, w)[:2])
    assert torch.equal(h, pkg.gated_linear(x, layer, act))


@pytest.mark.parametrize("fmt,i", [("mxfp4", 16), ("mxfp4", 48), ("mxfp6", 80), ("mxfp6_e3m2", 1040)])
def test_widths_of_sixteen(pkg, dev, fmt, i):
    g = torch.Generator().manual_seed(i)
    method, layer, w = ref.make_layer(pkg, fmt, [i, i], 256, dev, g)
    for m in (2, 70):
        x = torch.randn(m, 256, generator=g).bfloat16().to(dev)
        ref.check(pkg.gated_linear(x, layer), *_want(fmt, "silu", x, w)[:2])


@pytest.mark.parametrize("fmt,m,i,k", [("mxfp8", 1024, 2560, 512), ("mxfp8", 700, 9216, 256), ("mxfp4", 2048, 1536, 512),
                                       ("mxfp6", 513, 4096, 384)])
def test_every_tile(pkg, dev, fmt, m, i, k):
    """Enough rows and columns for the large tiles, whole and in quarters."""
    g = torch.Generator().manual_seed(i)
    method, layer, w = ref.make_layer(pkg, fmt, [i, i], k, dev, g)
    x = torch.randn(m, k, generator=g).bfloat16().to(dev)
    ref.check(pkg.gated_linear(x, layer), *_want(fmt, "silu", x, w)[:2])


@pytest.mark.parametrize("fmt", MX)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,i,k", [(2, 64, 128), (67, 320, 384), (300, 576, 640)])
def test_gradients(pkg, dev, fmt, act, m, i, k):
    """Of both products (``gated_grad``) and of the input: two bf16 roundings on the way to it."""
    gen = torch.Generator().manual_seed(m + i)
    method, layer, w = ref.make_layer(pkg, fmt, [i, i], k, dev, gen)
    x = torch.randn(m, k, generator=gen).bfloat16().to(dev).requires_grad_()
    dh = torch.randn(m, i, generator=gen).bfloat16().to(dev)
    h, bound, g, u, go, uo = _want(fmt, act, x.detach(), w)
    y = pkg.gated_linear(x, layer, act)
    ref.check(y, h, bound)
    a, slope = ref.act(act, g)
    d = dh.double().abs()
    dg, du = dh.double() * u * slope, dh.double() * a
    # (second derivatives of both activations are below 1.2; the slope's arithmetic is within 2^-15 of 1 + |g|)
    so = 1.2 * go + 2.0 ** -15 * (1 + g.abs())
    dgo = ref.U * dg.abs() + (1 + ref.U) * d * (uo * (slope.abs() + so) + u.abs() * so) + 1e-30
    duo = ref.U * du.abs() + (1 + ref.U) * d * (1.13 * go + 2.0 ** -16 * g.abs()) + 1e-30
    w8, sw8, n, kk, f, _ = pkg.adapters.grad_of(layer)
    both = pkg.ops.gated_grad(x.detach(), dh, w8, sw8, i, f, pkg.linear.ACTIVATIONS[act])
    ref.check(both, torch.cat([dg, du], 1), torch.cat([dgo, duo], 1))
    dx, = torch.autograd.grad(y, x, dh)
    want = torch.cat([dg, du], 1) @ w
    off = torch.cat([dgo, duo], 1) @ w.abs() + (2 * i * 2.0 ** -24) * (torch.cat([dg, du], 1).abs() @ w.abs())
    ref.check(dx, want, ref.U * want.abs() + (1 + ref.U) * off)


def test_weight_changed_before_backward(pkg, dev):
    g = torch.Generator().manual_seed(2)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [64, 64], 256, dev, g)
    x = torch.randn(3, 256, generator=g).bfloat16().to(dev).requires_grad_()
    for loss in (pkg.gated_linear(x, layer).sum(), method.apply(layer, x).sum()):
        with torch.no_grad():
            layer.weight[:1].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_extremes(pkg, dev):
    """Gates far out: 0 and the gate itself, with finite slopes; a NaN or infinite row stays a row."""
    n, k = 64, 128
    layer = torch.nn.Module()
    method = pkg.MxLinearMethod(pkg.linear.MXFP8_STATIC)
    method.create_weights(layer, k, [n, n], k, 2 * n, torch.bfloat16, device=dev)
    w = torch.zeros(2 * n, k)
    w[:n, 0] = 1
    w[n:, 1] = 1
    layer.weight.weight_loader(layer.weight, w.to(torch.float8_e4m3fn).to(dev))
    layer.weight_scale.weight_loader(layer.weight_scale, torch.full((2 * n, k // 32), 127, dtype=torch.uint8, device=dev))
    method.process_weights_after_loading(layer)
    x = torch.zeros(6, k)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = 2.0 ** 100, -(2.0 ** 100), 240, -240
    x[0:4, 1] = torch.tensor([2.0 ** 92, 2.0 ** 92, 1.0, 1.0])
    x[4, 0] = float("nan")
    x = x.bfloat16().to(dev)
    for act in ("silu", "gelu_tanh"):
        xg = x.clone().requires_grad_()
        h = pkg.gated_linear(xg, layer, act)
        assert torch.equal(h[2], torch.full_like(h[2], 240)) and bool((h[1] == 0).all())
        assert float(h[3].detach().abs().max()) < 1e-30
        assert bool(h[4].isnan().all()) and bool((h[5] == 0).all())
        both = pkg.ops.gated_grad(x, torch.ones_like(h), layer.weight, layer.weight_scale, n, layer.mxl_format,
                                  pkg.linear.ACTIVATIONS[act])
        assert bool(both[:4].isfinite().all())
        assert torch.equal(both[2, :n], torch.full_like(both[2, :n], 1.0))


def test_shapes_strides_and_device_state(pkg, dev):
    gen = torch.Generator().manual_seed(5)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [128, 128], 256, dev, gen)
    x = torch.randn(2, 5, 256, generator=gen).bfloat16().to(dev)
    h = pkg.gated_linear(x.view(10, 256), layer)
    assert torch.equal(pkg.gated_linear(x, layer), h.view(2, 5, 128))
    wide = torch.randn(10, 300, generator=gen).bfloat16().to(dev)
    wide[:, 3:259] = x.view(10, 256)
    assert torch.equal(pkg.gated_linear(wide[:, 3:259], layer), h)
    assert torch.equal(pkg.gated_linear(x.view(10, 256).t().contiguous().t(), layer), h)
    empty = torch.empty(0, 256, dtype=torch.bfloat16, device=dev, requires_grad=True)
    y = pkg.gated_linear(empty, layer)
    assert y.shape == (0, 128) and torch.autograd.grad(y, empty, y.detach())[0].shape == (0, 256)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        other = pkg.gated_linear(x, layer)
    stream.synchronize()
    assert torch.equal(other.view(10, 128), h)


def test_captured(pkg, dev):
    gen = torch.Generator().manual_seed(6)
    method, layer, w = ref.make_layer(pkg, "mxfp4", [512, 512], 1024, dev, gen)
    x = torch.randn(16, 1024, generator=gen).bfloat16().to(dev)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        pkg.gated_linear(x, layer)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = pkg.gated_linear(x, layer)
    for _ in range(3):
        x.copy_(torch.randn(16, 1024, generator=gen).bfloat16())
        eager = pkg.gated_linear(x, layer)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
