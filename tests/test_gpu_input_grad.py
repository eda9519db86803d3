"""The input gradient of frozen quantized layers against the product in 64 bits."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu


def _want(dy, w):
    want, off = ref.product(dy.double(), w.t().contiguous())
    return want, off + ref.U * want.abs() + 1e-30


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (5, 256, 384), (130, 640, 1152), (257, 1280, 640)])
def test_against_64_bits(pkg, dev, fmt, m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    method, layer, w = ref.make_layer(pkg, fmt, [n], k, dev, g)
    dy = torch.randn(m, n, generator=g).bfloat16().to(dev)
    dx = pkg.ops.input_grad(dy, *pkg.adapters.grad_of(layer))
    ref.check(dx, *_want(dy, w))
    assert torch.equal(dx, pkg.ops.input_grad(dy, *pkg.adapters.grad_of(layer)))


@pytest.mark.parametrize("fmt,n", [("mxfp4", 8), ("mxfp4", 24), ("mxfp6", 136), ("mxfp6_e3m2", 1000), ("block", 131), ("block", 77)])
@pytest.mark.parametrize("m", [3, 65])
def test_odd_widths(pkg, dev, fmt, n, m):
    """Rows of W that end inside a stage: what lies behind the last column of dy is not read into the sums."""
    g = torch.Generator().manual_seed(n)
    method, layer, w = ref.make_layer(pkg, fmt, [n], 256, dev, g)
    wide = torch.full((m, n + 64), float("nan"), dtype=torch.bfloat16)
    wide[:, :n] = torch.randn(m, n, generator=g)
    dy = wide.to(dev)[:, :n]
    ref.check(pkg.ops.input_grad(dy, *pkg.adapters.grad_of(layer)), *_want(dy, w))


@pytest.mark.parametrize("m,n,k", [(513, 5120, 2688), (64, 17408, 512), (2048, 1024, 256)])
def test_larger(pkg, dev, m, n, k):
    g = torch.Generator().manual_seed(n)
    for fmt in ("mxfp8", "block", "mxfp4"):
        method, layer, w = ref.make_layer(pkg, fmt, [n], k, dev, g)
        dy = torch.randn(m, n, generator=g).bfloat16().to(dev)
        ref.check(pkg.ops.input_grad(dy, *pkg.adapters.grad_of(layer)), *_want(dy, w), fmt)


def test_special_values(pkg, dev):
    """An infinity or NaN of dy stays in its row, a NaN scale of W in its columns; the smallest and largest scales of
    normal bf16 values are exact."""
    g = torch.Generator().manual_seed(1)
    codes, s, _ = ref.draw_weight("mxfp4", 64, 256, g)
    s[:] = 127
    s[3, 0] = 255
    s[5, 1], s[6, 1] = 3, 250
    layer = torch.nn.Module()
    method = pkg.MxLinearMethod(pkg.linear.MXFP4_STATIC)
    method.create_weights(layer, 256, [64], 256, 64, torch.bfloat16, device=dev)
    layer.weight.weight_loader(layer.weight, codes.to(dev))
    layer.weight_scale.weight_loader(layer.weight_scale, s.to(dev))
    method.process_weights_after_loading(layer)
    dy = torch.zeros(6, 64)
    dy[0, 2], dy[1, 5], dy[2, 6], dy[3, 1] = 1, 2.0 ** 20, 2.0 ** -30, float("nan")
    dx = pkg.ops.input_grad(dy.bfloat16().to(dev), *pkg.adapters.grad_of(layer)).cpu()
    t = torch.cat([ref._E2M1, -ref._E2M1])
    c = torch.stack([codes & 15, codes >> 4], -1).view(64, 256).long()
    assert bool(dx[3].isnan().all())
    assert bool(dx[:, :32].isnan().all())  # 0 times the NaN block
    assert torch.equal(dx[0, 32:].double(), t[c[2, 32:]])
    assert torch.equal(dx[1, 32:64].double(), t[c[5, 32:64]] * 2.0 ** (20 + 3 - 127))
    assert torch.equal(dx[2, 32:64].double(), t[c[6, 32:64]] * 2.0 ** (250 - 127 - 30))


@pytest.mark.parametrize("fmt", ref.FORMATS)
def test_autograd_of_a_layer(pkg, dev, fmt):
    """``apply`` differentiates in x (any leading shape, no rows, a bias with and without gradient) and computes what it
    does without gradients."""
    g = torch.Generator().manual_seed(7)
    method, layer, w = ref.make_layer(pkg, fmt, [256], 384, dev, g)
    bias = torch.randn(256, generator=g).bfloat16().to(dev)
    for shape in ((3, 7, 384), (33, 384), (384,), (0, 384)):
        x = torch.randn(*shape, generator=g).bfloat16().to(dev)
        for b in (None, bias, bias.clone().requires_grad_()):
            xg = x.clone().requires_grad_()
            y = method.apply(layer, xg, b)
            with torch.no_grad():
                assert torch.equal(y, method.apply(layer, x, b))
            dy = torch.randn(*shape[:-1], 256, generator=g).bfloat16().to(dev)
            dx, = torch.autograd.grad(y, xg, dy)
            assert dx.shape == x.shape
            ref.check(dx.view(-1, 384), *_want(dy.view(-1, 256), w))


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4", "block"])
def test_compiled(pkg, dev, fmt):
    """One graph of a layer whose input takes a gradient."""
    g = torch.Generator().manual_seed(9)
    method, layer, w = ref.make_layer(pkg, fmt, [128], 256, dev, g)
    x = torch.randn(40, 256, generator=g).bfloat16().to(dev).requires_grad_()
    dy = torch.randn(40, 128, generator=g).bfloat16().to(dev)
    y, want = torch.compile(lambda t: method.apply(layer, t), fullgraph=True, backend="eager")(x), method.apply(layer, x)
    assert torch.equal(y, want)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(want, x, dy)[0])


def test_gradient_of_an_expanded_output(pkg, dev):
    """A gradient that autograd hands over expanded (of a sum) or transposed."""
    g = torch.Generator().manual_seed(3)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [128], 256, dev, g)
    x = torch.randn(9, 256, generator=g).bfloat16().to(dev).requires_grad_()
    dx, = torch.autograd.grad(method.apply(layer, x).sum(), x)
    ref.check(dx, *_want(torch.ones(9, 128, device=dev), w))
    dyt = torch.randn(128, 9, generator=g).bfloat16().to(dev)
    dx, = torch.autograd.grad(method.apply(layer, x), x, dyt.t())
    ref.check(dx, *_want(dyt.t(), w))
