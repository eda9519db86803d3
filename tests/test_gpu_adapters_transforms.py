"""torch.func's transforms of layers, adapters and gated blocks, and what autograd's hooks see of them."""
import pytest
import torch

import adapters_reference as ref
from test_gpu_adapters import _case, _ids

pytestmark = pytest.mark.gpu


def _layer_case(pkg, dev, fmt="mxfp8"):
    g = torch.Generator().manual_seed(8)
    method, layer, _ = ref.make_layer(pkg, fmt, [64, 64], 256, dev, g)
    x = torch.randn(6, 256, generator=g).bfloat16().to(dev)
    return g, method, layer, x, torch.randn(6, 128, generator=g).bfloat16().to(dev)


def _want(f, x, dy):
    x = x.clone().requires_grad_()
    y = f(x)
    return y.detach(), torch.autograd.grad(y, x, dy)[0]


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4", "block"])
@pytest.mark.parametrize("biased", [False, True])
def test_layers(pkg, dev, fmt, biased):
    if fmt == "block":
        g = torch.Generator().manual_seed(8)
        method, layer, _ = ref.make_layer(pkg, "block", [128], 256, dev, g)
        x, dy = torch.randn(6, 256, generator=g).bfloat16().to(dev), torch.randn(6, 128, generator=g).bfloat16().to(dev)
    else:
        g, method, layer, x, dy = _layer_case(pkg, dev, fmt)
    bias = torch.randn(128, generator=g).bfloat16().to(dev) if biased else None
    f = lambda t: method.apply(layer, t, bias)  # noqa: E731
    y, dx = _want(f, x, dy)
    z, back = torch.func.vjp(f, x)
    assert torch.equal(z, y) and torch.equal(back(dy)[0], dx)
    loss = lambda t, d: (f(t).float() * d.float()).sum()  # noqa: E731
    assert torch.equal(torch.func.grad(loss)(x, dy), dx)
    # gradients of a batch of inputs
    xs, ds = x.view(3, 2, 256), dy.view(3, 2, 128)
    each = torch.stack([_want(f, t, d)[1] for t, d in zip(xs, ds)])
    assert torch.equal(torch.vmap(torch.func.grad(loss))(xs, ds), each)


def test_gated(pkg, dev):
    g, method, layer, x, _ = _layer_case(pkg, dev)
    dh = torch.randn(6, 64, generator=g).bfloat16().to(dev)
    f = lambda t: pkg.gated_linear(t, layer)  # noqa: E731
    y, dx = _want(f, x, dh)
    z, back = torch.func.vjp(f, x)
    assert torch.equal(z, y) and torch.equal(back(dh)[0], dx)
    grad = torch.func.grad(lambda t, d: (f(t).float() * d.float()).sum())
    each = torch.stack([_want(f, t, d)[1] for t, d in zip(x.view(3, 2, 256), dh.view(3, 2, 64))])
    assert torch.equal(torch.vmap(grad)(x.view(3, 2, 256), dh.view(3, 2, 64)), each)


@pytest.mark.parametrize("m", [6, 100])
def test_adapters(pkg, dev, m):
    """In the input, and in the adapters as a function of their values."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 3, 8, _ids(m, 3, 1), 2, True)
    batch = pkg.AdapterBatch(ids, 3)
    dy = torch.randn(m, 128, generator=g).bfloat16().to(dev)
    leaves = [x.requires_grad_(), ad.lora_a, ad.lora_b]
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    want = torch.autograd.grad(y, leaves, dy)
    z, back = torch.func.vjp(lambda t: method.apply(layer, t, None, adapters=ad, batch=batch), x.detach())
    assert torch.equal(z, y) and torch.equal(back(dy)[0], want[0])

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.adapters = ad

        def forward(self, t):
            return method.apply(layer, t, None, adapters=self.adapters, batch=batch)

    block = Block()
    values = {name: p.detach() for name, p in block.named_parameters()}
    got = torch.func.grad(lambda v: (torch.func.functional_call(block, v, (x.detach(),)).float() * dy.float()).sum())(values)
    assert torch.equal(got["adapters.lora_a"], want[1]) and torch.equal(got["adapters.lora_b"], want[2])


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("m", [1, 40])
def test_recorded_layers_save(pkg, dev, fmt, m):
    """A layer recorded with an input that takes a gradient holds operators only, as one without does."""
    import io
    g = torch.Generator().manual_seed(m)
    method, layer, _ = ref.make_layer(pkg, fmt, [128], 256, dev, g)
    x = torch.randn(m, 256, generator=g).bfloat16().to(dev)
    want, file = method.apply(layer, x), io.BytesIO()
    torch.jit.save(torch.jit.trace(lambda t: method.apply(layer, t), x.clone().requires_grad_(), check_trace=False), file)
    file.seek(0)
    with torch.no_grad():
        assert torch.equal(torch.jit.load(file)(x), want)
