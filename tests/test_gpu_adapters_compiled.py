"""Layers with adapters traced into one graph: forward and gradients, with and without the adapters in the product."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("fmt,m,slots", [("mxfp8", 200, 1), ("mxfp8", 200, 30), ("mxfp6", 7, 3), ("mxfp4", 200, 4), ("mxfp4", 9, 2),
                                         ("block", 100, 2), ("block", 1, 2)])
def test_compiled(pkg, dev, backend, fmt, m, slots):
    torch._dynamo.reset()
    g = torch.Generator().manual_seed(m)
    method, layer, w = ref.make_layer(pkg, fmt, [128, 128], 256, dev, g)
    ad = pkg.LowRankAdapters(layer, slots, 8)
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) / 16)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.fill_(0.5)
    x = torch.randn(m, 256, generator=g).bfloat16().to(dev)
    bias = torch.randn(256, generator=g).bfloat16().to(dev)
    dy = torch.randn(m, 256, generator=g).bfloat16().to(dev)
    batch = pkg.AdapterBatch(torch.randint(-1, slots, (m,), generator=g).to(dev), slots)
    call = lambda t, b: method.apply(layer, t, b, adapters=ad, batch=batch)  # noqa: E731
    traced = torch.compile(call, fullgraph=True, backend=backend)
    for b in (None, bias):
        assert torch.equal(traced(x, b), call(x, b))
    ad.requires_grad_()
    for b in (None, bias, bias.clone().requires_grad_()):
        leaves = [t for t in (x.requires_grad_(), ad.lora_a, ad.lora_b, b) if t is not None and t.requires_grad]
        y, want = traced(x, b), call(x, b)
        assert torch.equal(y, want)
        for p, q in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, leaves, dy)):
            assert torch.equal(p, q)


def test_block_of_a_model(pkg, dev):
    """A gated block and a down projection with adapters in one graph."""
    g = torch.Generator().manual_seed(4)
    _, gate_up, _ = ref.make_layer(pkg, "mxfp8", [256, 256], 128, dev, g)
    method, down, _ = ref.make_layer(pkg, "mxfp8", [128], 256, dev, g)
    ad = pkg.LowRankAdapters(down, 2, 8).requires_grad_()
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) / 16)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.fill_(1)
    batch = pkg.AdapterBatch(torch.randint(-1, 2, (40,), generator=g).to(dev), 2)
    x = torch.randn(40, 128, generator=g).bfloat16().to(dev).requires_grad_()

    def block(t):
        return t + method.apply(down, pkg.gated_linear(t, gate_up), None, adapters=ad, batch=batch)

    torch._dynamo.reset()
    dy = torch.randn(40, 128, generator=g).bfloat16().to(dev)
    y, want = torch.compile(block, fullgraph=True, backend="aot_eager")(x), block(x)
    assert torch.equal(y, want)
    leaves = [x, ad.lora_a, ad.lora_b]
    for p, q in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert torch.equal(p, q)
