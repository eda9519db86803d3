"""Row counts that a layer serves with two-limb activations keep both limbs beside adapters and in gradients."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,slots", [(32, 1), (64, 1), (64, 2), (17, 1), (8, 1)])
def test_adapters_keep_both_limbs(pkg, dev, m, slots):
    g = torch.Generator().manual_seed(m)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [256], 512, dev, g)
    method.kernel = layer.mxl_kernel = pkg.Mxfp8LinearKernel(dual_m=(8, 17, 32, 64))
    ad = pkg.LowRankAdapters(layer, slots, 16)
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) / 16)
    ad.scaling.fill_(1)
    x = torch.randn(m, 512, generator=g).bfloat16().to(dev)
    ids = torch.randint(0, slots, (m,), generator=g).to(dev)
    batch = pkg.AdapterBatch(ids, slots)
    bias = torch.randn(256, generator=g).bfloat16().to(dev)
    for b in (None, bias):  # an adapter of zeros changes nothing
        assert torch.equal(method.apply(layer, x, b, adapters=ad, batch=batch), method.apply(layer, x, b))
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    xg = x.clone().requires_grad_()
    y = method.apply(layer, xg, None, adapters=ad, batch=batch)
    delta, off, _ = ref.adapters(x, ad.lora_a, ad.lora_b, ad.scaling, ids, [256], 16)
    base = method.apply(layer, x).double()
    ref.check(y, base + delta, ref.U * (base + delta).abs() + (1 + ref.U) * off)
    assert torch.equal(y, method.apply(layer, x, None, adapters=ad, batch=batch))
    dx, = torch.autograd.grad(method.apply(layer, xg), xg, torch.ones_like(y))
    assert torch.equal(dx, pkg.ops.input_grad(torch.ones_like(y), *pkg.adapters.grad_of(layer)))


def test_gated_rows(pkg, dev):
    g = torch.Generator().manual_seed(3)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [128, 128], 256, dev, g)
    x = torch.randn(64, 256, generator=g).bfloat16().to(dev)
    want = pkg.gated_linear(x, layer)
    layer.mxl_kernel = pkg.Mxfp8LinearKernel(dual_m=(32, 64))
    for bad in (x, x[:32], x[:32].view(4, 8, 256), x.clone().requires_grad_()):
        with pytest.raises(ValueError, match="one limb"):
            pkg.gated_linear(bad, layer)
    assert torch.equal(pkg.gated_linear(x[:33], layer), want[:33])
