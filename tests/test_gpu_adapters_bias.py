"""Biases that no epilogue adds, beside adapters: other types, shapes and strides, with and without gradients."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4", "block"])
@pytest.mark.parametrize("m", [5, 100])
def test_other_biases(pkg, dev, fmt, m):
    g = torch.Generator().manual_seed(m)
    method, layer, w = ref.make_layer(pkg, fmt, [128], 256, dev, g)
    ad = pkg.LowRankAdapters(layer, 2, 8)
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) / 16)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.fill_(1)
    x = torch.randn(m, 256, generator=g).bfloat16().to(dev)
    batch = pkg.AdapterBatch(torch.randint(-1, 2, (m,), generator=g).to(dev), 2)
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    b = torch.randn(128, generator=g).to(dev)
    b16 = b.bfloat16()
    for bias in (b, b.half(), b16[None], b16.repeat_interleave(2)[::2], torch.randn(m, 128, generator=g).to(dev), b[0]):
        want = y + bias
        got = method.apply(layer, x, bias, adapters=ad, batch=batch)
        assert got.dtype == want.dtype and torch.equal(got, want)
        xg, bg = x.clone().requires_grad_(), bias.detach().requires_grad_()  # (of the same strides)
        got = method.apply(layer, xg, bg, adapters=ad, batch=batch)
        assert torch.equal(got, want)
        dx, db = torch.autograd.grad(got, [xg, bg], torch.ones_like(got))
        assert dx.shape == x.shape and db.shape == bias.shape and db.dtype == bias.dtype
