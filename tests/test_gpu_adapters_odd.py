"""Gradients of adapters beside layers whose width is no multiple of eight, and of rows far apart."""
import pytest
import torch

import adapters_reference as ref
from test_gpu_adapters import _case, _check_gradients, _ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 77, 131, 260, 1027])
@pytest.mark.parametrize("m", [5, 150])
def test_odd_widths(pkg, dev, n, m):
    case = _case(pkg, dev, "block", [n], 256, 3, 16, _ids(m, 3, n), n, True)
    _check_gradients(pkg, "block", *case)


def test_odd_widths_one_gradient_at_a_time(pkg, dev):
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "block", [131], 256, 2, 8, _ids(9, 2, 1), 2, True)
    batch = pkg.AdapterBatch(ids, 2)
    bias = torch.randn(131, generator=g).bfloat16().to(dev).requires_grad_()
    leaves = [x.requires_grad_(), ad.lora_a, ad.lora_b, bias]
    dy = torch.randn(9, 131, generator=g).bfloat16().to(dev)
    together = torch.autograd.grad(method.apply(layer, x, bias, adapters=ad, batch=batch), leaves, dy)
    for leaf, want in zip(leaves, together):
        for other in leaves:
            other.requires_grad_(other is leaf)
        one, = torch.autograd.grad(method.apply(layer, x, bias, adapters=ad, batch=batch), leaf, dy)
        assert torch.equal(one, want) and one.shape == leaf.shape and one.is_contiguous()
