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


def test_rows_far_apart(pkg, dev):
    """Gradients, inputs and outputs whose rows lie more than 2^22 values apart."""
    far = (1 << 22) + 64
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 2, 8, [0, 1, -1], 2, True)
    dy = torch.randn(3, 128, generator=g).bfloat16().to(dev)
    apart = lambda t: torch.zeros(3, far, dtype=torch.bfloat16, device=dev)[:, :t.shape[1]].copy_(t)  # noqa: E731
    of = pkg.adapters.grad_of(layer)
    assert torch.equal(pkg.ops.input_grad(apart(dy), *of), pkg.ops.input_grad(dy, *of))
    assert torch.equal(pkg.ops.bias_grad(apart(dy)), pkg.ops.bias_grad(dy))
    batch = pkg.AdapterBatch(ids, 2)
    bias = torch.randn(128, generator=g).bfloat16().to(dev).requires_grad_()
    near, wide = x.clone().requires_grad_(), apart(x).detach().requires_grad_()
    results = []
    for t, d in ((near, dy), (wide, dy), (near, apart(dy)), (wide, apart(dy))):
        y = method.apply(layer, t, bias, adapters=ad, batch=batch)
        results.append((y, *torch.autograd.grad(y, [t, ad.lora_a, ad.lora_b, bias], d)))
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(other, results[0]))
    gate_up = ref.make_layer(pkg, "mxfp8", [64, 64], 256, dev, g)[1]
    dh = dy[:, :64].contiguous()
    want = torch.autograd.grad(pkg.gated_linear(near, gate_up), near, dh)[0]
    assert torch.equal(torch.autograd.grad(pkg.gated_linear(wide, gate_up), wide, apart(dh))[0], want)
