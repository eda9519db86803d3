"""What autograd keeps of a layer with adapters: saved-tensor hooks and checkpoints see all of it."""
import pytest
import torch

from test_gpu_adapters import _case, _ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [6, 100])
def test_hooks_see_what_is_kept(pkg, dev, m):
    """Everything of a batch's size that a backward keeps goes through saved-tensor hooks, and comes back through them."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 3, 8, _ids(m, 3, 1), 2, True)
    batch = pkg.AdapterBatch(ids, 3)
    dy = torch.randn(m, 128, generator=g).bfloat16().to(dev)
    leaves = [ad.lora_a, ad.lora_b]
    want = torch.autograd.grad(method.apply(layer, x, None, adapters=ad, batch=batch), leaves, dy)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(tuple(t.shape)), t.cpu())[1], lambda t: t.to(dev)):
        y = method.apply(layer, x, None, adapters=ad, batch=batch)
    got = torch.autograd.grad(y, leaves, dy)
    assert (m, 256) in seen and (m, 32) in seen  # x, and v: two bf16 of 16 padded ranks
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_checkpointed(pkg, dev):
    from torch.utils.checkpoint import checkpoint
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 3, 8, _ids(70, 3, 1), 2, True)
    batch = pkg.AdapterBatch(ids, 3)
    dy = torch.randn(70, 128, generator=g).bfloat16().to(dev)
    leaves = [x.requires_grad_(), ad.lora_a, ad.lora_b]
    f = lambda t: method.apply(layer, t, None, adapters=ad, batch=batch)  # noqa: E731
    want = torch.autograd.grad(f(x), leaves, dy)
    got = torch.autograd.grad(checkpoint(f, x, use_reentrant=False), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
