"""The gradient of a layer's bias: column sums, eager and in replays of a captured backward."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu


def _check(got, dy):
    """One rounding; a sum of M terms in 128 rows' shares, 2^-24 of the absolute sum for each of its additions at most."""
    d = dy.double()
    ref.check(got, d.sum(0), ref.U * d.sum(0).abs() + (dy.shape[0] * 2.0 ** -24) * (1 + ref.U) * d.abs().sum(0) + 1e-30)


@pytest.mark.parametrize("m", [0, 1, 2, 127, 128, 129, 1025, 4097])
@pytest.mark.parametrize("n", [1, 7, 8, 64, 72, 131, 1000])
def test_against_64_bits(pkg, dev, m, n):
    g = torch.Generator().manual_seed(m + n)
    dy = torch.randn(m, n, generator=g).bfloat16().to(dev)
    out = pkg.ops.bias_grad(dy)
    assert out.shape == (n,) and out.dtype == torch.bfloat16
    _check(out, dy)
    assert torch.equal(out, pkg.ops.bias_grad(dy))
    wide = torch.full((m, n + 70), float("nan"), dtype=torch.bfloat16, device=dev)
    for at in (0, 3, 8):
        wide[:, at:at + n] = dy
        assert torch.equal(pkg.ops.bias_grad(wide[:, at:at + n]), out)
    assert torch.equal(pkg.ops.bias_grad(dy.t().contiguous().t()), out)


def test_special_values(pkg, dev):
    dy = torch.zeros(300, 80, dtype=torch.bfloat16, device=dev)
    dy[299, 3], dy[0, 79], dy[5, 78], dy[6, 78] = float("nan"), float("inf"), float("inf"), float("-inf")
    out = pkg.ops.bias_grad(dy)
    assert bool(out[3].isnan()) and float(out[79]) == float("inf") and bool(out[78].isnan())
    assert int((out == 0).sum()) == 77
    one = pkg.ops.bias_grad(torch.ones(70000, 8, device=dev).bfloat16()[:, :1].expand(70000, 8))
    assert torch.equal(one, torch.full_like(one, 70000))


@pytest.mark.parametrize("m,n", [(16384, 128), (8192, 1024), (333, 512)])
@pytest.mark.parametrize("adapters", [False, True])
def test_captured(pkg, dev, m, n, adapters):
    """Forward and backward in one graph: every replay has the gradients of its own inputs."""
    g = torch.Generator().manual_seed(n)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [n], 128, dev, g)
    ad = pkg.LowRankAdapters(layer, 1, 8)
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) / 16)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.fill_(1)
    batch = pkg.AdapterBatch(torch.zeros(m, dtype=torch.int32, device=dev), 1)
    x = torch.randn(m, 128, generator=g).bfloat16().to(dev).requires_grad_()
    bias = torch.randn(n, generator=g).bfloat16().to(dev).requires_grad_()
    dy = torch.randn(m, n, generator=g).bfloat16().to(dev)
    more = dict(adapters=ad, batch=batch) if adapters else {}

    def step():
        return torch.autograd.grad(method.apply(layer, x, bias, **more), [x, bias], dy)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for _ in range(4):
        dy.copy_(torch.randn(m, n, generator=g).bfloat16())
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        _check(out[1], dy)


def test_refusals(pkg, dev):
    dy = torch.zeros(4, 16, dtype=torch.bfloat16, device=dev)
    for bad, match in ((dy[0], "bf16"), (dy.float(), "bf16"), (dy[:, :0], "N > 0"), (dy.cpu(), "HIP device")):
        with pytest.raises(ValueError, match=match):
            pkg.ops.bias_grad(bad)
