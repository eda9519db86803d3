"""Batches of many tiles: the kernels that take two and four groups of ranks at once, in the product and apart."""
import pytest
import torch

import adapters_reference as ref
from test_gpu_adapters import _case, _check_gradients, _ids, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [16, 24, 40, 64, 120, 256])
@pytest.mark.parametrize("slots", [1, 20])
def test_gradients(pkg, dev, rank, slots):
    case = _case(pkg, dev, "mxfp8", [256, 128], 384, slots, rank, _ids(4200, slots, rank, slots == 1), rank, True)
    _check_gradients(pkg, "mxfp8", *case)


@pytest.mark.parametrize("fmt", ["mxfp4", "block"])
@pytest.mark.parametrize("m,slots,rank", [(4096, 2048, 24), (9000, 17, 72), (33000, 300, 8)])
def test_many_tiles(pkg, dev, fmt, m, slots, rank):
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, [128, 128], 256, slots, rank, _ids(m, slots, m), m)
    bias = torch.randn(256, generator=g).bfloat16().to(dev)
    y = method.apply(layer, x, None, adapters=ad, batch=pkg.AdapterBatch(ids, slots))
    ref.check(y, *_want(fmt, x, w, ad, ids))
    z = method.apply(layer, x, bias, adapters=ad, batch=pkg.AdapterBatch(ids, slots))
    ref.check(z, *_want(fmt, x, w, ad, ids, bias))
