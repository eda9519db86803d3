"""The token sort of many chunks of 1024 routes: a stable sort by expert, routes outside the experts dropped."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,topk,E", [
    (0, 2, 2000), (3, 1, 2560), (40000, 1, 1), (34000, 1, 3), (5000, 8, 17), (16384, 8, 256), (131072, 1, 256),
    (50000, 8, 1024), (9000, 8, 1025), (20001, 5, 2560), (600000, 1, 40), (7000, 8, 256), (5120, 8, 256),
    (6144, 8, 60), (6145, 8, 256), (4096, 8, 1000), (4097, 8, 1000), (16384, 8, 64)])
def test_sort_of_many_chunks(pkg, dev, T, topk, E):
    g = torch.Generator().manual_seed(T + E)
    ids = torch.randint(0, E, (T, topk), generator=g, dtype=torch.int32)
    if T > 100:
        ids[7:90] = E // 2  # a run of one expert
        ids[50, 0] = -1
        ids[-1, -1] = E
    routes, offsets, inverse = (t.cpu().long() for t in torch.ops.mach_amd.moe_route(ids.to(dev), E))
    flat = ids.flatten().long()
    real = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(real, stable=True).indices
    count = int((real < E).sum())
    assert torch.equal(offsets, torch.searchsorted(real[order], torch.arange(E + 1)))
    assert torch.equal(routes[:count], order[:count])
    want = torch.full((T * topk,), -1)
    want[order[:count]] = torch.arange(count)
    assert torch.equal(inverse, want)
