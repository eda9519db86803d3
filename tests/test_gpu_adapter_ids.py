"""The adapters' ids as integers of every type, strides and sources."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int8, torch.int16, torch.int32, torch.int64, torch.uint8, torch.uint16, torch.uint32,
                                   torch.uint64])
@pytest.mark.parametrize("slots", [3, 300])
def test_types(pkg, dev, dtype, slots):
    top = torch.iinfo(dtype).max
    values = [0, 2, 1, min(top, 299), 2, top, 0] + ([] if dtype in (torch.uint8, torch.uint16, torch.uint32, torch.uint64) else [-1, torch.iinfo(dtype).min])
    ids = torch.tensor(values, dtype=dtype).to(dev)
    own = [v if 0 <= v < slots else -1 for v in values]
    _, order, offsets, tiles = pkg.AdapterBatch(ids, slots).tensors
    at = offsets.tolist()
    for s in range(slots):
        assert order[at[s]:at[s + 1]].tolist() == [i for i, v in enumerate(own) if v == s]
    assert at[-1] == sum(v >= 0 for v in own)


def test_strides_and_own_values(pkg, dev):
    ids = torch.randint(-1, 5, (2, 64), device=dev)
    for t in (ids[0], ids.t()[:, 1], ids[:, ::2].reshape(-1)[3:40], ids.int().t()[:, 0]):
        want = pkg.AdapterBatch(t.contiguous(), 5)
        got = pkg.AdapterBatch(t, 5)
        n = int(want.tensors[2][-1])
        assert torch.equal(got.tensors[1][:n], want.tensors[1][:n]) and all(torch.equal(p, q) for p, q in
                                                                            zip(got.tensors[2:], want.tensors[2:]))
        got.update(got.tensors[0])  # its own ids again
        assert torch.equal(got.tensors[0], want.tensors[0]) and torch.equal(got.tensors[3], want.tensors[3])
