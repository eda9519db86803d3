"""An infinity or NaN of one adapter stays with the tokens of that adapter, and within a merged part, whether the layer's
product adds the adapters or a launch of their own; in the input gradient as well."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu
BAD = 1  # the slot that is not finite


def _case(pkg, dev, fmt, widths, k, slots, rank, m):
    g = torch.Generator().manual_seed(m + k + rank)
    method, layer, w = ref.make_layer(pkg, fmt, widths, k, dev, g)
    ad = pkg.LowRankAdapters(layer, slots, rank)
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) * k ** -0.5)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.copy_(torch.rand(slots, generator=g) + 0.5)
    ad.requires_grad_()
    x = torch.randn(m, k, generator=g).bfloat16().to(dev).requires_grad_()
    ids = torch.randint(-1, slots, (m,), generator=g, dtype=torch.int32).to(dev)
    dy = torch.randn(m, sum(widths), generator=g).bfloat16().to(dev)
    batch = pkg.AdapterBatch(ids, slots)

    def step():
        y = method.apply(layer, x, None, adapters=ad, batch=batch)
        return (y.detach(), *torch.autograd.grad(y, [x, ad.lora_a, ad.lora_b], dy))

    step.x, step.dy = x, dy
    return ad, ids, step


CASES = [("mxfp8", [128, 48, 80], 256, 3, 24, 200), ("mxfp6", [256, 128], 384, 3, 16, 200), ("mxfp4", [80, 176], 256, 3, 8, 200),
         ("block", [128, 256], 256, 3, 40, 200), ("mxfp8", [1040, 1520], 256, 3, 16, 1100), ("mxfp4", [2048, 2560], 384, 3, 24, 700),
         # the adapters apart: few rows, and more slots than a product takes
         ("mxfp8", [128, 48, 80], 256, 3, 24, 50), ("mxfp4", [256, 128], 384, 20, 16, 800)]


@pytest.mark.parametrize("fmt,widths,k,slots,rank,m", CASES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_b_stays_with_its_tokens(pkg, dev, fmt, widths, k, slots, rank, m, bad):
    ad, ids, step = _case(pkg, dev, fmt, widths, k, slots, rank, m)
    y, dx, da, db = step()
    for col, j in ((0, 0), (widths[0] - 1, rank - 1), (widths[0], 3), (sum(widths) - 1, 5)):
        kept = ad.lora_b.data[BAD, col, j].clone()
        ad.lora_b.data[BAD, col, j] = bad
        y2, dx2, da2, db2 = step()
        ad.lora_b.data[BAD, col, j] = kept
        mine, cols = ids == BAD, torch.arange(y.shape[1], device=dev) != col
        assert torch.equal(y2[~mine], y[~mine]) and torch.equal(y2[:, cols], y[:, cols])
        assert not bool(y2[mine, col].isfinite().any())
        assert torch.equal(dx2[~mine], dx[~mine]) and not bool(dx2[mine].isfinite().any())  # (its dv, of every column)
        others = torch.arange(slots, device=dev) != BAD
        assert torch.equal(da2[others], da[others]) and torch.equal(db2, db)


@pytest.mark.parametrize("fmt,widths,k,slots,rank,m", CASES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_stays_with_its_tokens(pkg, dev, fmt, widths, k, slots, rank, m, bad):
    ad, ids, step = _case(pkg, dev, fmt, widths, k, slots, rank, m)
    y, dx, da, db = step()
    for row, col in ((0, 0), (rank - 1, k - 1), (rank, 5), (len(widths) * rank - 1, k // 2)):
        kept = ad.lora_a.data[BAD, row, col].clone()
        ad.lora_a.data[BAD, row, col] = bad
        y2, dx2, da2, db2 = step()
        ad.lora_a.data[BAD, row, col] = kept
        mine, part = ids == BAD, row // rank
        of_part = torch.zeros(y.shape[1], dtype=torch.bool, device=dev)
        of_part[ad.cols[part]:ad.cols[part + 1]] = True
        assert torch.equal(y2[~mine], y[~mine]) and torch.equal(y2[:, ~of_part], y[:, ~of_part])
        assert not bool(y2[mine][:, of_part].isfinite().any())
        cols = torch.arange(k, device=dev) != col
        assert torch.equal(dx2[~mine], dx[~mine]) and torch.equal(dx2[:, cols], dx[:, cols])
        assert not bool(dx2[mine, col].isfinite().any())
        others = torch.arange(slots, device=dev) != BAD
        assert torch.equal(da2, da) and torch.equal(db2[others], db[others])


@pytest.mark.parametrize("m", [50, 200])
def test_a_token_stays_in_its_row(pkg, dev, m):
    """A NaN or infinity of x, in batches of both kinds."""
    g = torch.Generator().manual_seed(m)
    method, layer, w = ref.make_layer(pkg, "mxfp8", [128, 128], 256, dev, g)
    ad = pkg.LowRankAdapters(layer, 2, 8)
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) / 16)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.fill_(1)
    x = torch.randn(m, 256, generator=g).bfloat16().to(dev)
    batch = pkg.AdapterBatch(torch.randint(-1, 2, (m,), generator=g).to(dev), 2)
    clean = method.apply(layer, x, None, adapters=ad, batch=batch)
    x[2, 7], x[3, 9] = float("nan"), float("inf")
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    keep = torch.ones(m, dtype=torch.bool, device=dev)
    keep[2:4] = False
    assert torch.equal(y[keep], clean[keep]) and not bool(y[2:4].isfinite().any())


@pytest.mark.parametrize("m,slots", [(4, 2), (50, 2), (200, 3), (800, 20), (1500, 1)])
def test_an_infinity_is_an_infinity(pkg, dev, m, slots):
    """Of B, x and dy: with the sign that the product has in 64 bits."""
    k, n, rank = 256, 128, 16
    ad, ids, step = _case(pkg, dev, "mxfp8", [n], k, slots, rank, m)
    mine = (ids == 0).nonzero().squeeze(-1)
    x, dy = step.x, step.dy
    ad.lora_b.data[0, 5, 3] = 0.5
    scale = ad.scaling[0].double()
    v = scale * (x[mine].double() @ ad.lora_a[0].double().t())
    dv = scale * (dy[mine].double() @ ad.lora_b[0].double())
    for bad in (float("inf"), float("-inf")):
        ad.lora_b.data[0, 5, 3] = bad
        z = step()[0]
        ad.lora_b.data[0, 5, 3] = 0.5
        assert torch.equal(z[mine, 5].double(), bad * v[:, 3].sign())
        kept = ad.lora_a.data[0, 2, 7].clone()
        ad.lora_a.data[0, 2, 7] = bad
        assert torch.equal(step()[1][mine, 7].double(), bad * dv[:, 2].sign())
        ad.lora_a.data[0, 2, 7] = kept
        t = int(mine[-1])
        kept = x.data[t, 9].clone()
        x.data[t, 9] = bad
        assert torch.equal(step()[2][0, :, 9].double(), bad * dv[-1].sign())
        x.data[t, 9] = kept
        kept = dy[t, 6].clone()
        dy[t, 6] = bad
        assert torch.equal(step()[3][0, 6].double(), bad * v[-1].sign())
        dy[t, 6] = kept


@pytest.mark.parametrize("n,m", [(131, 200), (77, 100), (260, 700)])
def test_odd_widths(pkg, dev, n, m):
    """Columns that do not end on a store's: the product's other way out."""
    ad, ids, step = _case(pkg, dev, "block", [n], 256, 3, 24, m)
    y, dx, da, db = step()
    mine, cols = ids == BAD, torch.arange(n, device=dev)
    for col in (0, n // 2, n - 1):
        kept = ad.lora_b.data[BAD, col, 5].clone()
        ad.lora_b.data[BAD, col, 5] = float("inf")
        y2, dx2, da2, db2 = step()
        ad.lora_b.data[BAD, col, 5] = kept
        assert torch.equal(y2[~mine], y[~mine]) and torch.equal(y2[:, cols != col], y[:, cols != col])
        assert not bool(y2[mine, col].isfinite().any())
        assert torch.equal(dx2[~mine], dx[~mine]) and torch.equal(db2, db)
