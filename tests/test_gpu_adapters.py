"""Low-rank adapters of many requests beside a quantized layer, and their gradients, against 64 bits."""
import pytest
import torch

import adapters_reference as ref

pytestmark = pytest.mark.gpu


def _case(pkg, dev, fmt, widths, k, slots, rank, ids, seed, train=False):
    g = torch.Generator().manual_seed(seed)
    method, layer, w = ref.make_layer(pkg, fmt, widths, k, dev, g)
    ad = pkg.LowRankAdapters(layer, slots, rank)
    ad.lora_a.data.copy_(torch.randn(ad.lora_a.shape, generator=g) * k ** -0.5)
    ad.lora_b.data.copy_(torch.randn(ad.lora_b.shape, generator=g))
    ad.scaling.copy_(torch.rand(slots, generator=g) + 0.5)
    ad.requires_grad_(train)
    x = torch.randn(len(ids), k, generator=g).bfloat16().to(dev)
    return g, method, layer, w, ad, x, torch.as_tensor(ids, dtype=torch.int32).to(dev)


def _want(fmt, x, w, ad, ids, bias=None):
    base, off = ref.product(ref.quantized(fmt, x), w, scaled=True)
    delta, doff, _ = ref.adapters(x, ad.lora_a, ad.lora_b, ad.scaling, ids, ad.widths, ad.rank)
    roundings = 1
    if bias is not None:
        base, roundings = base + bias.double(), 2
    want = base + delta
    # the layer's rounding (twice with a bias), then the sum's
    return want, ref.U * want.abs() + (1 + ref.U) * (roundings * ref.U * (base.abs() + (0 if bias is None else bias.double().abs()))
                                                     + 2 * off + doff) + 1e-30


def _ids(m, slots, seed, runs=False):
    g = torch.Generator().manual_seed(seed)
    if runs:
        return torch.randint(-1, slots, (m // 37 + 1,), generator=g).repeat_interleave(37)[:m]
    return torch.randint(-1, slots, (m,), generator=g)


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("m,widths,k,slots,rank", [(1, [128], 128, 1, 8), (1, [640], 2048, 4, 16), (16, [256, 128], 384, 3, 8),
                                                   (33, [128, 256, 128], 640, 9, 24), (130, [512], 1152, 5, 64),
                                                   (600, [384, 256], 1280, 4, 32)])
def test_against_64_bits(pkg, dev, fmt, m, widths, k, slots, rank):
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, widths, k, slots, rank, _ids(m, slots, m + k), m + k)
    batch = pkg.AdapterBatch(ids, slots)
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    ref.check(y, *_want(fmt, x, w, ad, ids))
    assert torch.equal(y, method.apply(layer, x, None, adapters=ad, batch=batch))
    none = ids < 0
    if not pkg.ops.adapter_linear_supported(m, sum(widths), k, 0, False, slots, len(widths), rank):
        assert torch.equal(y[none], method.apply(layer, x)[none])  # untouched where there is no adapter


@pytest.mark.parametrize("rank", [8, 40, 104, 256])
@pytest.mark.parametrize("m", [5, 700])
def test_ranks(pkg, dev, rank, m):
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128, 128, 128], 256, 3, rank, _ids(m, 3, rank, True), rank)
    y = method.apply(layer, x, None, adapters=ad, batch=pkg.AdapterBatch(ids, 3))
    ref.check(y, *_want("mxfp8", x, w, ad, ids))


@pytest.mark.parametrize("ids,slots", [([-1] * 20, 4), ([3] * 20, 4), ([0], 1), ([-1], 1), ([7, -5, 99, 2 ** 31 - 1, 0, 7], 8),
                                       (list(range(300)) * 2, 300), ([2] * 15 + [0] + [2] * 50, 3), ([5] * 1025, 2000)])
def test_batches(pkg, dev, ids, slots):
    """Nobody with an adapter, all with the same, everybody with another, ids out of range, requests in turns."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp4", [128], 128, slots, 8, ids, len(ids))
    y = method.apply(layer, x, None, adapters=ad, batch=pkg.AdapterBatch(ids, slots))
    ref.check(y, *_want("mxfp4", x, w, ad, torch.where((ids >= 0) & (ids < slots), ids, -1)))


def test_batch_contents(pkg, dev):
    for m, slots in ((1, 1), (100, 7), (513, 40), (5000, 3), (70000, 2048)):
        ids = _ids(m, slots, m).to(dev)
        for kind in (ids.int(), ids.long(), ids.to(torch.int16) if slots < 2 ** 15 else ids.int()):
            b = pkg.AdapterBatch(kind, slots)
            want = torch.sort(torch.where(ids < 0, slots, ids), stable=True)
            n = int((ids >= 0).sum())
            _, order, offsets, tiles_ = b.tensors
            assert torch.equal(order[:n].long(), want.indices[:n])
            assert torch.equal(offsets, torch.searchsorted(want.values[:n].contiguous(), torch.arange(slots + 1, device=dev)))
        at = offsets.tolist()
        tiles = [(s, p, min(p + 16, at[s + 1]), 0) for s in range(slots) for p in range(at[s], at[s + 1], 16)]
        got = [tuple(t) for t in tiles_.tolist()]
        assert got[:len(tiles)] == tiles and all(t[0] == -1 for t in got[len(tiles):])
    big = pkg.AdapterBatch(torch.tensor([2 ** 32, 1, -2 ** 40, 0], device=dev), 2)
    assert big.tensors[2].tolist() == [0, 1, 2] and big.tensors[1][:2].tolist() == [3, 1]


@pytest.mark.parametrize("fmt", ref.FORMATS)
def test_bias_strides_and_shapes(pkg, dev, fmt):
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, [256], 384, 3, 16, _ids(24, 3, 1), 11)
    batch = pkg.AdapterBatch(ids, 3)
    bias = torch.randn(256, generator=g).bfloat16().to(dev)
    y = method.apply(layer, x, bias, adapters=ad, batch=batch)
    ref.check(y, *_want(fmt, x, w, ad, ids, bias))
    assert torch.equal(method.apply(layer, x.view(2, 3, 4, 384), bias, adapters=ad, batch=batch), y.view(2, 3, 4, 256))
    wide = torch.zeros(24, 401, dtype=torch.bfloat16, device=dev)
    wide[:, 5:389] = x
    assert torch.equal(method.apply(layer, wide[:, 5:389], bias, adapters=ad, batch=batch), y)


def test_special_rows(pkg, dev):
    """NaN and infinities stay in their token's row, whichever adapter it shares."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 2, 8, [0, 1, 0, 1, -1, 0], 5)
    batch = pkg.AdapterBatch(ids, 2)
    clean = method.apply(layer, x, None, adapters=ad, batch=batch)
    x[2, 7], x[3, 9] = float("nan"), float("inf")
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    keep = torch.tensor([0, 1, 4, 5], device=dev)
    assert torch.equal(y[keep], clean[keep]) and not bool(y[2].isfinite().any()) and not bool(y[3].isfinite().any())


def test_slots(pkg, dev):
    """load pads smaller ranks, clear takes a slot back; the other slots stay."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128, 256], 256, 3, 16, [0, 1, 2, 1, 0, -1], 9)
    batch = pkg.AdapterBatch(ids, 3)
    before = method.apply(layer, x, None, adapters=ad, batch=batch)
    a, b = torch.randn(6, 256, generator=g), torch.randn(256, 6, generator=g)
    ad.load(1, a.to(dev), b.to(dev), 0.25, part=1)
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    ref.check(y, *_want("mxfp8", x, w, ad, ids))
    keep = ids != 1
    assert torch.equal(y[keep], before[keep])
    assert torch.equal(ad.lora_a[1, 16:22].float(), a.bfloat16().float().to(dev)) and not bool(ad.lora_a[1, 22:].any())
    ad.clear(1)
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    plain = method.apply(layer, x)
    assert torch.equal(y[~keep], plain[~keep])


def _check_gradients(pkg, fmt, g, method, layer, w, ad, x, ids, bias=None):
    x = x.clone().requires_grad_()
    batch = pkg.AdapterBatch(ids, ad.slots)
    y = method.apply(layer, x, bias, adapters=ad, batch=batch)
    ref.check(y.detach(), *_want(fmt, x.detach(), w, ad, ids, bias))
    dy = torch.randn(y.shape, generator=g).bfloat16().to(x.device)
    dx, da, db = torch.autograd.grad(y, [x, ad.lora_a, ad.lora_b], dy)
    xd, a, b, dyd, rank = x.detach().double(), ad.lora_a.double(), ad.lora_b.double(), dy.double(), ad.rank
    m, k, eps = x.shape[0], x.shape[1], 2.0 ** -24
    base, boff = ref.product(dyd, w.t().contiguous())
    want_x, off_x = base.clone(), torch.zeros_like(base)
    want_a, off_a = torch.zeros_like(a), torch.zeros_like(a)
    want_b, off_b = torch.zeros_like(b), torch.zeros_like(b)
    for s in range(ad.slots):
        t, lo, f = (ids == s).nonzero().squeeze(-1), 0, float(ad.scaling[s])
        for p, width in enumerate(ad.widths):
            r0, cols = slice(p * rank, (p + 1) * rank), slice(lo, lo + width)
            ap, bp, gt, xt = a[s, r0], b[s, cols], dyd[t, cols], xd[t]
            v, dv = f * (xt @ ap.t()), f * (gt @ bp)
            # of v and dv: their sums, and 2^-16 that their halves leave out
            vo = f * (xt.abs() @ ap.abs().t()) * ((k + 2) * eps) + v.abs() * 2.0 ** -16
            dvo = f * (gt.abs() @ bp.abs()) * ((width + 2) * eps) + dv.abs() * 2.0 ** -16
            want_x[t] += dv @ ap
            off_x[t] += (dvo + dv.abs() * (2 * len(ad.widths) * rank * eps)) @ ap.abs()
            want_a[s, r0] = dv.t() @ xt
            off_a[s, r0] = (dvo + dv.abs() * ((2 * m + 16) * eps)).t() @ xt.abs()
            want_b[s, cols] = gt.t() @ v
            off_b[s, cols] = gt.abs().t() @ (vo + v.abs() * ((2 * m + 16) * eps))
            lo += width
    ref.check(dx, want_x, ref.U * want_x.abs() + (1 + ref.U) * (ref.U * base.abs() + 2 * boff + off_x) + 1e-30, "dx")
    ref.check(da, want_a, ref.U * want_a.abs() + (1 + ref.U) * off_a + 1e-30, "da")
    ref.check(db, want_b, ref.U * want_b.abs() + (1 + ref.U) * off_b + 1e-30, "db")
    again = torch.autograd.grad(method.apply(layer, x, bias, adapters=ad, batch=batch), [x, ad.lora_a, ad.lora_b], dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, da, db)))


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("m,widths,k,slots,rank", [(1, [128], 128, 1, 8), (35, [128, 256], 384, 3, 24), (200, [512], 640, 4, 16)])
def test_gradients(pkg, dev, fmt, m, widths, k, slots, rank):
    case = _case(pkg, dev, fmt, widths, k, slots, rank, _ids(m, slots, m), m, True)
    _check_gradients(pkg, fmt, *case)


@pytest.mark.parametrize("m,widths,slots,rank,runs", [(1300, [256, 256], 1, 16, True), (777, [128, 384, 128], 6, 64, True),
                                                      (700, [256, 128], 20, 24, False), (520, [256], 2, 256, False), (40, [128, 128, 128], 2, 104, False)])
def test_gradients_of_larger_batches(pkg, dev, m, widths, slots, rank, runs):
    case = _case(pkg, dev, "mxfp8", widths, 384, slots, rank, _ids(m, slots, m, runs), m, True)
    _check_gradients(pkg, "mxfp8", *case)


def test_which_gradients(pkg, dev):
    """Each leaf alone gets the gradient that it gets with the others; a slot without tokens gets zeros; no rows, too."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 3, 8, [0, 2, 2, -1, 0], 2, True)
    batch = pkg.AdapterBatch(ids, 3)
    dy = torch.randn(5, 128, generator=g).bfloat16().to(dev)
    leaves = [x.requires_grad_(), ad.lora_a, ad.lora_b]
    all_ = torch.autograd.grad(method.apply(layer, x, None, adapters=ad, batch=batch), leaves, dy)
    assert not bool(all_[1][1].any()) and not bool(all_[2][1].any()) and bool(all_[1][0].any())
    for i, leaf in enumerate(leaves):
        for other in leaves:
            other.requires_grad_(other is leaf)
        one, = torch.autograd.grad(method.apply(layer, x, None, adapters=ad, batch=batch), leaf, dy)
        assert torch.equal(one, all_[i])
    ad.requires_grad_()
    empty = pkg.AdapterBatch(torch.empty(0, dtype=torch.int32, device=dev), 3)
    y = method.apply(layer, x[:0], None, adapters=ad, batch=empty)
    da, db = torch.autograd.grad(y, [ad.lora_a, ad.lora_b], torch.empty_like(y))
    assert y.shape == (0, 128) and not bool(da.any()) and not bool(db.any())


def test_batch_updated_before_backward(pkg, dev):
    """A batch that is updated between a forward and its backward is refused, not mixed up."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 3, 8, [0, 2, 2, -1, 0], 2, True)
    batch = pkg.AdapterBatch(ids, 3)
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    batch.update(ids.flip(0))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("which", ["scaling", "weight", "scales"])
def test_changed_before_backward(pkg, dev, which):
    """What a backward reads again has to be what its forward read."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp6", [128], 256, 3, 8, [0, 2, 2, -1, 0], 2, True)
    y = method.apply(layer, x, None, adapters=ad, batch=pkg.AdapterBatch(ids, 3))
    with torch.no_grad():
        {"scaling": ad.scaling, "weight": layer.weight, "scales": layer.weight_scale}[which][:1].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("m", [5, 80])
def test_gradient_of_the_bias_alone(pkg, dev, m):
    """Nothing but the bias is trained: in one product (80 rows) and apart (5)."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp4", [128], 256, 2, 8, _ids(m, 2, 1), 2)
    bias, dy = torch.randn(128, generator=g).bfloat16().to(dev), torch.randn(m, 128, generator=g).bfloat16().to(dev)
    batch = pkg.AdapterBatch(ids, 2)
    want = method.apply(layer, x, bias, adapters=ad, batch=batch)
    bias.requires_grad_()
    y = method.apply(layer, x, bias, adapters=ad, batch=batch)
    assert torch.equal(y, want)
    db, = torch.autograd.grad(y, bias, dy)
    ref.check(db, dy.double().sum(0), ref.U * dy.double().sum(0).abs() + m * 2.0 ** -24 * dy.double().abs().sum(0))


def test_apply_counts_as_a_write(pkg, dev):
    """``adapter_apply`` into a tensor that a backward needs is found out."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 2, 8, [0, 1, 1], 2)
    z = torch.randn(3, 128, generator=g).bfloat16().to(dev).requires_grad_()
    y = z.exp()  # (keeps its result)
    with torch.no_grad():
        pkg.ops.adapter_apply(y, x, ad.lora_a, ad.lora_b, ad.scaling, *pkg.AdapterBatch(ids, 2).tensors, ad.cols)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("m,widths,k,slots,rank", [(48, [192, 64], 2560, 32, 24), (2, [128], 5120, 3, 256),
                                                   (16, [64] * 8, 1024, 1, 8), (31, [256], 2176, 2, 40)])
def test_few_rows_of_many_columns(pkg, dev, m, widths, k, slots, rank):
    """The columns in shares over workgroups, joined by the product with b."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", widths, k, slots, rank, _ids(m, slots, 3), m)
    y = method.apply(layer, x, None, adapters=ad, batch=pkg.AdapterBatch(ids, slots))
    ref.check(y, *_want("mxfp8", x, w, ad, ids))


@pytest.mark.parametrize("m,fmt", [(1, "mxfp8"), (40, "mxfp4"), (600, "mxfp6")])
def test_captured(pkg, dev, m, fmt):
    """A captured step, replayed with other inputs and another batch in the same memory; two graphs in turns."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, [256], 512, 4, 16, _ids(m, 4, 1), 3)
    batch = pkg.AdapterBatch(ids, 4)
    stream = torch.cuda.Stream()
    call = lambda: method.apply(layer, x, None, adapters=ad, batch=batch)  # noqa: E731
    graphs = []
    for _ in range(2):
        with torch.cuda.stream(stream):
            call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
        graphs.append((graph, out))
    for i in range(4):
        x.copy_(torch.randn(m, 512, generator=g).bfloat16())
        batch.update(_ids(m, 4, 10 + i).int().to(dev))
        eager = call()
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_captured_batch_and_gradients(pkg, dev):
    """Sorting, forward and backward in one graph, replayed against the eager step."""
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [256, 128], 384, 4, 16, _ids(150, 4, 1), 3, True)
    x.requires_grad_()
    dy = torch.randn(150, 384, generator=g).bfloat16().to(dev)
    batch = pkg.AdapterBatch(ids, 4)

    def step():
        batch.update(ids)
        y = method.apply(layer, x, None, adapters=ad, batch=batch)
        return (y.detach(), *torch.autograd.grad(y, [x, ad.lora_a, ad.lora_b], dy))

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(150, 384, generator=g).bfloat16())
        dy.copy_(torch.randn(150, 384, generator=g).bfloat16())
        ids.copy_(_ids(150, 4, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        with torch.cuda.stream(stream):
            eager = step()
        stream.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, eager))


def test_mlp_with_adapters(pkg, dev):
    """A block as it is used: gate/up with its activation, the down projection with adapters, both directions."""
    g, method, down, w2, ad, h0, ids = _case(pkg, dev, "mxfp8", [256], 512, 3, 8, _ids(50, 3, 4), 21, True)
    _, gate_up, w1 = ref.make_layer(pkg, "mxfp8", [512, 512], 256, dev, g)
    batch = pkg.AdapterBatch(ids, 3)
    x = torch.randn(50, 256, generator=g).bfloat16().to(dev).requires_grad_()
    y = x + method.apply(down, pkg.gated_linear(x, gate_up), None, adapters=ad, batch=batch)
    dy = torch.randn(50, 256, generator=g).bfloat16().to(dev)
    dx, da, db = torch.autograd.grad(y, [x, ad.lora_a, ad.lora_b], dy)
    # the same, operator by operator
    with torch.no_grad():
        h = pkg.gated_linear(x, gate_up)
    hg = h.clone().requires_grad_()
    z = method.apply(down, hg, None, adapters=ad, batch=batch)
    dh, da2, db2 = torch.autograd.grad(z, [hg, ad.lora_a, ad.lora_b], dy)
    assert torch.equal(y.detach(), (x + z).detach()) and torch.equal(da, da2) and torch.equal(db, db2)
    both = pkg.ops.gated_grad(x.detach(), dh, gate_up.weight, gate_up.weight_scale, 512, gate_up.mxl_format)
    assert torch.equal(dx, dy + pkg.ops.input_grad(both, *pkg.adapters.grad_of(gate_up)))


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("m,widths,k,slots,rank,runs", [(33, [128], 128, 1, 8, False), (100, [256, 128], 384, 3, 24, False),
                                                        (300, [1024, 128], 1152, 5, 64, True), (1024, [2560], 256, 2, 16, True),
                                                        (700, [128, 8320], 384, 4, 104, False)])
def test_one_product(pkg, dev, fmt, m, widths, k, slots, rank, runs):
    """The adapters inside the layer's product: one rounding, whichever tile; mixed and whole tiles, with a bias."""
    n = sum(widths)
    assert pkg.ops.adapter_linear_supported(m, n, k, 0, False, slots, len(widths), rank)
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, widths, k, slots, rank, _ids(m, slots, m, runs), m)
    batch = pkg.AdapterBatch(ids, slots)
    base, off = ref.product(ref.quantized(fmt, x), w, scaled=True)
    delta, doff, _ = ref.adapters(x, ad.lora_a, ad.lora_b, ad.scaling, ids, widths, rank)
    want, bound = base + delta, off + doff + 1e-30
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    ref.check(y, want, ref.U * want.abs() + (1 + ref.U) * bound)
    assert torch.equal(y, method.apply(layer, x, None, adapters=ad, batch=batch))
    bias = torch.randn(n, generator=g).bfloat16().to(dev)
    z = method.apply(layer, x, bias, adapters=ad, batch=batch)
    if fmt == "mxfp4":  # (joins the sum)
        ref.check(z, want + bias.double(), ref.U * (want + bias.double()).abs() + (1 + ref.U) * (bound + (want + bias.double()).abs() * 2.0 ** -23))
    else:
        assert torch.equal(z, y + bias)


def test_one_product_of_odd_columns(pkg, dev):
    """A last part whose columns end inside an n-tile, and columns that a tile has beyond the layer's."""
    for fmt, widths in (("mxfp4", [136]), ("mxfp6", [40]), ("block", [32, 99])):
        n = sum(widths)
        g = torch.Generator().manual_seed(n)
        method, layer, w = ref.make_layer(pkg, fmt, [n], 256, dev, g)
        a = (torch.randn(2, len(widths) * 16, 256, generator=g) / 16).bfloat16().to(dev)
        b = torch.randn(2, n, 16, generator=g).bfloat16().to(dev)
        scaling = torch.tensor([0.5, 2.0], device=dev)
        ids = _ids(80, 2, n).int().to(dev)
        x = torch.randn(80, 256, generator=g).bfloat16().to(dev)
        wt, sw, _, k, f, block = pkg.adapters.grad_of(layer)
        cols = [0, *torch.tensor(widths).cumsum(0).tolist()]
        batch = pkg.ops.adapter_batch(ids, 2)
        y, v = pkg.ops.adapter_linear(x, wt, sw, f, block, 0, None, a, b, scaling, *batch, cols)
        base, off = ref.product(ref.quantized(fmt, x), w, scaled=True)
        delta, doff, _ = ref.adapters(x, a, b, scaling, ids, widths, 16)
        ref.check(y, base + delta, ref.U * (base + delta).abs() + (1 + ref.U) * (off + doff))
        z = method.apply(layer, x)
        assert torch.equal(pkg.ops.adapter_apply(z, x, a, b, scaling, *batch, cols)[ids >= 0], v[ids >= 0])
        ref.check(z, base + delta, ref.U * ((base + delta).abs() + base.abs()) + (1 + ref.U) * (2 * off + doff))


def test_refusals(pkg, dev):
    g, method, layer, w, ad, x, ids = _case(pkg, dev, "mxfp8", [128], 256, 3, 8, [0, 1, 2], 1)
    batch = pkg.AdapterBatch(ids, 3)
    call = lambda **kw: method.apply(layer, **{"x": x, "adapters": ad, "batch": batch, **kw})  # noqa: E731
    for kw in (dict(batch=None), dict(adapters=None), dict(batch=ids), dict(adapters=ad.lora_a)):
        with pytest.raises(ValueError, match="go together"):
            call(**kw)
    with pytest.raises(ValueError, match="3 rows"):
        call(x=x[:2])
    with pytest.raises(ValueError, match="bf16"):
        call(x=x.float())
    with pytest.raises(ValueError, match="slots"):
        call(batch=pkg.AdapterBatch(ids, 4))
    _, other, _ = ref.make_layer(pkg, "mxfp8", [256], 256, dev, g)
    with pytest.raises(ValueError, match="not of this layer"):
        call(adapters=pkg.LowRankAdapters(other, 3, 8))
    with pytest.raises(ValueError, match="update needs"):
        batch.update(ids[:2])
    for bad in (ids.float(), ids.view(1, 3), ids.bool()):
        with pytest.raises(ValueError, match="integers"):
            pkg.AdapterBatch(bad, 3)
    for slots in (0, 2049):
        with pytest.raises(ValueError, match="adapters"):
            pkg.AdapterBatch(ids, slots)
    o, t, cols = pkg.ops, batch.tensors, [0, 128]
    y = method.apply(layer, x)
    args = dict(y=y, x=x, a=ad.lora_a, b=ad.lora_b, scaling=ad.scaling, ids=t[0], order=t[1], offsets=t[2], tiles=t[3], cols=cols)
    for name, bad, match in (("a", ad.lora_a[:2], "do not fit"), ("b", ad.lora_b.float(), "bf16"), ("cols", [0, 64], "do not fit"),
                             ("cols", [0, 8, 128], "multiples of 16"), ("scaling", ad.scaling.double(), "scaling"),
                             ("tiles", t[3][:1], "batch"), ("order", t[1].long(), "batch"), ("y", y[:, ::2], "unit column"),
                             ("y", y[:2], "y must be"), ("ids", t[0].cpu(), "HIP device|tensors on")):
        with pytest.raises(ValueError, match=match):
            o.adapter_apply(**{**args, name: bad})
    wt, sw, n, k, f, block = pkg.adapters.grad_of(layer)
    with pytest.raises(ValueError, match="one product"):
        o.adapter_linear(x, wt, sw, f, block, 0, None, ad.lora_a, ad.lora_b, ad.scaling, *t, cols)
    v = o.adapter_apply(**args)
    for dy, vv, match in ((y[:2], v, "rows"), (y.float(), v, "bf16"), (y, v[:, :16], "not adapter_apply's")):
        with pytest.raises(ValueError, match=match):
            o.adapter_grad(dy, x, wt, sw, f, block, ad.lora_a, ad.lora_b, ad.scaling, vv, *t, cols)
    with pytest.raises(ValueError, match="tiled layout"):
        o.input_grad(y, wt[:-1], sw, n, k, f, block)
    with pytest.raises(ValueError, match="tiled layout"):
        o.gated_linear(x, wt, sw[:-1], 64, f)
