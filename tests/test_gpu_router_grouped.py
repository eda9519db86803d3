"""The grouped router on the GPU against its formulas in 64 bits: ids and the sort exactly, weights to one fp32
rounding."""
import math

import pytest
import torch

import mxfp4_reference as ref

pytestmark = pytest.mark.gpu


def _check(pkg, logits, bias, topk, sigmoid, groups, keep, renorm, factor):
    T, E = logits.shape
    w, ids, routes, offsets, inverse = pkg.ops.moe_router_grouped(
        logits.cuda(), None if bias is None else bias.cuda(), topk, int(sigmoid), groups, keep, renorm, factor)
    want, want_ids = ref.route(logits, bias, topk, sigmoid, groups, keep, renorm, factor)
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu().long(), torch.from_numpy(want_ids))
    want = torch.from_numpy(want)
    assert w.dtype == torch.float32 and torch.equal(torch.isnan(w.cpu()), torch.isnan(want))
    # one rounding to fp32 (half a step, 2^-24) after sums in binary64; tiny weights round to fp32's subnormal grid
    off = (w.cpu().double() - want).abs().nan_to_num()
    assert bool((off <= (2.0 ** -24 + 1e-12) * want.abs().nan_to_num() + 2.0 ** -150).all())
    flat = ids.cpu().flatten().long()
    order = torch.sort(flat, stable=True).indices
    assert torch.equal(routes.cpu().long(), order)
    assert torch.equal(offsets.cpu(), torch.searchsorted(flat[order], torch.arange(E + 1)))
    assert torch.equal(inverse.cpu().long()[order], torch.arange(T * topk))
    two = pkg.grouped_topk(logits.cuda(), topk, renorm, groups, keep, "sigmoid" if sigmoid else "softmax",
                           None if bias is None else bias.cuda(), factor)
    assert torch.equal(two[0].nan_to_num(), w.nan_to_num()) and torch.equal(two[1], ids)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("T,E,topk,groups,keep", [
    (1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (5, 8, 8, 1, 1), (16, 64, 6, 8, 3), (17, 160, 6, 8, 3), (130, 256, 8, 8, 4),
    (40, 16, 4, 16, 4), (33, 72, 2, 1, 1), (200, 512, 10, 8, 2), (9, 1000, 64, 4, 3), (3, 1024, 8, 64, 8),
    (1, 255, 5, 3, 2), (65, 96, 1, 2, 1), (1100, 24, 3, 4, 2), (2049, 256, 8, 8, 4), (2500, 160, 6, 8, 3),
    (2301, 100, 4, 5, 2)])
def test_router(pkg, dev, T, E, topk, groups, keep, biased, sigmoid):
    g = torch.Generator().manual_seed(T * E + topk)
    x = torch.randn(T, E, generator=g) * 2
    bias = torch.randn(E, generator=g) * 0.1 if biased else None
    for bf16 in (False, True):
        _check(pkg, x.bfloat16() if bf16 else x, bias, topk, sigmoid, groups, keep, not bf16, 2.5 if biased else 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_ties_go_to_the_lower_index(pkg, dev, groups, keep, sigmoid):
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-1, 2, (50, 32), generator=g).float()
    x[0] = 0.0
    _check(pkg, x, None, 6, sigmoid, groups, keep, True, 1.0)
    bias = torch.randint(0, 2, (32,), generator=g).float()
    _check(pkg, x, bias, 6, sigmoid, groups, keep, True, 1.0)


def test_scores_closer_than_an_fp32_step(pkg, dev):
    """Sigmoid scores near 1 that are equal in fp32 and not in 64 bits are told apart."""
    x = torch.stack([torch.linspace(18.0, 20.0, 32).flip(0), torch.linspace(30.0, 31.0, 32)])
    _check(pkg, x, None, 8, True, 4, 2, True, 1.0)
    _check(pkg, x, torch.full((32,), 0.5), 8, True, 4, 2, True, 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups,keep", [(1, 1), (8, 3)])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("T,E", [(400, 64), (400, 96), (2200, 96)])
def test_calls_closer_than_binary32(pkg, dev, T, E, biased, groups, keep, sigmoid):
    """Scores that binary32 cannot order, in the middle of the choice, at its end and between groups: logits a few
    steps of fp32 apart, with biases that make up for them."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(T, E, generator=g)
    steps = torch.randint(0, 4, (T, E), generator=g).float() * 2.0 ** -22
    x = (x * 4).round() / 4 + steps
    bias = (torch.randn(E, generator=g) * 8).round() / 64 + torch.randint(0, 3, (E,), generator=g) * 2.0 ** -26 if biased else None
    _check(pkg, x, bias, 6, sigmoid, groups, keep, True, 1.0)
    _check(pkg, x * 30, bias, 6, sigmoid, groups, keep, False, 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T", [70, 2100])
@pytest.mark.parametrize("E,groups,keep", [(32, 4, 2), (60, 5, 3), (256, 8, 4), (640, 1, 1)])
def test_zeros_of_both_signs_and_tiny_logits_tie(pkg, dev, E, groups, keep, T, sigmoid):
    """Logits whose exponentials are equal in 64 bits: -0 and 0, subnormals, and (sigmoid) those far above 37."""
    g = torch.Generator().manual_seed(5)
    pool = torch.tensor([0.0, -0.0, 1e-40, -1e-40, 1e-30] + ([100.0, 101.0] if sigmoid else []))
    x = pool[torch.randint(0, len(pool), (T, E), generator=g)]
    _check(pkg, x, None, 6, sigmoid, groups, keep, True, 1.0)
    _check(pkg, x.bfloat16(), None, 6, sigmoid, groups, keep, True, 1.0)
    _check(pkg, x, torch.zeros(E), 6, sigmoid, groups, keep, True, 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_large_biases(pkg, dev, sigmoid):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(64, 96, generator=g)
    for scale in (1e3, 1e6, 1e30):
        _check(pkg, x, torch.randn(96, generator=g) * scale, 7, sigmoid, 4, 2, True, 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_masked_infinite_and_nan_logits(pkg, dev, sigmoid):
    """Masked experts (-inf, the lowest finite value), infinities and NaN; a row with nothing left but masks."""
    low = torch.finfo(torch.float32).min
    g = torch.Generator().manual_seed(2)
    x = torch.randn(8, 32, generator=g)
    x[0, 5:] = -math.inf
    x[1, 3:] = low
    x[2] = -math.inf
    x[3] = low
    x[4, 7] = math.inf
    x[5, 9] = math.nan
    x[6] = math.nan
    x[7, ::2] = 800.0
    for bias in (None, torch.randn(32, generator=g) * 0.1):
        for groups, keep in ((1, 1), (8, 3)):
            _check(pkg, x, bias, 4, sigmoid, groups, keep, True, 1.0)


def test_infinite_and_nan_bias(pkg, dev):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 32, generator=g)
    bias = torch.randn(32, generator=g) * 0.1
    bias[3], bias[9], bias[10], bias[20], bias[21] = -math.inf, math.nan, math.inf, math.inf, -math.inf
    _check(pkg, x, bias, 5, True, 8, 4, True, 2.5)


def test_strided_logits_and_no_tokens(pkg, dev):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(40, 64, generator=g)
    a = pkg.ops.moe_router_grouped(x.cuda()[::2, 8:40], None, 4, 1, 4, 2)
    b = pkg.ops.moe_router_grouped(x[::2, 8:40].contiguous().cuda(), None, 4, 1, 4, 2)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    w, ids, routes, offsets, inverse = pkg.ops.moe_router_grouped(x[:0].cuda(), None, 4)
    assert w.shape == (0, 4) and routes.numel() == 0 and offsets.tolist() == [0] * 65


def test_softmax_without_groups_is_the_router(pkg, dev):
    """The same experts as the softmax router's, and its weights to fp32's accuracy: an exp (two roundings there and
    the division's), a sum of up to 8 terms."""
    x = torch.randn(300, 256, generator=torch.Generator().manual_seed(6)).cuda()
    a, b = pkg.ops.moe_router_grouped(x, None, 8), pkg.ops.moe_router(x, 8)
    assert all(torch.equal(u, v) for u, v in zip(a[1:], b[1:]))
    assert bool(((a[0] - b[0]).abs() <= 16 * 2.0 ** -24 * a[0]).all())


def test_mxfp6_experts_take_the_routing(pkg, dev):
    g = torch.Generator().manual_seed(8)
    e, h, i, t = 8, 256, 128, 12
    packed = lambda n, k: torch.randint(0, 256, (e, n, k * 3 // 4), generator=g, dtype=torch.uint8).cuda()  # noqa: E731
    scales = lambda n, k: torch.full((e, n, k // 32), 118, dtype=torch.uint8).cuda()  # noqa: E731
    experts = pkg.Mxfp6Experts(fmt=2)
    w1, w2 = experts.process_weights_after_loading(packed(2 * i, h), scales(2 * i, h), packed(h, i), scales(h, i))
    x, z = torch.randn(t, h, generator=g).bfloat16().cuda(), torch.randn(t, e, generator=g).cuda()
    bias = (torch.randn(e, generator=g) * 0.1).cuda()
    out = torch.empty_like(x)
    experts.apply_router(out, x, w1, w2, z, 3, True, pkg.GroupedRouting("sigmoid", bias, 4, 2, 2.5))
    p, ids = pkg.grouped_topk(z, 3, True, 4, 2, "sigmoid", bias, 2.5)
    assert torch.equal(out, experts(x, w1, w2, p, ids))


@pytest.mark.parametrize("T,E,groups", [(20, 256, 8), (3000, 64, 4), (7, 512, 1)])
def test_operands_off_their_alignment(pkg, dev, T, E, groups):
    """Logits and a bias that start one element behind an aligned address."""
    g = torch.Generator().manual_seed(T)
    x, bias = torch.randn(T * E + 1, generator=g).cuda(), (torch.randn(E + 1, generator=g) * 0.1).cuda()
    for cast in (torch.float32, torch.bfloat16):
        xs = x.to(cast)
        off, aligned = xs[1:].view(T, E), xs[1:].view(T, E).clone()
        a = pkg.ops.moe_router_grouped(off, bias[1:], 4, 1, groups, 1, True, 1.0)
        b = pkg.ops.moe_router_grouped(aligned, bias[1:].clone(), 4, 1, groups, 1, True, 1.0)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        _check(pkg, off.cpu(), bias[1:].cpu(), 4, True, groups, 1, True, 1.0)


def test_a_token_routes_alike_in_any_batch(pkg, dev):
    """The choices of a token do not depend on the tokens beside it, nor on which of the layouts their number takes."""
    g = torch.Generator().manual_seed(2)
    x, bias = torch.randn(5000, 192, generator=g).cuda(), (torch.randn(192, generator=g) * 0.1).cuda()
    whole = pkg.ops.moe_router_grouped(x, bias, 6, 1, 8, 3, True, 2.0)
    for lo, hi in ((0, 1), (5, 21), (100, 1100), (4990, 5000)):
        part = pkg.ops.moe_router_grouped(x[lo:hi], bias, 6, 1, 8, 3, True, 2.0)
        assert torch.equal(part[1], whole[1][lo:hi])
        # (binary64 sums in another order, then one rounding to fp32)
        assert bool(((part[0] - whole[0][lo:hi]).abs() <= 2.0 ** -23 * whole[0][lo:hi]).all())


@pytest.mark.parametrize("T", [1, 40, 3000])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_group_scores_past_the_largest_fp32(pkg, dev, T, sigmoid):
    """Biases whose sum of two passes the largest fp32 value, in every group: the groups' order is that of the sums."""
    g = torch.Generator().manual_seed(T)
    top = torch.finfo(torch.float32).max
    # groups of two, of which the second has the larger sum (-1.03 of `top`) and not the larger value
    bias = torch.tensor([-.3, -.75, -.31, -.72, -.4, -.7, -.33, -.73]) * top
    for keep, topk in ((1, 1), (1, 2), (2, 1), (3, 3)):
        _check(pkg, torch.randn(T, 8, generator=g), bias, topk, sigmoid, 4, keep, True, 1.0)
    share = torch.tensor([[.9, .7, .69, .6], [.85, .84, .2, .19], [.95, .94, .93, .92], [1.0, .81, .99, .8]])
    for sign in (-1.0, 1.0):
        bias = (share * top * sign).flatten()
        for keep, topk in ((1, 4), (2, 5), (3, 12)):
            _check(pkg, torch.randn(T, 16, generator=g), bias, topk, sigmoid, 4, keep, True, 1.0)
