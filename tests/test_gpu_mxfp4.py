"""MXFP4 on the GPU against the formulas in 64 bits: quantization, SwiGLU producer, products dense and grouped,
layers and experts."""
import math

import pytest
import torch

import mxfp4_reference as ref

pytestmark = pytest.mark.gpu
RULES = (ref.FLOOR_CARRY175, ref.FLOOR_OCP)


def _x(g, m, k):
    x = torch.randn(m, k, generator=g)
    x[:, ::97] *= 20
    return x.bfloat16()


def _equal(got, want):
    for x, y in zip(got, want):
        assert x.dtype == torch.uint8 and torch.equal(x.cpu(), y)


def _weight(pkg, g, n, k):
    codes, scales = ref.random_operand(g, n, k)
    return pkg.ops.pack_weight(codes.cuda(), scales.cuda(), pkg.ops.E2M1), ref.dequantize(codes, scales)


# ------------------------------------------------------------------ quantization

@pytest.mark.parametrize("rule", RULES)
def test_quantize_every_bf16_value(pkg, dev, rule):
    """Every bf16 value as its block's amax and, at every scale it can meet, as another value of the block: the 31
    others lie 0 to 18 powers of two below a larger one."""
    top = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    below = torch.arange(32, dtype=torch.int32)
    bits = top.view(torch.int16).int() & 0xFFFF
    e = (bits >> 7 & 255).unsqueeze(1) - (below * 19 // 32).unsqueeze(0)
    others = torch.where(e > 0, (e << 7) | (bits.unsqueeze(1) * 37 + below * 11 & 127), 0) | (below & 1) << 15
    x = others.to(torch.int16).view(torch.bfloat16)
    x = torch.where((bits >> 7 & 255).unsqueeze(1) < 255, x, torch.ones_like(x))
    x[:, 0] = top
    _equal(pkg.ops.quantize_mxfp4(x.to(dev), rule), ref.quantize(x, rule))


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("m,k", [(1, 32), (3, 96), (17, 2048), (333, 2688), (64, 9216)])
def test_quantize_shapes(pkg, dev, m, k, rule):
    x = _x(torch.Generator().manual_seed(m * k), m, k)
    x[m // 2, :32] = 0.0
    _equal(pkg.ops.quantize_mxfp4(x.to(dev), rule), ref.quantize(x, rule))


def test_quantize_borders(pkg, dev):
    """Ties go to the even code, 1.75 2^e doubles the scale (or saturates), infinities and NaN make the block NaN,
    signed zeros keep their sign."""
    x = torch.zeros(6, 32)
    x[0, :12] = torch.tensor([4.0, .25, .75, 1.25, 1.75, 2.5, 3.5, -0.25, -0.75, -2.5, -3.5, 6.0])
    x[1, :3] = torch.tensor([6.96875, 5.0, -5.0])
    x[2, :3] = torch.tensor([7.0, 5.0, -5.0])
    x[3, :2] = torch.tensor([math.inf, 1.0])
    x[4, :2] = torch.tensor([-1.0, math.nan])
    x[5, :2] = torch.tensor([-0.0, 0.0])
    x = x.bfloat16()
    for rule in RULES:
        codes, scales = pkg.ops.quantize_mxfp4(x.to(dev), rule)
        _equal((codes, scales), ref.quantize(x, rule))
    v = ref.dequantize(*pkg.ops.quantize_mxfp4(x.to(dev), ref.FLOOR_CARRY175))
    assert v[0, :12].tolist() == [4, 0, 1, 1, 2, 2, 4, -0.0, -1, -2, -4, 6]
    assert v[1, :3].tolist() == [6, 4, -4] and v[2, :3].tolist() == [8, 4, -4]
    assert torch.isnan(v[3]).all() and torch.isnan(v[4]).all()
    v = ref.dequantize(*pkg.ops.quantize_mxfp4(x.to(dev), ref.FLOOR_OCP))
    assert v[2, :3].tolist() == [6, 4, -4]


def test_quantize_strides_and_empty(pkg, dev):
    g = torch.Generator().manual_seed(5)
    big = _x(g, 24, 512).to(dev)
    for x in (big[:, 64:320], big[::3, :256], big[:, 8:264], big[:, 3:259], big.t()[:, :0], big[:16].t().contiguous().t()[:, :256]):
        if x.shape[1] == 0:
            continue
        _equal(pkg.ops.quantize_mxfp4(x), ref.quantize(x.contiguous()))
    codes, scales = pkg.ops.quantize_mxfp4(big[:0])
    assert codes.shape == (0, 256) and scales.shape == (0, 16)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("m,k", [(1, 32), (5, 640), (130, 512), (1031, 2560)])
def test_swiglu_producer(pkg, dev, m, k, rule):
    """The quantization of the MXFP8 producer's activation, whose bits the oracle pins; against the float64
    activation a value next to a rounding border may fall to its other side (the device's exp is a binary32 one),
    which moves at most one value in 2^12."""
    x = torch.randn(m, 2 * k, generator=torch.Generator().manual_seed(m + k)).bfloat16()
    x[0, :4] = torch.tensor([100.0, -100.0, 0.0, -0.0]).bfloat16()
    codes, scales = pkg.ops.swiglu_mxfp4(x.to(dev), rule)
    want_codes, want_scales = ref.quantize(ref.silu_activation(x), rule)
    assert (codes.cpu() != want_codes).double().mean() <= 2.0 ** -12
    assert (scales.cpu() != want_scales).double().mean() <= 2.0 ** -12


def test_swiglu_every_gate(pkg, dev, oracle_mod):
    """Every bf16 gate against the activation with the oracle's exp: exact."""
    gates = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, 32)
    up = (torch.randn(2048, 32, generator=torch.Generator().manual_seed(1)) * 2).bfloat16()
    x = torch.cat([gates, up], 1)
    for rule in RULES:
        _equal(pkg.ops.swiglu_mxfp4(x.to(dev), rule), ref.quantize(_activation(oracle_mod, x), rule))


def _activation(oracle_mod, x):
    """bf16(bf16(silu(g)) u) by the oracle's exp: silu(g) = g / (1 + exp(-g)) in binary32."""
    import numpy as np
    f = x.float().numpy()
    g, u = f[:, : f.shape[1] // 2], f[:, f.shape[1] // 2:]
    lib = oracle_mod.lib()
    e = np.array([lib.mxo_exp(float(-v)) for v in g.ravel()], dtype=np.float32).reshape(g.shape)
    with np.errstate(all="ignore"):
        s = torch.from_numpy((g / (np.float32(1) + e)).astype(np.float32)).bfloat16().float().numpy()
        return torch.from_numpy(s * u).bfloat16()


# ------------------------------------------------------------------ dense products

SHAPES = [(1, 16, 128), (1, 8, 256), (2, 2048, 2048), (7, 40, 384), (16, 4608, 2048), (17, 512, 640), (27, 1032, 5120),
          (32, 100, 512), (33, 2048, 1152), (48, 264, 2688), (64, 4100, 512), (65, 128, 256), (100, 1000, 896),
          (128, 2560, 9216), (129, 640, 128), (333, 5120, 2688), (512, 520, 1024), (777, 1030, 384)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm(pkg, dev, m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    (w, sw), wv = _weight(pkg, g, n, k)
    a, sa = ref.random_operand(g, m, k)
    y = pkg.ops.mxfp4_gemm(a.to(dev), sa.to(dev), w, sw, n, k)
    assert y.dtype == torch.bfloat16
    ref.check_product(y, ref.dequantize(a, sa), wv)


@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (5, 100, 640), (48, 1030, 512), (300, 520, 1152), (700, 2048, 512),
                                   (40, 100, 640), (200, 1028, 1152), (1000, 36, 384), (33, 24, 128)])
def test_gemm_bias(pkg, dev, m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    (w, sw), wv = _weight(pkg, g, n, k)
    a, sa = ref.random_operand(g, m, k)
    bias = (torch.randn(n, generator=g) * 50).bfloat16()
    y = pkg.ops.mxfp4_gemm(a.to(dev), sa.to(dev), w, sw, n, k, bias.to(dev))
    ref.check_product(y, ref.dequantize(a, sa), wv, bias)


@pytest.mark.parametrize("m", [1, 20, 64, 200])
def test_gemm_extreme_scales(pkg, dev, m):
    """The largest and smallest scales of either side next to each other, NaN scales only in their own rows and
    columns, in the last K128 slice of a part super-tile too."""
    n, k = 80, 640
    g = torch.Generator().manual_seed(m)
    a, sa = ref.random_operand(g, m, k)
    wc, ws = ref.random_operand(g, n, k)
    sa[0] = 0
    sa[m - 1] = 200
    ws[3] = 1
    ws[5] = 180
    sa[m // 2, k // 32 - 1] = 255
    ws[7, k // 32 - 1] = 255
    ws[n - 1, 0] = 255
    w, sw = pkg.ops.pack_weight(wc.to(dev), ws.to(dev), pkg.ops.E2M1)
    y = pkg.ops.mxfp4_gemm(a.to(dev), sa.to(dev), w, sw, n, k)
    ref.check_product(y, ref.dequantize(a, sa), ref.dequantize(wc, ws))


@pytest.mark.parametrize("m", [1, 16, 30, 64, 150, 600])
def test_gemm_leaves_the_rest(pkg, dev, m):
    """Rows of a wider output keep their other columns, rows behind the last stay as they were, and neither the
    activations' neighbours nor the scales' are read into the sums: all of them hold NaN."""
    n, k, ld = 200, 896, 256
    g = torch.Generator().manual_seed(m)
    (w, sw), wv = _weight(pkg, g, n, k)
    a, sa = ref.random_operand(g, m, k)
    codes = torch.full((m * k // 2 + 4096,), 0x77, dtype=torch.uint8, device=dev)
    scales = torch.full((m * k // 32 + 4096,), 255, dtype=torch.uint8, device=dev)
    codes[: m * k // 2] = a.flatten().to(dev)
    scales[: m * k // 32] = sa.flatten().to(dev)
    out = torch.full((m + 4, ld), 7.0, dtype=torch.bfloat16, device=dev)
    from vllm_mach_amd import _lib
    nbytes = _lib.query("mxl_mxfp4_gemm_workspace_bytes", m, n, k)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
    _lib.call("mxl_mxfp4_gemm", codes.data_ptr(), scales.data_ptr(), m, w.data_ptr(), sw.data_ptr(), n, k, None,
              out.data_ptr(), ld, ws.data_ptr(), nbytes, _lib.stream_handle(out.device))
    ref.check_product(out[:m, :n], ref.dequantize(a, sa), wv)
    assert bool((out[m:] == 7).all()) and bool((out[:, n:] == 7).all())


def test_gemm_unaligned_and_strided_inputs(pkg, dev):
    m, n, k = 9, 72, 256
    g = torch.Generator().manual_seed(2)
    (w, sw), wv = _weight(pkg, g, n, k)
    a, sa = ref.random_operand(g, m, k)
    wide = torch.zeros(m, 300, dtype=torch.uint8, device=dev)
    wide[:, 5:5 + k // 2] = a.to(dev)
    scales = sa.to(dev).t().contiguous().t()
    ref.check_product(pkg.ops.mxfp4_gemm(wide[:, 5:5 + k // 2], scales, w, sw, n, k), ref.dequantize(a, sa), wv)
    assert pkg.ops.mxfp4_gemm(a[:0].to(dev), sa[:0].to(dev), w, sw, n, k).shape == (0, n)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 40, 130])
@pytest.mark.parametrize("n,k", [(16, 128), (72, 896), (4608, 2048), (1030, 5120), (2560, 9216), (104, 16384)])
def test_linear_is_quantizer_and_product(pkg, dev, m, n, k, rule):
    """The layer in one call (one launch for few rows) against its parts.  Sums may be joined in another order; of
    their roundings at most one in 2^7 falls to its other side, by a step."""
    g = torch.Generator().manual_seed(m + n + k)
    (w, sw), wv = _weight(pkg, g, n, k)
    x, bias = _x(g, m, k).to(dev), torch.randn(n, generator=g).bfloat16().to(dev)
    a, sa = pkg.ops.quantize_mxfp4(x, rule)
    for b in (None, bias):
        y, z = pkg.ops.mxfp4_linear(x, w, sw, n, rule, b), pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k, b)
        ref.check_product(y, ref.dequantize(a, sa), wv, b)
        assert float((y != z).double().mean()) <= 2.0 ** -7
    assert torch.equal(torch.ops.mach_amd.mxfp4_linear(x, w, sw, n, rule, bias), y)


def test_operators_under_transforms(pkg, dev):
    """The short way of eager calls is not taken where something looks on: gradients, tracing, compile-time fakes."""
    g = torch.Generator().manual_seed(1)
    (w, sw), _ = _weight(pkg, g, 64, 256)
    x = _x(g, 5, 256).to(dev)
    y = pkg.ops.mxfp4_linear(x, w, sw, 64)
    lin = lambda v: pkg.ops.mxfp4_linear(v, w, sw, 64)  # noqa: E731
    assert torch.equal(lin(x.clone().requires_grad_()).detach(), y)
    with torch.no_grad():
        assert torch.equal(lin(x.clone().requires_grad_()), y)
    z = _x(g, 5, 256).to(dev)
    traced = torch.jit.trace(lin, (x,), check_trace=False)
    assert torch.equal(traced(z), lin(z))
    from torch.fx.experimental.proxy_tensor import make_fx
    assert torch.equal(make_fx(lin)(x)(z), lin(z))
    with torch.inference_mode():
        assert torch.equal(lin(x), y)


@pytest.mark.parametrize("m,n,k", [(16, 40, 20480), (1, 24, 21504), (12, 1000, 17408)])
def test_gemm_past_lds(pkg, dev, m, n, k):
    """Few rows of a K that does not fit in LDS."""
    g = torch.Generator().manual_seed(m + n + k)
    (w, sw), wv = _weight(pkg, g, n, k)
    a, sa = ref.random_operand(g, m, k)
    ref.check_product(pkg.ops.mxfp4_gemm(a.to(dev), sa.to(dev), w, sw, n, k), ref.dequantize(a, sa), wv)


@pytest.mark.parametrize("m,n,k", [(1, 2048, 2048), (40, 1024, 2560), (600, 512, 1024)])
def test_gemm_is_deterministic_and_row_independent(pkg, dev, m, n, k):
    g = torch.Generator().manual_seed(11)
    (w, sw), _ = _weight(pkg, g, n, k)
    a, sa = (t.to(dev) for t in ref.random_operand(g, m, k))
    first = pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k)
    assert torch.equal(first, pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k))


# ------------------------------------------------------------------ layers

def _layer(pkg, codes, scales):
    n, k = codes.shape[0], codes.shape[1] * 2
    method, layer = pkg.MxLinearMethod(pkg.linear.MXFP4_STATIC), torch.nn.Module()
    method.create_weights(layer, k, [n], k, n, torch.bfloat16, device="cuda")
    layer.weight.weight_loader(layer.weight, codes.cuda())
    layer.weight_scale.weight_loader(layer.weight_scale, scales.cuda())
    method.process_weights_after_loading(layer)
    return method, layer


@pytest.mark.parametrize("m", [1, 3, 16, 17, 40, 333])
@pytest.mark.parametrize("n,k", [(200, 384), (2048, 2048)])
def test_linear_layer(pkg, dev, m, n, k):
    g = torch.Generator().manual_seed(m + n)
    codes, scales = ref.random_operand(g, n, k)
    method, layer = _layer(pkg, codes, scales)
    x, bias = _x(g, m, k), torch.randn(n, generator=g).bfloat16()
    a, w = ref.dequantize(*ref.quantize(x)), ref.dequantize(codes, scales)
    ref.check_product(method.apply(layer, x.to(dev)), a, w)
    ref.check_product(method.apply(layer, x.to(dev), bias.to(dev)), a, w, bias)
    # leading dimensions, strided rows, no rows
    y = method.apply(layer, x.to(dev).view(1, m, k))
    assert y.shape == (1, m, n) and torch.equal(y[0], method.apply(layer, x.to(dev)))
    wide = torch.zeros(m, k + 64, dtype=torch.bfloat16, device=dev)
    wide[:, 8:8 + k] = x.to(dev)
    assert torch.equal(method.apply(layer, wide[:, 8:8 + k]), y[0])
    assert method.apply(layer, x[:0].to(dev)).shape == (0, n)


@pytest.mark.parametrize("m", [1, 16, 64])
def test_linear_layer_propagates_nan(pkg, dev, m):
    g = torch.Generator().manual_seed(m)
    codes, scales = ref.random_operand(g, 96, 512)
    method, layer = _layer(pkg, codes, scales)
    x = _x(g, m, 512)
    x[m // 2, 77] = math.nan
    y = method.apply(layer, x.to(dev))
    bad = torch.zeros(m, dtype=torch.bool)
    bad[m // 2] = True
    assert torch.equal(torch.isnan(y).any(1).cpu(), bad) and torch.isnan(y[m // 2]).all()


@pytest.mark.parametrize("m", [1, 5, 100])
def test_swiglu_down(pkg, dev, m):
    g = torch.Generator().manual_seed(m)
    codes, scales = ref.random_operand(g, 264, 640)
    method, layer = _layer(pkg, codes, scales)
    x = torch.randn(m, 1280, generator=g).bfloat16().to(dev)
    a, sa = pkg.ops.swiglu_mxfp4(x)
    y = pkg.swiglu_mxfp4_down(x, layer)
    ref.check_product(y, ref.dequantize(a, sa), ref.dequantize(codes, scales))
    assert torch.equal(pkg.swiglu_mxfp4_down(x.view(1, m, -1), layer)[0], y)
    assert pkg.swiglu_mxfp4_down(x[:0], layer).shape == (0, 264)


# ------------------------------------------------------------------ experts

def _experts(pkg, g, e, h, i):
    c1, s1 = ref.random_operand(g, e * 2 * i, h)
    c2, s2 = ref.random_operand(g, e * h, i)
    c1, s1, c2, s2 = c1.view(e, 2 * i, -1), s1.view(e, 2 * i, -1) - 6, c2.view(e, h, -1), s2.view(e, h, -1) - 6
    experts = pkg.Mxfp4Experts()
    w1, w2 = experts.process_weights_after_loading(c1.cuda(), s1.cuda(), c2.cuda(), s2.cuda())
    return experts, w1, w2, ref.dequantize(c1, s1), ref.dequantize(c2, s2)


def _routes(g, t, e, topk, only=None):
    pool = torch.tensor(only if only else list(range(e)))
    return torch.stack([pool[torch.randperm(len(pool), generator=g)[:topk]] for _ in range(t)]).int()


@pytest.mark.parametrize("t,e,topk,only", [(1, 8, 2, None), (3, 4, 1, [2]), (17, 16, 4, None), (64, 5, 2, [0, 4]),
                                           (150, 3, 2, None), (300, 6, 3, None), (40, 33, 8, None)])
@pytest.mark.parametrize("n,k", [(136, 384), (256, 1024)])
def test_grouped_gemm(pkg, dev, t, e, topk, only, n, k):
    """Experts without rows, with one, with many; gathered rows and rows in order."""
    g = torch.Generator().manual_seed(t + e + n)
    wc, ws = ref.random_operand(g, e * n, k)
    wv = ref.dequantize(wc, ws).view(e, n, k)
    w, sw = pkg.ops.pack_weight(wc.view(e, n, -1).to(dev), ws.view(e, n, -1).to(dev), pkg.ops.E2M1)
    a, sa = ref.random_operand(g, t, k)
    ids = _routes(g, t, e, topk, only)
    routes, offsets, inverse = pkg.ops.moe_route(ids.to(dev), e)
    R = t * topk
    y = pkg.ops.mxfp4_grouped_gemm(a.to(dev), sa.to(dev), routes, topk, offsets, R, w, sw, n, k)
    order, off = routes.cpu().long(), offsets.cpu().tolist()
    rows = ref.dequantize(a, sa)[order // topk]
    for x in range(e):
        ref.check_product(y[off[x]:off[x + 1]], rows[off[x]:off[x + 1]], wv[x])
    b, sb = a[order // topk].to(dev), sa[order // topk].to(dev)
    assert torch.equal(y, pkg.ops.mxfp4_grouped_gemm(b, sb, None, 1, offsets, R, w, sw, n, k))


def test_grouped_gemm_of_many_experts(pkg, dev):
    """More than 1024 experts with many rows each, and as many with few."""
    g = torch.Generator().manual_seed(12)
    e, n, k = 1030, 24, 128
    wc, ws = ref.random_operand(g, e * n, k)
    wv = ref.dequantize(wc, ws).view(e, n, k)
    w, sw = pkg.ops.pack_weight(wc.view(e, n, -1).to(dev), ws.view(e, n, -1).to(dev), pkg.ops.E2M1)
    for t in (17 * e, 40):
        ids = torch.randint(0, e, (t, 1), generator=g).int()
        a, sa = ref.random_operand(g, t, k)
        routes, offsets, _ = pkg.ops.moe_route(ids.to(dev), e)
        y = pkg.ops.mxfp4_grouped_gemm(a.to(dev), sa.to(dev), routes, 1, offsets, t, w, sw, n, k)
        rows, of = ref.dequantize(a, sa)[routes.cpu().long()], ids[routes.cpu().long(), 0].long()
        want = torch.cat([(r.unsqueeze(1) @ wv[o].transpose(1, 2)).squeeze(1) for r, o in zip(rows.split(4096), of.split(4096))])
        assert float((y.cpu().double() - want).abs().max() / want.abs().max()) <= 2.0 ** -8
        assert float((y.cpu().double() - want).norm() / want.norm()) <= 2.0 ** -8


def test_gemm_past_four_gib(pkg, dev):
    """Activation codes past 4 GiB: rows on both sides of the borders and the last ones."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB")
    n, k = 8, 128
    m = (1 << 32) // (k // 2) + 1000
    g = torch.Generator().manual_seed(13)
    (w, sw), wv = _weight(pkg, g, n, k)
    a = torch.randint(0, 256, (m, k // 2), dtype=torch.uint8, device=dev)
    sa = torch.randint(124, 131, (m, k // 32), dtype=torch.uint8, device=dev)
    y = pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k)
    at = torch.cat([torch.arange(0, 300), torch.arange(m // 2, m // 2 + 300), torch.arange(m - 1600, m)]).to(dev)
    ref.check_product(y[at], ref.dequantize(a[at], sa[at]), wv)


def test_grouped_gemm_leaves_dropped_rows(pkg, dev):
    """Routes to no expert end behind the last offset: their output rows are not written."""
    g = torch.Generator().manual_seed(3)
    e, n, k, t = 4, 64, 256, 50
    wc, ws = ref.random_operand(g, e * n, k)
    w, sw = pkg.ops.pack_weight(wc.view(e, n, -1).to(dev), ws.view(e, n, -1).to(dev), pkg.ops.E2M1)
    a, sa = ref.random_operand(g, t, k)
    ids = _routes(g, t, e, 2)
    ids[::3, 1] = -1
    routes, offsets, inverse = pkg.ops.moe_route(ids.to(dev), e)
    kept = int(offsets[-1])
    routes[kept:] = 1 << 30  # whatever the sort left there
    from vllm_mach_amd import _lib
    out = torch.full((t * 2, n), 7.0, dtype=torch.bfloat16, device=dev)
    ad, sd = a.to(dev), sa.to(dev)
    _lib.call("mxl_mxfp4_grouped_gemm", ad.data_ptr(), sd.data_ptr(), t, routes.data_ptr(), 2, offsets.data_ptr(), e, t * 2,
              w.data_ptr(), sw.data_ptr(), n, k, out.data_ptr(), _lib.stream_handle(out.device))
    assert bool((out[kept:] == 7).all()) and not bool((out[:kept] == 7).all(1).any())


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("t,e,topk,only", [(1, 8, 2, None), (2, 40, 3, None), (17, 16, 4, None), (17, 5, 2, [0, 4]),
                                           (32, 33, 8, None), (60, 70, 2, [3, 69])])
@pytest.mark.parametrize("i,k", [(128, 384), (160, 1024), (32, 5120)])
def test_grouped_swiglu_is_the_separate_launches(pkg, dev, t, e, topk, only, i, k, rule):
    """Quantization, gate/up product and SwiGLU producer in one launch.  The two ways may add a K sum's parts in
    another order, so a bf16 gate or up next to a border may fall to its other side and move a code: at most one in
    2^9 codes and scales; decoded, both stand within that of each other."""
    assert pkg.ops.mxfp4_grouped_swiglu_supported(t * topk, e, i, k)
    g = torch.Generator().manual_seed(t + e + i)
    wc, ws = ref.random_operand(g, e * 2 * i, k)
    w, sw = pkg.ops.pack_weight(wc.view(e, 2 * i, -1).to(dev), (ws - 6).view(e, 2 * i, -1).to(dev), pkg.ops.E2M1)
    x = _x(g, t, k).to(dev)
    routes, offsets, _ = pkg.ops.moe_route(_routes(g, t, e, topk, only).to(dev), e)
    R = t * topk
    codes, scales = pkg.ops.mxfp4_grouped_swiglu(x, routes, topk, offsets, R, w, sw, i, rule)
    a, sa = pkg.ops.quantize_mxfp4(x, rule)
    gate_up = pkg.ops.mxfp4_grouped_gemm(a, sa, routes, topk, offsets, R, w, sw, 2 * i, k)
    want = pkg.ops.swiglu_mxfp4(gate_up, rule)
    for u, v in zip((codes, scales), want):
        assert u.shape == v.shape and float((u != v).double().mean()) <= 2.0 ** -9
    u, v = ref.dequantize(codes, scales), ref.dequantize(*want)
    assert float((u - v).norm() / v.norm()) <= 2.0 ** -4


def _exact_layer(x, p, ids, w1, w2):
    a, out = ref.dequantize(*ref.quantize(x)), torch.zeros(x.shape, dtype=torch.float64)
    for e in range(w1.shape[0]):
        t, slot = (ids == e).nonzero(as_tuple=True)
        if len(t):
            mid = (a[t] @ w1[e].t()).bfloat16()
            act = ref.dequantize(*ref.quantize(ref.silu_activation(mid)))
            out.index_add_(0, t, (act @ w2[e].t()).bfloat16().double() * p[t, slot].double().unsqueeze(-1))
    return out


@pytest.mark.parametrize("fuse", [True, False])
@pytest.mark.parametrize("t,e,topk,h,i", [(1, 8, 2, 256, 128), (20, 16, 4, 384, 256), (200, 6, 2, 512, 384),
                                          (2, 300, 8, 256, 128), (600, 16, 4, 1152, 640)])
def test_experts_layer(pkg, dev, t, e, topk, h, i, fuse):
    """The layer against the chain in 64 bits.  Its outputs are sums of bf16 values (half a step each, 2^-8) rounded
    once more, and where a sum in fp32 rounds to another bf16 gate or up value the activation's code can move by a
    step of E2M1, a third of its value: one in 2^10 of them at most, 3 / 2^5 / 2^5 of the norm."""
    g = torch.Generator().manual_seed(t)
    experts, w1, w2, v1, v2 = _experts(pkg, g, e, h, i)
    experts.fuse = fuse
    x, ids = _x(g, t, h), _routes(g, t, e, topk)
    p = torch.rand(t, topk, generator=g)
    got = experts(x.to(dev), w1, w2, p.to(dev), ids.to(dev)).cpu().double()
    want = _exact_layer(x, p, ids, v1, v2)
    assert float((got - want).norm() / want.norm()) <= 2 * 2.0 ** -8 + 2.0 ** -10 * 3


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("t,e,topk,h,i", [(300, 6, 2, 640, 128), (700, 16, 4, 1152, 640), (130, 3, 1, 128, 256),
                                          (900, 5, 3, 2048, 384), (1500, 64, 2, 512, 512)])
def test_swiglu_in_the_tiles_is_the_separate_launches(pkg, dev, t, e, topk, h, i, rule):
    """Many rows an expert: the producer in the epilogue of the gate/up product against a launch of its own, bit for
    bit, with ordinary gates, rows of zeros, gates past the table's both ends and NaN, one expert with most of the
    rows, one with none and some ids of no expert."""
    g = torch.Generator().manual_seed(t + i)
    experts, w1, w2, _, _ = _experts(pkg, g, e, h, i)
    experts.rule = rule
    x = _x(g, t, h)
    x[3::50] = 0.0
    x[4::50] *= 2.0 ** 20
    x[5::50] *= 2.0 ** -30
    x[6, 7] = math.nan
    x[8, 9] = math.inf
    ids = torch.where(torch.rand(t, topk, generator=g) < 0.5, e - 1, torch.randint(0, e - 1, (t, topk), generator=g)).int()
    ids[ids == 0] = -1 if e > 4 else 1
    p = torch.rand(t, topk, generator=g).to(dev)
    args = (x.to(dev), w1, w2, p, ids.to(dev))
    one = experts(*args)
    experts.fuse = False
    two = experts(*args)
    assert torch.equal(one.view(torch.int16), two.view(torch.int16))
    assert bool(one[6].isnan().all()) and not bool(one[10].isnan().any())


@pytest.mark.parametrize("t,e,topk,h,i", [(1, 256, 8, 2048, 512), (2, 6, 2, 128, 128), (4, 4, 4, 640, 384),
                                          (16, 8, 1, 256, 128), (5, 300, 3, 1152, 256), (32, 9, 1, 384, 256),
                                          (1, 1, 1, 128, 128)])
def test_few_routes_unsorted(pkg, dev, t, e, topk, h, i):
    """Up to 32 routes run as they come: the bits of the sorted launches, with an expert twice in a token, ids of no
    expert, a token with nothing but those, strided rows and a NaN row."""
    g = torch.Generator().manual_seed(t + e)
    experts, w1, w2, v1, v2 = _experts(pkg, g, e, h, i)
    wide = _x(g, t, 2 * h).to(dev)
    x, p = wide[:, 8:8 + h], torch.rand(t, topk, generator=g).to(dev)
    ids = torch.randint(0, e, (t, topk), generator=g).int()
    if t > 3:
        ids[0] = -1
        ids[1, 0] = e
        ids[2] = ids[2, 0]
        wide[3, 10] = math.nan
    ids = ids.to(dev)
    got = experts(x, w1, w2, p, ids)
    experts.fuse = False
    want = experts(x, w1, w2, p, ids)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    if t > 3:
        assert bool((got[0] == 0).all())
        assert bool(got[3].isnan().all()) == bool(((ids[3] >= 0) & (ids[3] < e)).any())
    if t < 4:
        exact = _exact_layer(x.cpu(), p.cpu(), ids.cpu(), v1, v2)
        assert float((got.cpu().double() - exact).norm() / exact.norm()) <= 2 * 2.0 ** -8 + 2.0 ** -10 * 3


def test_experts_map_and_method(pkg, dev):
    """An expert map drops the experts of other ranks; the method object runs the same layer."""
    g = torch.Generator().manual_seed(9)
    e, h, i, t, topk = 4, 256, 128, 12, 2
    experts, w1, w2, v1, v2 = _experts(pkg, g, e, h, i)
    x, ids = _x(g, t, h).to(dev), _routes(g, t, 8, topk).to(dev)
    p = torch.rand(t, topk, generator=g).to(dev)
    table = torch.tensor([0, -1, 1, -1, 2, -1, 3, -1], dtype=torch.int32, device=dev)
    out = torch.empty_like(x)
    experts.apply(out, x, w1, w2, p, ids, "silu", 8, table, None, None, None, None, None, False)
    local = table[ids.long()]
    want = _exact_layer(x.cpu(), p.cpu(), local.cpu(), v1, v2)
    keep = (local >= 0).any(1).cpu()
    assert float((out.cpu().double() - want)[keep].norm() / want.norm()) <= 2 * 2.0 ** -8 + 2.0 ** -10 * 3
    assert bool((out.cpu()[~keep] == 0).all())


# ------------------------------------------------------------------ a run of them together

@pytest.mark.parametrize("t", [1, 16, 70])
def test_block_router_experts_linear(pkg, dev, t):
    """As a model's block uses them: a linear layer, the grouped router on its logits, the experts on its routes;
    eager, and captured once and replayed on new inputs with eager work in between."""
    g = torch.Generator().manual_seed(t)
    e, h, i, topk = 16, 256, 128, 4
    experts, w1, w2, v1, v2 = _experts(pkg, g, e, h, i)
    codes, scales = ref.random_operand(g, h, h)
    method, layer = _layer(pkg, codes, scales - 6)
    bias = (torch.randn(e, generator=g) * 0.1).to(dev)
    routing = pkg.GroupedRouting("sigmoid", bias, 4, 2, 2.5)
    xs = [_x(g, t, h).to(dev) for _ in range(4)]
    logits = [torch.randn(t, e, generator=g).to(dev) for _ in range(4)]

    def block(x, z):
        y = method.apply(layer, x)
        out = torch.empty_like(y)
        experts.apply_router(out, y, w1, w2, z, topk, True, routing)
        return y, out

    eager = [[v.clone() for v in block(x, z)] for x, z in zip(xs, logits)]
    for (y, out), x, z in zip(eager, xs, logits):
        ref.check_product(y, ref.dequantize(*ref.quantize(x)), ref.dequantize(codes, scales - 6))
        p, ids = pkg.grouped_topk(z, topk, True, 4, 2, "sigmoid", bias, 2.5)
        assert torch.equal(out, experts(y, w1, w2, p, ids))
        want = _exact_layer(y.cpu(), p.cpu(), ids.cpu(), v1, v2)
        assert float((out.cpu().double() - want).norm() / want.norm()) <= 2 * 2.0 ** -8 + 2.0 ** -10 * 3
    stream, sx, sz = torch.cuda.Stream(), xs[0].clone(), logits[0].clone()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(sx, sz)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = block(sx, sz)
    for (y, out), x, z in list(zip(eager, xs, logits)) * 2:
        sx.copy_(x)
        sz.copy_(z)
        graph.replay()
        block(xs[1], logits[1])  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(captured[0], y) and torch.equal(captured[1], out)


def test_two_streams_at_once(pkg, dev):
    """Calls on two streams use workspaces of their own."""
    g = torch.Generator().manual_seed(4)
    n, k = 512, 4096
    (w, sw), wv = _weight(pkg, g, n, k)
    rows = [tuple(t.to(dev) for t in ref.random_operand(g, m, k)) for m in (40, 70)]
    want = [pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k) for a, sa in rows]
    streams = [torch.cuda.Stream() for _ in rows]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for j, (s, (a, sa)) in enumerate(zip(streams, rows)):
            with torch.cuda.stream(s):
                got[j].append(pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(y, want[j]) for y in got[j])


def test_graphs_of_one_layer_replayed_together(pkg, dev):
    """Graphs of the same layers captured on two streams share no scratch: replayed at once, again and again, with
    eager work between, each gives its own input's result."""
    g = torch.Generator().manual_seed(3)
    e, h, i, topk = 12, 640, 256, 3
    experts, w1, w2, _, _ = _experts(pkg, g, e, h, i)
    codes, scales = ref.random_operand(g, 520, h)
    method, layer = _layer(pkg, codes, scales - 6)
    sets = []
    for t in (400, 9, 150):
        x, z = _x(g, t, h).to(dev), torch.randn(t, e, generator=g).to(dev)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

        def run(x=x, z=z):
            w, ids, routes, offsets, inverse = pkg.ops.moe_router_grouped(z, None, topk, pkg.ops.SIGMOID, 4, 2, True, 1.5)
            return method.apply(layer, x), experts(x, w1, w2, w, ids)

        want = [v.clone() for v in run()]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            run()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = run()
        sets.append((stream, graph, out, want, run))
    torch.cuda.synchronize()
    for _ in range(5):
        for _, _, out, _, _ in sets:
            for v in out:
                v.zero_()
        torch.cuda.synchronize()
        for stream, graph, _, _, _ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = sets[1][4]()
        torch.cuda.synchronize()
        for _, _, out, want, _ in sets:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(eager, sets[1][3]))


def test_warmup_runs_the_layers(pkg, dev):
    """``warmup`` finds prepared MXFP4 layers and experts and runs each; they keep no workspace to reserve."""
    g = torch.Generator().manual_seed(4)
    codes, scales = ref.random_operand(g, 264, 384)
    _, layer = _layer(pkg, codes, scales)
    c1, s1 = ref.random_operand(g, 4 * 256, 256)
    c2, s2 = ref.random_operand(g, 4 * 256, 128)
    method, moe = pkg.Mxfp4MoEMethod(), torch.nn.Module()
    method.create_weights(moe, 4, 256, 128, torch.bfloat16)
    for name, v in (("w13_weight", c1.view(4, 256, -1)), ("w13_weight_scale", s1.view(4, 256, -1)),
                    ("w2_weight", c2.view(4, 256, -1)), ("w2_weight_scale", s2.view(4, 256, -1))):
        getattr(moe, name).data = v.to(dev)
    method.process_weights_after_loading(moe)
    before = pkg.ops.inspect()
    done = pkg.warmup.warmup([layer, moe], (1, 16, 200))
    assert [k[0] for k in done["dense"]] == ["Mxfp4LinearKernel"] and len(done["moe"]) == 1
    assert {1, 16, 64, 128, 200} == set(done["sizes"])
    after = pkg.ops.inspect()
    for op in ("mxfp4_linear", "mxfp4_experts"):
        assert after["counts"][op] - before["counts"].get(op, 0) == 5
    assert after["workspaces"] == before["workspaces"]


def test_gemm_of_codes_past_4_gib(pkg, dev):
    """Rows whose codes pass 32-bit offsets: those around the border and the last against the 64-bit product."""
    g = torch.Generator().manual_seed(6)
    m, n, k = (1 << 20) + 777, 40, 8192
    (w, sw), wv = _weight(pkg, g, n, k)
    border = (1 << 32) // (k // 2)
    rows = torch.cat([torch.arange(40), torch.arange(border - 300, border + 300), torch.arange(m - 40, m)])
    codes, scales = ref.random_operand(g, len(rows), k)
    a, sa = torch.zeros(m, k // 2, dtype=torch.uint8, device=dev), torch.full((m, k // 32), 127, dtype=torch.uint8, device=dev)
    a[rows.to(dev)], sa[rows.to(dev)] = codes.to(dev), scales.to(dev)
    y = pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k)
    ref.check_product(y[rows.to(dev)], ref.dequantize(codes, scales), wv)


# ------------------------------------------------------------------ one rounding with a bias

# by kernel: few rows in one wave and in several over K, tiles with 16- and 8-byte stores and through LDS, a K split
BIASED = [(5, 100, 640), (1, 2048, 2048), (200, 1032, 1152), (200, 1028, 1152), (48, 1030, 512), (17, 256, 8192),
          (40, 130, 8192)]


@pytest.mark.parametrize("m,n,k", BIASED)
def test_bias_joins_the_sum_ahead_of_the_rounding(pkg, dev, m, n, k):
    """A bias next to minus the sums of row 0, whose outputs are what is left of them: an output is off by half a
    step of its own value, not of the sum's, besides fp32's K products (K 2^-23 of their magnitudes) and sum (2^-24)."""
    g = torch.Generator().manual_seed(m + n + k)
    (w, sw), wv = _weight(pkg, g, n, k)
    x = _x(g, m, k)
    a, sa = ref.quantize(x)
    av, wv = ref.dequantize(a, sa).cuda(), wv.cuda()
    sums, most = av @ wv.t(), av.abs() @ wv.abs().t()
    bias = (-sums[0]).bfloat16()
    want = sums + bias.double()
    room = 2.0 ** -8 * want.abs() + (k * 2.0 ** -23 * most + 2.0 ** -24 * want.abs()) * (1 + 2.0 ** -8)
    split = pkg.ops.query("mxl_mxfp4_gemm_workspace_bytes", m, n, k) > 0
    assert split == (k == 8192)
    for y in (pkg.ops.mxfp4_gemm(a.to(dev), sa.to(dev), w, sw, n, k, bias),
              pkg.ops.mxfp4_linear(x.to(dev), w, sw, n, ref.FLOOR_CARRY175, bias)):
        off = (y.double() - want).abs()
        assert bool((off <= room).all()), float((off / room).max())


# ------------------------------------------------------------------ rows far apart, large operands

def _need(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB")


@pytest.mark.parametrize("rows,gib", [((1 << 26) + 999, 6), ((1 << 30) + 999, 72)])
@pytest.mark.parametrize("routed", [20, 9000])
def test_grouped_gemm_of_rows_past_32_bit_offsets(pkg, dev, rows, gib, routed):
    """Activations past 4 GiB, and past 2^32 pieces of 16 bytes, gathered from both sides of the border: few routed
    rows an expert and many."""
    _need(gib)
    e, n, k = 4, 72, 128
    g = torch.Generator().manual_seed(routed)
    wc, ws = ref.random_operand(g, e * n, k)
    wv = ref.dequantize(wc, ws).view(e, n, k)
    w, sw = pkg.ops.pack_weight(wc.view(e, n, -1).to(dev), ws.view(e, n, -1).to(dev), pkg.ops.E2M1)
    border = 1 << (rows.bit_length() - 1)
    at = torch.cat([torch.arange(999), torch.arange(border - 999, border + 999)])
    codes, scales = ref.random_operand(g, len(at), k)
    a = torch.empty(rows, k // 2, dtype=torch.uint8, device=dev)
    sa = torch.empty(rows, k // 32, dtype=torch.uint8, device=dev)
    a[at.to(dev)], sa[at.to(dev)] = codes.to(dev), scales.to(dev)
    pick = torch.randint(0, len(at), (routed,), generator=g)
    offsets = torch.arange(e + 1) * routed // e
    y = pkg.ops.mxfp4_grouped_gemm(a, sa, at[pick].int().to(dev), 1, offsets.to(dev), routed, w, sw, n, k)
    values = ref.dequantize(codes, scales)[pick]
    for x in range(e):
        lo, hi = offsets[x], offsets[x + 1]
        ref.check_product(y[lo:hi], values[lo:hi], wv[x])


# ------------------------------------------------------------------ the routes sorted and as they come

@pytest.mark.parametrize("t,e,topk,h,i", [(16, 8, 2, 2048, 128), (8, 3, 2, 1024, 1024), (16, 5, 2, 2048, 512),
                                          (4, 8, 8, 5120, 128), (1, 8, 4, 2048, 512)])
def test_experts_of_a_router_and_of_its_ids_give_the_same_bits(pkg, dev, t, e, topk, h, i):
    """``apply_router`` (sorted routes) against ``apply`` of the same ids (up to 32 routes as they come), where the order
    of a K sum shows: half of K cancels the other's large values, which cost the rest of the sum its low bits."""
    g = torch.Generator().manual_seed(t + e + h)
    c1, s1 = ref.random_operand(g, e * 2 * i, h)
    c2, s2 = ref.random_operand(g, e * h, i)
    c1, s1, c2, s2 = c1.view(e, 2 * i, -1), s1.view(e, 2 * i, -1) - 8, c2.view(e, h, -1), s2.view(e, h, -1) - 6
    half = h // 2  # 32 columns in the middle: the weights of the first 32
    c1[..., half // 2:half // 2 + 16], s1[..., half // 32] = c1[..., :16], s1[..., 0]
    experts = pkg.Mxfp4Experts()
    w1, w2 = experts.process_weights_after_loading(c1.to(dev), s1.to(dev), c2.to(dev), s2.to(dev))
    x = _x(g, t, h)
    x[:, :32] *= 2.0 ** 18
    x[:, half:half + 32] = -x[:, :32]
    x, z = x.to(dev), torch.randn(t, e, generator=g).to(dev)
    p, ids = pkg.select_experts(z, topk)
    one, two = experts(x, w1, w2, p, ids), torch.empty_like(x)
    experts.apply_router(two, x, w1, w2, z, topk)
    assert bool(one.isfinite().all()) and torch.equal(one, two)


@pytest.mark.parametrize("m,k", [(16, 2048), (64, 2048), (5, 512)])
@pytest.mark.parametrize("beyond", [-8, 0, 8])
def test_rows_up_to_four_gib_apart(pkg, dev, m, k, beyond):
    """Rows that end within 2^31 values of the first (32-bit byte offsets), by a hair or by a row's, and rows further
    apart: the layer and the experts give what they give for the same rows side by side."""
    _need(16)
    g = torch.Generator().manual_seed(m + k)
    ld = ((1 << 31) - k) // (m - 1) // 8 * 8 + beyond
    x = torch.empty((m - 1) * ld + k, dtype=torch.bfloat16, device=dev).as_strided((m, k), (ld, 1))
    near = _x(g, m, k).to(dev)
    x.copy_(near)
    (w, sw), _ = _weight(pkg, g, 72, k)
    assert torch.equal(pkg.ops.mxfp4_linear(x, w, sw, 72), pkg.ops.mxfp4_linear(near, w, sw, 72))
    _equal(pkg.ops.quantize_mxfp4(x), ref.quantize(near))
    e, topk = 40, 2
    experts, w1, w2, _, _ = _experts(pkg, g, e, k, 128)
    ids, p = _routes(g, m, e, topk).to(dev), torch.rand(m, topk, generator=g).to(dev)
    assert torch.equal(experts(x, w1, w2, p, ids), experts(near, w1, w2, p, ids))
    routes, offsets, _ = pkg.ops.moe_route(ids, e)
    one, two = (pkg.ops.mxfp4_grouped_swiglu(v, routes, topk, offsets, m * topk, w1, experts.w1_scale, 128)
                for v in (x, near))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_pack_experts_past_64_gib(pkg, dev):
    """Experts whose tiled codes together pass 2^32 pieces of 16 bytes: the first, one in the middle, those on both
    sides of the border and the last against each packed by itself."""
    n, k = 8192, 8192
    e = (1 << 36) // (n * k // 2) + 2
    _need(145)
    codes = torch.empty(e, n, k // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(e, n, k // 32, dtype=torch.uint8, device=dev)
    at = [0, e // 2 - 2, e // 2 - 1, e // 2, e - 3, e - 2, e - 1]
    for x in at:
        codes[x].random_(0, 256)
        scales[x].random_(0, 255)
    w, sw = pkg.ops.pack_weight(codes, scales, pkg.ops.E2M1)
    for x in at:
        one, s = pkg.ops.pack_weight(codes[x], scales[x], pkg.ops.E2M1)
        assert torch.equal(w[x], one) and torch.equal(sw[x], s)


def test_rows_past_2_31_values(pkg, dev):
    """Contiguous activations of more than 2^31 values: the rows around the border and the last."""
    m, n, k = (1 << 19) + 999, 40, 4096
    _need(16)
    g = torch.Generator().manual_seed(m)
    (w, sw), wv = _weight(pkg, g, n, k)
    at = torch.cat([torch.arange(300), torch.arange((1 << 19) - 300, (1 << 19) + 300), torch.arange(m - 300, m)])
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=dev)
    rows = _x(g, len(at), k)
    x[at.to(dev)] = rows.to(dev)
    want = ref.quantize(rows)
    _equal([t[at.to(dev)] for t in pkg.ops.quantize_mxfp4(x)], want)
    ref.check_product(pkg.ops.mxfp4_linear(x, w, sw, n)[at.to(dev)], ref.dequantize(*want), wv)


@pytest.mark.parametrize("m,n,k,split", [(16, 264, 1152, False), (5, 2048, 2048, False), (200, 1032, 384, False),
                                         (48, 1030, 640, False), (40, 130, 8192, True)])
def test_rows_do_not_reach_each_other(pkg, dev, m, n, k, split):
    """An output row is that of its own activations, bit for bit, whatever the others hold, NaN scales among them: few
    rows, tiles with an odd number of K128 slices (whose last copy ends in the row behind), a K split."""
    g = torch.Generator().manual_seed(m + n)
    (w, sw), _ = _weight(pkg, g, n, k)
    assert (pkg.ops.query("mxl_mxfp4_gemm_workspace_bytes", m, n, k) > 0) == split
    a, sa = (t.to(dev) for t in ref.random_operand(g, m, k))
    whole = pkg.ops.mxfp4_gemm(a, sa, w, sw, n, k)
    for row in sorted({0, 1, m // 2, m - 2, m - 1}):
        b, sb = (t.to(dev) for t in ref.random_operand(g, m, k, 20))
        sb[row ^ 1 if row ^ 1 < m else row - 1] = 255
        b[row], sb[row] = a[row], sa[row]
        y = pkg.ops.mxfp4_gemm(b, sb, w, sw, n, k)
        assert torch.equal(y[row], whole[row])
        assert bool(y[row ^ 1 if row ^ 1 < m else row - 1].isnan().all())


def test_vmap_and_forward_mode(pkg, dev):
    """Under vmap and forward-mode differentiation the operator itself is called: its values are those of plain calls."""
    g = torch.Generator().manual_seed(2)
    (w, sw), _ = _weight(pkg, g, 64, 256)
    x = _x(g, 6, 256).to(dev)
    lin = lambda v: pkg.ops.mxfp4_linear(v, w, sw, 64)  # noqa: E731
    want = lin(x)
    assert torch.equal(torch.func.vmap(lin)(x.view(2, 3, 256)).flatten(0, 1), torch.cat([lin(x[:3]), lin(x[3:])]))
    assert torch.equal(torch.func.jvp(lin, (x,), (x,))[0], want)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        assert torch.equal(torch.autograd.forward_ad.unpack_dual(lin(dual)).primal, want)


@pytest.mark.parametrize("t,e,topk", [(1, 8, 2), (20, 3, 2), (90, 3, 2)])
def test_experts_wider_than_one_launch(pkg, dev, t, e, topk):
    """Hidden sizes past what a workgroup's waves hold of K: quantizer, product and producer are launches of their own,
    from ids and from a router's logits alike."""
    h, i = 7168, 384
    assert not pkg.ops.mxfp4_grouped_swiglu_supported(t * topk, e, i, h)
    g = torch.Generator().manual_seed(t)
    experts, w1, w2, v1, v2 = _experts(pkg, g, e, h, i)
    x, z = _x(g, t, h), torch.randn(t, e, generator=g).to(dev)
    p, ids = pkg.select_experts(z, topk)
    got, routed = experts(x.to(dev), w1, w2, p, ids), torch.empty(t, h, dtype=torch.bfloat16, device=dev)
    experts.apply_router(routed, x.to(dev), w1, w2, z, topk)
    assert torch.equal(got, routed)
    want = _exact_layer(x, p.cpu(), ids.cpu(), v1, v2)
    # (see test_experts_layer)
    assert float((got.cpu().double() - want).norm() / want.norm()) <= 2 * 2.0 ** -8 + 2.0 ** -10 * 3
