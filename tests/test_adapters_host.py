"""CPU checks of the adapters, gated blocks and input gradients: refusals before any launch, shapes under tracing, and
the 64-bit definitions that the GPU tests compare with."""
import ctypes

import pytest
import torch

import adapters_reference as ref


def _prepared(n=128, k=256, widths=None):
    layer = torch.nn.Module()
    layer.mxl_shape, layer.mxl_format = (n, k), 0
    layer.weight = torch.nn.Parameter(torch.zeros(1), requires_grad=False)
    layer.weight_scale = layer.weight
    if widths:
        layer.logical_widths = widths
    return layer


def test_adapter_set_refusals(pkg):
    with pytest.raises(ValueError, match="prepared"):
        pkg.LowRankAdapters(torch.nn.Module(), 2, 8)
    for rank in (0, 4, 12, 264):
        with pytest.raises(ValueError, match="multiples of 8"):
            pkg.LowRankAdapters(_prepared(), 2, rank)
    for slots in (0, 2049):
        with pytest.raises(ValueError, match="slots"):
            pkg.LowRankAdapters(_prepared(), slots, 8)
    for widths in ([64, 32], [120, 8], [8] * 16):
        with pytest.raises(ValueError, match="merged parts"):
            pkg.LowRankAdapters(_prepared(widths=widths), 2, 8)
    ad = pkg.LowRankAdapters(_prepared(widths=[64, 64]), 3, 16)
    assert tuple(ad.lora_a.shape) == (3, 32, 256) and tuple(ad.lora_b.shape) == (3, 128, 16)
    assert not ad.lora_a.requires_grad and set(ad.state_dict()) == {"lora_a", "lora_b", "scaling"}
    a, b = torch.randn(4, 256), torch.randn(64, 4)
    with pytest.raises(ValueError, match="name one"):
        ad.load(0, a, b, 1.0)
    with pytest.raises(ValueError, match="part 2"):
        ad.load(0, a, b, 1.0, part=2)
    with pytest.raises(ValueError, match="slot 3"):
        ad.load(3, a, b, 1.0, part=0)
    with pytest.raises(ValueError, match="no adapter"):
        ad.load(0, torch.randn(17, 256), torch.randn(64, 17), 1.0, part=0)
    with pytest.raises(ValueError, match="no adapter"):
        ad.load(0, a, b[:, :3], 1.0, part=0)
    with pytest.raises(ValueError, match="slot -1"):
        ad.clear(-1)
    ad.load(2, a, b, 0.5, part=1)
    assert torch.equal(ad.lora_a[2, 16:20], a.bfloat16()) and torch.equal(ad.lora_b[2, 64:, :4], b.bfloat16())
    assert float(ad.scaling[2]) == 0.5 and not bool(ad.lora_a[2, :16].any())
    ad.clear(2)
    assert not bool(ad.lora_a.any()) and not bool(ad.lora_b.any()) and not bool(ad.scaling.any())


def test_operators_need_the_gpu(pkg):
    with pytest.raises(ValueError, match="HIP device"):
        pkg.AdapterBatch(torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="HIP device"):
        pkg.ops.input_grad(torch.zeros(1, 128).bfloat16(), torch.zeros(1), torch.zeros(1), 128, 128, 0)
    with pytest.raises(ValueError, match="HIP device"):
        pkg.ops.gated_linear(torch.zeros(1, 128).bfloat16(), torch.zeros(1), torch.zeros(1), 64, 0)


def test_gated_refusals(pkg):
    x = torch.zeros(2, 256).bfloat16()
    with pytest.raises(ValueError, match="unknown activation"):
        pkg.gated_linear(x, _prepared(), "relu")
    with pytest.raises(ValueError, match="MX kernel"):
        pkg.gated_linear(x, torch.nn.Module())
    with pytest.raises(ValueError, match="multiple of 16"):
        pkg.gated_linear(x, _prepared(n=120))
    with pytest.raises(ValueError, match="multiple of 16"):
        pkg.gated_linear(x, _prepared(widths=[96, 32]))
    with pytest.raises(ValueError, match="matching K"):
        pkg.gated_linear(x[:, :128], _prepared())
    with pytest.raises(ValueError, match="BF16"):
        pkg.gated_linear(x.float(), _prepared())


def _cols(*c):
    return (ctypes.c_int64 * len(c))(*c)


def test_entry_points_refuse(pkg):
    """Bad arguments return before any launch, with a message (the pointers are never read)."""
    from vllm_mach_amd import _lib
    err, call = _lib.MxlError, _lib.call
    with pytest.raises(err, match="unknown format"):
        call("mxl_input_grad", 16, 4, 128, 128, 16, 16, 128, 1, 0, 16, 128, None, 0, None)
    with pytest.raises(err, match="E4M3"):
        call("mxl_input_grad", 16, 4, 128, 128, 16, 16, 128, 4, 1, 16, 128, None, 0, None)
    for n, k in ((0, 128), (12, 128), (128, 64), (128, 0), (1 << 23, 128)):
        with pytest.raises(err, match="N % 8"):
            call("mxl_input_grad", 16, 4, n, n, 16, 16, k, 0, 0, 16, k, None, 0, None)
    with pytest.raises(err, match="lddy"):
        call("mxl_input_grad", 16, 4, 128, 120, 16, 16, 128, 0, 0, 16, 128, None, 0, None)
    with pytest.raises(err, match="misaligned"):
        call("mxl_input_grad", 24, 4, 128, 128, 16, 16, 128, 0, 0, 16, 128, None, 0, None)
    gated = [16, 4, 128, 128, 0, 16, 16, 64, 0, 0, 16, 64, 256, 1 << 30, None]
    for at, bad, match in ((8, 1, "unknown format"), (9, 2, "unknown activation"), (7, 24, "I % 16"), (2, 64, "K % 128"),
                           (3, 100, "row stride"), (11, 32, "row stride"), (0, 8, "misaligned"), (13, 100, "workspace"),
                           (12, 128, "workspace")):
        args = list(gated)
        args[at] = bad
        with pytest.raises(err, match=match):
            call("mxl_gated_linear", *args)
    with pytest.raises(err, match="needs dh"):
        call("mxl_gated_grad", 16, 4, 128, 128, 0, 16, 16, 64, 0, 0, None, 64, 16, 128, 256, 1 << 30, None)
    tiles = _lib.query("mxl_adapter_tile_count", 4, 2)
    v = _lib.query("mxl_adapter_v_elems", 4, 1, 8)
    assert v == 4 * 2 * 16
    apply = [16, 4, 128, 128, 16, 16, 16, 2, 1, _cols(0, 128), 8, 16, 16, 16, tiles, 16, v, 16, 128, 16, 1 << 20, None]
    for at, bad, match in ((7, 0, "slots"), (14, tiles + 1, "tiles"), (8, 9, "parts"), (10, 12, "rank"), (10, 264, "rank"),
                           (2, 100, "K % 8"), (9, _cols(0, 0), "no columns"), (9, _cols(16, 128), "start at column 0"),
                           (3, 64, "ldx"), (18, 64, "ldy"), (0, 8, "aligned"), (16, v - 1, "values"), (11, None, "order")):
        args = list(apply)
        args[at] = bad
        with pytest.raises(err, match=match):
            call("mxl_adapter_apply", *args)
    with pytest.raises(err, match="multiple of 16"):
        call("mxl_adapter_apply", 16, 4, 128, 128, 16, 16, 16, 2, 2, _cols(0, 24, 128), 8, 16, 16, 16, tiles, 16, 1 << 20, 16,
             128, 16, 1 << 20, None)
    grad = [16, 4, 128, 128, 16, 128, 16, 16, 0, 0, 16, 16, 16, 2, 1, _cols(0, 128), 8, 16, 16, 16, 16, tiles, 16, v, 16, 128,
            16, 16, 256, 1 << 30, None]
    for at, bad, match in ((15, _cols(0, 100), "N % 8"), (29, 100, "workspace"), (28, 128, "workspace"), (4, 8, "aligned"),
                           (5, 64, "lddy"), (17, None, "ids"), (23, 0, "values"), (21, 0, "tiles")):
        args = list(grad)
        args[at] = bad
        with pytest.raises(err, match=match):
            call("mxl_adapter_grad", *args)
    many = _lib.query("mxl_adapter_tile_count", 64, 2)
    layer = [16, 64, 128, 128, 0, 16, 16, 0, 0, None, 16, 16, 16, 2, 1, _cols(0, 128), 8, 16, 16, 16, 16, many, 16, 1 << 20, 16,
             128, 256, 1 << 30, None]
    for at, bad, match in ((7, 1, "unknown format"), (3, 100, "ldx"), (25, 64, "ldy"), (17, None, "ids"), (23, 0, "values"),
                           (27, 64, "workspace"), (5, 8, "aligned"), (8, 1, None)):
        args = list(layer)
        args[at] = bad
        if at == 8:  # block-FP8 rows are contiguous
            args[3], match = 256, "contiguous"
        with pytest.raises(err, match=match):
            call("mxl_adapter_linear", *args)
    ok = lambda m, slots: _lib.query("mxl_adapter_linear_supported", m, 128, 128, 0, 0, slots, 1, 8)  # noqa: E731
    assert ok(64, 2) and not ok(16, 1) and not ok(64, 3) and not ok(0, 1)
    assert ok(512, 16) and not ok(1 << 20, 17)  # (a tile walks its rows' adapters in turn)
    few = _lib.query("mxl_adapter_tile_count", 16, 1)
    with pytest.raises(err, match="one product"):
        call("mxl_adapter_linear", 16, 16, 128, 128, 0, 16, 16, 0, 0, None, 16, 16, 16, 1, 1, _cols(0, 128), 8, 16, 16, 16, 16,
             few, 16, 1 << 20, 16, 128, 256, 1 << 30, None)


def test_no_rows_is_no_launch(pkg):
    from vllm_mach_amd import _lib
    _lib.call("mxl_input_grad", 16, 0, 128, 128, 16, 16, 128, 0, 0, 16, 128, None, 0, None)
    _lib.call("mxl_gated_linear", 16, 0, 128, 128, 0, 16, 16, 64, 0, 0, 16, 64, None, 0, None)
    _lib.call("mxl_gated_grad", 16, 0, 128, 128, 0, 16, 16, 64, 0, 0, None, 64, 16, 128, None, 0, None)
    _lib.call("mxl_adapter_apply", 16, 0, 128, 128, 16, 16, 16, 2, 1, _cols(0, 128), 8, None, None, None, 0, 16, 0, 16, 128,
              None, 0, None)


def test_fakes(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(5, 256, dtype=torch.bfloat16), torch.empty(1, dtype=torch.uint8)
        ns = torch.ops.mach_amd
        assert ns.gated_linear(x, w, w, 64, 0, 0, 0).shape == (5, 64)
        assert ns.gated_grad(x, x, w, w, 64, 0, 0, 0).shape == (5, 128)
        assert ns.input_grad(x, w, w, 256, 384, 0, False).shape == (5, 384)
        a, b = torch.empty(3, 48, 256, dtype=torch.bfloat16), torch.empty(3, 96, 24, dtype=torch.bfloat16)
        y, v = ns.adapter_linear(x, w, w, 0, False, 0, None, a, b, w, w, w, w, w, [0, 32, 96])
        assert y.shape == (5, 96) and v.shape == (5, 128)
        assert ns.adapter_apply(y, x, a, b, w, w, w, w, w, [0, 32, 96]).shape == (5, 128)
        dx, da, db = ns.adapter_grad(y, x, w, w, 0, False, a, b, w, v, w, w, w, w, [0, 32, 96], True, False, True)
        assert dx.shape == (5, 256) and da.shape == (0,) and db.shape == b.shape


@pytest.mark.parametrize("fmt", ref.FORMATS)
def test_reference_values(pkg, oracle_mod, fmt):
    """The reference's quantized values are the oracle's codes; its weights decode as the formats' tables say."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(7, 256, generator=g) * torch.exp2(torch.randint(-9, 9, (7, 256), generator=g).float())).bfloat16()
    x[2] = 0
    if fmt == "block":
        codes, s = oracle_mod.quant_block_fp8(x)
        v = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().double().view(7, 2, 128)
        want = (v * torch.from_numpy(s).double().reshape(7, 2, 1)).view(7, 256)
    elif fmt != "mxfp4":
        codes, s = oracle_mod.quant_mxfp8(x, 0)
        v = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().double().view(7, 8, 32)
        want = (v * torch.exp2(torch.from_numpy(s).double() - 127)[..., None]).view(7, 256)
    else:
        import mxfp4_reference
        want = torch.as_tensor(mxfp4_reference.dequantize(*mxfp4_reference.quantize(x))).double()
    assert torch.equal(ref.quantized(fmt, x), want)


def test_activation_slopes():
    g = torch.linspace(-12, 12, 2001, dtype=torch.float64)
    for name in ("silu", "gelu_tanh"):
        d = (ref.act(name, g + 1e-5)[0] - ref.act(name, g - 1e-5)[0]) / 2e-5
        assert float((d - ref.act(name, g)[1]).abs().max()) < 1e-9
        assert float(ref.act(name, g)[1].abs().max()) < 1.13


def test_gradients_against_differences():
    """The formulas of the adapters' gradients, from 64-bit differences of the definition."""
    g = torch.Generator().manual_seed(1)
    x, a, b = torch.randn(5, 16, generator=g), torch.randn(2, 16, 16, generator=g), torch.randn(2, 48, 8, generator=g)
    scaling, ids, dy = torch.rand(2, generator=g) + 0.5, torch.tensor([0, 1, -1, 1, 0]), torch.randn(5, 48, generator=g).double()
    x, a, b = x.double(), a.double(), b.double()
    f = lambda *t: float((ref.adapters(*t, scaling, ids, [16, 32], 8)[0] * dy).sum())  # noqa: E731
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for s in range(2):
        t, lo = (ids == s).nonzero().squeeze(-1), 0
        for p, w in enumerate([16, 32]):
            ap, bp, gt = a[s, p * 8:p * 8 + 8], b[s, lo:lo + w], dy[t, lo:lo + w]
            dv = float(scaling[s]) * gt @ bp
            dx[t] += dv @ ap
            da[s, p * 8:p * 8 + 8] = dv.t() @ x[t]
            db[s, lo:lo + w] = gt.t() @ (float(scaling[s]) * x[t] @ ap.t())
            lo += w
    for i, (t, grad) in enumerate(((x, dx), (a, da), (b, db))):
        for at in torch.randint(0, t.numel(), (12,), generator=g).tolist():
            e = torch.zeros(t.numel(), dtype=torch.float64)
            e[at] = 1e-4
            up = f(*[u + e.view(u.shape) if j == i else u for j, u in enumerate((x, a, b))])
            down = f(*[u - e.view(u.shape) if j == i else u for j, u in enumerate((x, a, b))])
            assert abs((up - down) / 2e-4 - float(grad.flatten()[at])) < 1e-6 * (1 + abs(float(grad.flatten()[at])))
