"""CPU checks of MXFP4 and the grouped router: refusals of the C ABI and of the operators' arguments, fakes, weight
layout sizes, the layers' admission rules, checkpoint schemes."""
import json
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
LIB = ROOT / "vllm-mach_amd" / "libmxlinear.so"


@pytest.fixture
def c(pkg):
    from vllm_mach_amd import _lib
    if not LIB.exists():
        pytest.skip("libmxlinear.so not built")
    return _lib


def test_tiled_sizes(c):
    assert c.query("mxl_tiled_weight_bytes", 2048, 2048, 4) == 128 * 4 * 4 * 1024
    assert c.query("mxl_tiled_weight_bytes", 17, 640, 4) == 2 * 2 * 4 * 1024
    assert c.query("mxl_mxfp4_gemm_workspace_bytes", 0, 128, 128) == 0
    assert c.query("mxl_mxfp4_gemm_workspace_bytes", 4, 128, 100) == 0


@pytest.mark.parametrize("name,args,match", [
    ("mxl_quantize_mxfp4", (16, 4, 48, 48, 0, 16, 16, None), "K % 32"),
    ("mxl_quantize_mxfp4", (16, 4, 0, 0, 0, 16, 16, None), "K > 0"),
    ("mxl_quantize_mxfp4", (16, -1, 64, 64, 0, 16, 16, None), "M >= 0"),
    ("mxl_quantize_mxfp4", (16, 4, 64, 64, 1, 16, 16, None), "unknown rule"),
    ("mxl_quantize_mxfp4", (16, 4, 64, 60, 0, 16, 16, None), "ldx"),
    ("mxl_quantize_mxfp4", (16, 4, 64, 68, 0, 16, 16, None), "ldx"),
    ("mxl_quantize_mxfp4", (18, 4, 64, 64, 0, 16, 16, None), "aligned"),
    ("mxl_quantize_mxfp4", (16, 1 << 40, 64, 64, 0, 16, 16, None), "too large"),
    ("mxl_swiglu_mxfp4", (16, 4, 40, 0, 16, 16, None), "K % 32"),
    ("mxl_swiglu_mxfp4", (16, 4, 64, 2, 16, 16, None), "unknown rule"),
    ("mxl_swiglu_mxfp4", (24, 4, 64, 0, 16, 16, None), "aligned"),
    ("mxl_mxfp4_gemm", (16, 16, 1, 16, 16, 16, 64, None, 16, 16, None, 0, None), "K % 128"),
    ("mxl_mxfp4_gemm", (16, 16, 1, 16, 16, 0, 128, None, 16, 16, None, 0, None), "N > 0"),
    ("mxl_mxfp4_gemm", (16, 16, 1, 16, 16, 32, 128, None, 16, 16, None, 0, None), "ldc"),
    ("mxl_mxfp4_gemm", (16, 16, -1, 16, 16, 16, 128, None, 16, 16, None, 0, None), "M >= 0"),
    ("mxl_mxfp4_gemm", (8, 16, 1, 16, 16, 16, 128, None, 16, 16, None, 0, None), "aligned"),
    ("mxl_mxfp4_gemm", (16, 18, 1, 16, 16, 16, 128, None, 16, 16, None, 0, None), "aligned"),
    ("mxl_mxfp4_gemm", (16, 16, 1, 16, 16, 16, 128, None, 17, 16, None, 0, None), "misaligned"),
    ("mxl_mxfp4_grouped_gemm", (16, 16, 4, None, 1, 16, 0, 4, 16, 16, 16, 128, 16, None), "experts"),
    ("mxl_mxfp4_grouped_gemm", (16, 16, 4, None, 0, 16, 2, 4, 16, 16, 16, 128, 16, None), "row_div"),
    ("mxl_mxfp4_grouped_gemm", (16, 16, 4, None, 1, 16, 2, -4, 16, 16, 16, 128, 16, None), "row counts"),
    ("mxl_mxfp4_grouped_gemm", (16, 16, 4, None, 1, 16, 2, 4, 16, 16, 16, 96, 16, None), "K % 128"),
    ("mxl_mxfp4_quant_gemm", (16, 4, 256, 256, 1, 16, 16, 16, None, 16, 16, None), "unknown rule"),
    ("mxl_mxfp4_quant_gemm", (16, 4, 256, 248, 0, 16, 16, 16, None, 16, 16, None), "ldx"),
    ("mxl_mxfp4_quant_gemm", (16, 4, 256, 256, 0, 16, 16, 16, None, 16, 8, None), "ldc"),
    ("mxl_mxfp4_quant_gemm", (16, 40, 256, 256, 0, 16, 16, 16, None, 16, 16, None), "one launch"),
    ("mxl_mxfp4_quant_gemm", (8, 4, 256, 256, 0, 16, 16, 16, None, 16, 16, None), "aligned"),
    ("mxl_mxfp4_linear", (16, 40, 256, 256, 0, 0, 16, 16, 16, None, 16, 16, None, 0, None), "workspace"),
    ("mxl_mxfp4_linear", (16, 40, 256, 512, 0, 0, 16, 16, 16, None, 17, 16, 256, 1 << 20, None), "misaligned"),
    ("mxl_mxfp4_linear", (16, 40, 256, 256, 1, 0, 16, 16, 16, None, 16, 16, 256, 1 << 20, None), "2 K"),
    ("mxl_mxfp4_linear", (16, 40, 1 << 23, 1 << 23, 0, 0, 16, 16, 16, None, 16, 16, 256, 1 << 20, None), "0 < K"),
    ("mxl_mxfp4_gemm", (16, 16, 600, 16, 16, 16, 16384, None, 16, 16, None, 0, None), "workspace"),
    ("mxl_mxfp4_experts", (16, 4, 256, None, 16, 2, None, None, None, 4, 256, 128, 16, 16, 16, 16, 0, 1, 16, 256, 1 << 30, None), "ids"),
    ("mxl_mxfp4_experts", (16, 4, 256, 16, 16, 2, None, None, None, 4, 256, 100, 16, 16, 16, 16, 0, 1, 16, 256, 1 << 30, None), "by 128"),
    ("mxl_mxfp4_experts", (16, 4, 256, 16, 16, 2, None, None, None, 4, 256, 128, 16, 16, 16, 16, 0, 1, 16, None, 0, None), "workspace"),
    ("mxl_mxfp4_experts", (16, 4, 256, 16, 16, 0, None, None, None, 4, 256, 128, 16, 16, 16, 16, 0, 1, 16, 256, 1 << 30, None), "topk"),
    ("mxl_mxfp4_grouped_swiglu", (16, 4, 256, None, 1, 16, 2, 4, 16, 16, 48, 256, 0, 16, 16, None), "I % 32"),
    ("mxl_mxfp4_grouped_swiglu", (16, 4, 256, None, 1, 16, 2, 40, 16, 16, 64, 256, 0, 16, 16, None), "one launch"),
    ("mxl_mxfp4_grouped_swiglu", (16, 4, 256, None, 1, 16, 2, 4, 16, 16, 64, 256, 0, 18, 16, None), "aligned"),
    ("mxl_mxfp4_grouped_swiglu", (16, 0, 256, None, 1, 16, 2, 4, 16, 16, 64, 256, 0, 16, 16, None), "no activation"),
    ("mxl_mx_gemm", (16, 16, 1, 16, 16, 16, 128, 4, None, 16, 16, None, 0, None), "unknown weight format"),
    ("mxl_moe_router_grouped", (16, 0, None, 4, 1025, 8, 0, 1, 1, 1, 1.0, 16, 16, 16, 16, 16, 16, 1 << 20, None), "E <="),
    ("mxl_moe_router_grouped", (16, 0, None, 4, 64, 8, 0, 5, 1, 1, 1.0, 16, 16, 16, 16, 16, 16, 1 << 20, None), "groups"),
    ("mxl_moe_router_grouped", (16, 0, None, 4, 64, 8, 0, 8, 9, 1, 1.0, 16, 16, 16, 16, 16, 16, 1 << 20, None), "groups"),
    ("mxl_moe_router_grouped", (16, 0, None, 4, 64, 9, 0, 8, 1, 1, 1.0, 16, 16, 16, 16, 16, 16, 1 << 20, None), "topk"),
    ("mxl_moe_router_grouped", (16, 2, None, 4, 64, 8, 0, 8, 1, 1, 1.0, 16, 16, 16, 16, 16, 16, 1 << 20, None), "logits"),
    ("mxl_moe_router_grouped", (16, 0, None, 4, 64, 8, 2, 8, 1, 1, 1.0, 16, 16, 16, 16, 16, 16, 1 << 20, None), "scoring"),
    ("mxl_moe_router_grouped", (16, 0, None, 4, 64, 8, 0, 8, 1, 1, float("inf"), 16, 16, 16, 16, 16, 16, 1 << 20, None),
     "finite"),
    ("mxl_moe_router_grouped", (16, 0, None, 4, 64, 8, 0, 8, 1, 1, 1.0, 16, 16, 16, 16, 16, None, 0, None), "workspace"),
    ("mxl_moe_router_grouped", (16, 0, None, 1 << 30, 64, 8, 0, 8, 1, 1, 1.0, 16, 16, 16, 16, 16, 16, 1 << 50, None),
     "too many"),
])
def test_c_abi_refuses(c, name, args, match):
    with pytest.raises(c.MxlError, match=match):
        c.call(name, *args)


def test_nothing_to_do_launches_nothing(c):
    c.call("mxl_quantize_mxfp4", 16, 0, 64, 64, 0, 16, 16, None)
    c.call("mxl_swiglu_mxfp4", 16, 0, 64, 0, 16, 16, None)
    c.call("mxl_mxfp4_gemm", 16, 16, 0, 16, 16, 16, 128, None, 16, 16, None, 0, None)
    c.call("mxl_mxfp4_grouped_gemm", 16, 16, 4, None, 1, 16, 2, 0, 16, 16, 16, 128, 16, None)


def test_operators_refuse_host_tensors(pkg):
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    b = torch.zeros(2, 64, dtype=torch.uint8)
    for call in (lambda: pkg.ops.quantize_mxfp4(x), lambda: pkg.ops.swiglu_mxfp4(x),
                 lambda: pkg.ops.mxfp4_gemm(b, b, b, b, 16, 128),
                 lambda: pkg.ops.mxfp4_grouped_gemm(b, b, None, 1, torch.zeros(2, dtype=torch.int64), 2, b, b, 16, 128),
                 lambda: pkg.ops.moe_router_grouped(torch.zeros(2, 8), None, 2)):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_fakes_keep_shapes(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(5, 256, dtype=torch.bfloat16)
        a, sa = torch.ops.mach_amd.quantize_mxfp4(x)
        assert a.shape == (5, 128) and sa.shape == (5, 8) and a.dtype == torch.uint8
        assert [t.shape for t in torch.ops.mach_amd.swiglu_mxfp4(x)] == [(5, 64), (5, 4)]
        w, sw = torch.empty(4096, dtype=torch.uint8), torch.empty(256, dtype=torch.uint8)
        y = torch.ops.mach_amd.mxfp4_gemm(a, sa, w, sw, 24, 256)
        assert y.shape == (5, 24) and y.dtype == torch.bfloat16
        off = torch.empty(3, dtype=torch.int64)
        assert torch.ops.mach_amd.mxfp4_linear(x, w, sw, 24).shape == (5, 24)
        assert pkg.ops.mxfp4_linear(x, w, sw, 24, 0, None, True).shape == (5, 24)
        assert torch.ops.mach_amd.mxfp4_grouped_gemm(a, sa, None, 1, off, 5, w, sw, 24, 256).shape == (5, 24)
        out = torch.ops.mach_amd.moe_router_grouped(torch.empty(5, 16), None, 4)
        assert [tuple(t.shape) for t in out] == [(5, 4), (5, 4), (20,), (17,), (20,)]


def test_kernel_admission(pkg):
    L = pkg.linear
    ok = L.MxLinearLayerConfig(L.MXFP4_STATIC, L.MXFP4_DYNAMIC)
    assert L.Mxfp4LinearKernel.can_implement(ok) == (True, None)
    assert not L.Mxfp4LinearKernel.can_implement(L.MxLinearLayerConfig(L.MXFP4_STATIC, L.MXFP8_DYNAMIC))[0]
    assert not L.Mxfp4LinearKernel.can_implement(L.MxLinearLayerConfig())[0]
    assert not L.Mxfp6LinearKernel.can_implement(ok)[0]
    assert L.register_kernels({})["mxfp4"] == [L.Mxfp4LinearKernel]
    method, layer = L.MxLinearMethod(L.MXFP4_STATIC), torch.nn.Module()
    assert isinstance(method.kernel, L.Mxfp4LinearKernel) and method.config.activation_quant_key == L.MXFP4_DYNAMIC
    method.create_weights(layer, 256, [24, 40], 256, 64, torch.bfloat16)
    assert layer.weight.shape == (64, 128) and layer.weight_scale.shape == (64, 8)
    layer.weight.weight_loader(layer.weight, torch.ones(40, 128, dtype=torch.uint8), 1)
    assert bool((layer.weight[24:] == 1).all())


@pytest.mark.parametrize("n,packed,dtype,scale,match", [
    (20, 64, torch.uint8, (20, 4), "N % 8"), (16, 96, torch.uint8, (16, 6), "K % 128"),
    (16, 64, torch.int8, (16, 4), "packed uint8"), (16, 64, torch.uint8, (16, 2), "scales")])
def test_weight_refusals(pkg, n, packed, dtype, scale, match):
    layer = torch.nn.Module()
    layer.weight = torch.nn.Parameter(torch.zeros(n, packed, dtype=dtype), requires_grad=False)
    layer.weight_scale = torch.nn.Parameter(torch.zeros(scale, dtype=torch.uint8), requires_grad=False)
    with pytest.raises(ValueError, match=match):
        pkg.Mxfp4LinearKernel(pkg.MxLinearLayerConfig(pkg.linear.MXFP4_STATIC)).process_weights_after_loading(layer)


def test_layer_refusals(pkg):
    layer = torch.nn.Module()
    layer.mxl_shape, layer.mxl_format = (16, 128), pkg.ops.E2M1
    kernel = pkg.Mxfp4LinearKernel()
    for x in (torch.zeros(2, 128), torch.zeros(2, 64, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="BF16 activations"):
            kernel.apply_weights(layer, x)
    with pytest.raises(ValueError, match="twice"):
        pkg.swiglu_mxfp4_down(torch.zeros(2, 128, dtype=torch.bfloat16), layer)
    layer.mxl_format = pkg.ops.E4M3
    with pytest.raises(ValueError, match="not an MXFP4 layer"):
        pkg.swiglu_mxfp4_down(torch.zeros(2, 256, dtype=torch.bfloat16), layer)


def test_experts_refusals(pkg):
    with pytest.raises(ValueError, match="rule"):
        pkg.Mxfp4Experts(rule=1)
    experts = pkg.Mxfp4Experts()
    u = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    with pytest.raises(ValueError, match="inconsistent"):
        experts.process_weights_after_loading(u(2, 256, 128), u(2, 256, 8), u(2, 256, 32), u(2, 256, 4))
    with pytest.raises(ValueError, match="divisible by 128"):
        experts.process_weights_after_loading(u(2, 192, 128), u(2, 192, 8), u(2, 256, 48), u(2, 256, 3))
    x = torch.zeros(1, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="process_weights"):
        experts.apply_router(x, x, None, None, torch.zeros(1, 2), 1)
    with pytest.raises(ValueError, match="MXFP4 MoE currently supports only SiLU"):
        experts.apply(x, x, None, None, None, None, "gelu", 2, None, None, None, None, None, None, False)
    with pytest.raises(ValueError, match="unknown scoring"):
        pkg.grouped_topk(torch.zeros(1, 8), 2, scoring_func="tanh")
    method, layer = pkg.Mxfp4MoEMethod(), torch.nn.Module()
    method.create_weights(layer, 3, 256, 128, torch.bfloat16)
    assert layer.w13_weight.shape == (3, 256, 128) and layer.w2_weight.shape == (3, 256, 64)
    assert layer.w13_weight_scale.shape == (3, 256, 8) and layer.w2_weight_scale.shape == (3, 256, 4)
    with pytest.raises(ValueError, match="MXFP4 MoE needs"):
        method.create_weights(torch.nn.Module(), 3, 256, 100, torch.bfloat16)


def _quark(weight="fp4", act="fp4"):
    part = lambda dtype, dynamic: dict(dtype=dtype, group_size=32, qscheme="per_group", scale_format="e8m0",  # noqa: E731
                                       is_dynamic=dynamic, symmetric=True)
    return dict(quant_method="quark", exclude=["lm_head"],
                global_quant_config=dict(weight=part(weight, False), input_tensors=part(act, True)))


def test_checkpoint_scheme(pkg):
    assert pkg.linear_quant_key(_quark(), "model.layers.0.mlp.down_proj") == pkg.linear.MXFP4_STATIC
    assert pkg.moe_quant_key(_quark(), "model.layers.0.mlp") == pkg.linear.MXFP4_STATIC
    assert pkg.linear_quant_key(_quark(), "lm_head") is None
    assert pkg.linear_quant_key(_quark(act="fp8_e4m3"), "x") is None
    assert pkg.linear_quant_key(_quark(weight="fp6_e3m2"), "x") is None
    assert pkg.linear_quant_key(_quark("fp6_e3m2", "fp8_e4m3"), "x") == pkg.linear.MXFP6_E3M2_STATIC


def test_checkpoint_shapes(pkg, tmp_path, monkeypatch):
    """A merged layer and routed experts from safetensors, up to the packing (which needs a GPU)."""
    from safetensors.torch import save_file
    g = torch.Generator().manual_seed(0)
    u = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)  # noqa: E731
    tensors = {}
    for name, rows, cols in (("a.gate_proj", 128, 256), ("a.up_proj", 128, 256), ("a.down_proj", 256, 128)):
        for e in ("", *(f".experts.{i}" for i in range(2))):
            key = name.replace("a", f"m{e}" if e else "a", 1)
            tensors[f"{key}.weight"], tensors[f"{key}.weight_scale"] = u(rows, cols // 2), u(rows, cols // 32)
    save_file(tensors, tmp_path / "model.safetensors")
    (tmp_path / "config.json").write_text(json.dumps({"quantization_config": _quark()}))
    packed = []

    def pack(codes, scales, fmt):
        packed.append((codes.clone(), scales.clone(), fmt))
        return codes, scales

    monkeypatch.setattr(pkg.ops, "pack_weight", pack)
    ckpt = pkg.SafetensorsCheckpoint(tmp_path)
    layer = pkg.load_linear(ckpt, "a.gate_up", pkg.linear.MXFP4_STATIC, shards=["a.gate_proj", "a.up_proj"])
    assert layer.mxl_shape == (256, 256)
    assert torch.equal(packed[0][0], torch.cat([tensors["a.gate_proj.weight"], tensors["a.up_proj.weight"]]))
    experts = pkg.load_moe(ckpt, "m", 2, pkg.linear.MXFP4_STATIC)
    assert experts.mxl_experts.shapes == (2, 256, 128) and [p[2] for p in packed] == [4, 4, 4]
    assert torch.equal(packed[1][0][1, 128:], tensors["m.experts.1.up_proj.weight"])
    assert torch.equal(packed[2][1][0], tensors["m.experts.0.down_proj.weight_scale"])


@pytest.mark.parametrize("n,match", [(32768, "workspace"), (32769, "too large"), (40000, "too large")])
def test_weights_past_the_scale_offsets_are_refused(c, n, match):
    """The tiles index a weight's scales (256 bytes for 16 x 512 of it) in 32 bits: the largest K and the N at which
    they end, admitted as far as the missing workspace, and the next."""
    with pytest.raises(c.MxlError, match=match):
        c.call("mxl_mxfp4_gemm", 16, 16, 128, 16, 16, n, 1 << 22, None, 16, n, None, 0, None)


@pytest.mark.parametrize("name,head,tail", [
    ("mxl_mxfp4_quant_gemm", (16, 16, 2048), (0, 16, 16, 16, None, 16, 16, None)),
    ("mxl_mxfp4_linear", (16, 16, 2048), (0, 0, 16, 16, 16, None, 16, 16, None, 0, None)),
    ("mxl_mxfp4_experts", (16, 16), (16, 16, 2, None, None, None, 8, 2048, 128, 16, 16, 16, 16, 0, 1, 16, 256, 1 << 30, None)),
    ("mxl_mxfp4_grouped_swiglu", (16, 16), (None, 1, 16, 8, 16, 16, 16, 128, 2048, 0, 16, 16, None))])
def test_rows_past_32_bit_offsets_are_refused(c, name, head, tail):
    """16 rows of 2048 whose last ends 2^31 values behind the first's start are the furthest that one launch takes."""
    ld = ((1 << 31) - 2048) // 15
    assert 15 * ld + 2048 == 1 << 31 and ld % 8 == 0
    with pytest.raises(c.MxlError, match="span more than 4 GiB"):
        c.call(name, *head, ld + 8, *tail)


def test_only_rows_with_gaps_are_brought_together(pkg):
    """Contiguous rows are never copied for their size; rows with gaps only for a kernel of 32-bit offsets."""
    big = torch.empty((1 << 20) + 8, 4096, dtype=torch.bfloat16, device="meta")
    assert pkg.ops._rows16(big) is big and pkg.ops._rows16(big, True) is big
    ld = ((1 << 31) - 2048) // 15
    for step, copied in ((0, False), (8, True)):
        x = torch.empty(1 << 32, dtype=torch.bfloat16, device="meta").as_strided((16, 2048), (ld + step, 1))
        assert pkg.ops._rows16(x) is x
        assert (pkg.ops._rows16(x, True) is not x) == copied
