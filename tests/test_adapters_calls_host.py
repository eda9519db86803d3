"""CPU checks of the adapters', gated blocks' and gradients' entry points: refusals, queries, shapes under tracing."""
import pytest
import torch


def test_bias_grad_refuses(pkg):
    from vllm_mach_amd import _lib
    for args, match in (((2, 4, 0, 8, 2, None), "0 < N"), ((2, -1, 8, 8, 2, None), "M >= 0"), ((2, 4, 8, 7, 2, None), "lddy"),
                        ((3, 4, 8, 8, 2, None), "lddy")):
        with pytest.raises(_lib.MxlError, match=match):
            _lib.call("mxl_bias_grad", *args)
    with pytest.raises(ValueError, match="HIP device"):
        pkg.ops.bias_grad(torch.zeros(2, 8).bfloat16())


def test_bias_grad_shape(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        assert torch.ops.mach_amd.bias_grad(torch.empty(5, 24, dtype=torch.bfloat16)).shape == (24,)


def test_gated_refuses_two_limbs(pkg):
    layer = torch.nn.Module()
    layer.mxl_shape, layer.mxl_format, layer.mxl_kernel = (128, 256), 0, pkg.Mxfp8LinearKernel(dual_m=(2, 32))
    layer.weight = layer.weight_scale = torch.zeros(1)
    for shape in ((2, 256), (4, 8, 256)):
        with pytest.raises(ValueError, match="one limb"):
            pkg.gated_linear(torch.zeros(*shape).bfloat16(), layer)
    with pytest.raises(ValueError, match="HIP device"):
        pkg.gated_linear(torch.zeros(3, 256).bfloat16(), layer)


def test_supported_shapes_agree(pkg):
    """The Python rule is the library's, also next to its borders."""
    from vllm_mach_amd import _lib
    ask = lambda *a: bool(_lib.query("mxl_adapter_linear_supported", *a))  # noqa: E731
    rows = [0, 1, 16, 17, 31, 32, 63, 64, 511, 512, 513, 4096, 1 << 20, (1 << 22) - 1, 1 << 22, 1 << 25]
    for m in rows:
        for n, k in ((128, 128), (17408, 5120), (0, 128), (128, 100), (128, 32768), (128, 32896), (1 << 22, 128), (128, 1 << 12)):
            for fmt, block in ((0, 0), (0, 1), (4, 0), (4, 1), (1, 0), (2, 1), (5, 0)):
                for slots, parts, rank in ((1, 1, 8), (2, 8, 256), (16, 1, 24), (17, 1, 8), (0, 1, 8), (1, 9, 8), (1, 1, 12), (1, 1, 264)):
                    args = (m, n, k, fmt, block, slots, parts, rank)
                    assert pkg.ops.adapter_linear_supported(*args) == ask(*args), args
    assert pkg.ops.adapter_linear_supported(64, 128, 128, 0, False, 2, 1, 8)


@pytest.mark.parametrize("m,slots", [(200, 1), (200, 30), (7, 1), (1, 2)])
@pytest.mark.parametrize("grad", [False, True])
def test_a_layer_with_adapters_traces(pkg, m, slots, grad):
    """One graph, without running it."""
    from vllm_mach_amd import _lib
    n, k = 128, 256
    layer = torch.nn.Module()
    layer.mxl_shape, layer.mxl_format, layer.mxl_kernel = (n, k), 0, pkg.Mxfp8LinearKernel()
    layer.weight = torch.nn.Parameter(torch.zeros(8 * 8192, dtype=torch.uint8), requires_grad=False)
    layer.weight_scale = torch.nn.Parameter(torch.zeros(8 * 256, dtype=torch.uint8), requires_grad=False)
    ad = pkg.LowRankAdapters(layer, slots, 8).requires_grad_(grad)
    batch = object.__new__(pkg.AdapterBatch)
    batch.slots, batch.updates = slots, 0
    tiles = _lib.query("mxl_adapter_tile_count", m, slots)
    batch.tensors = (torch.zeros(m, dtype=torch.int32), torch.zeros(m, dtype=torch.int32),
                     torch.zeros(slots + 1, dtype=torch.int64), torch.zeros(tiles, 4, dtype=torch.int32))
    graphs = []

    def backend(gm, example_inputs):
        graphs.append(gm)
        return lambda *args: (torch.zeros(m, n),)

    torch._dynamo.reset()
    method = pkg.MxLinearMethod()
    call = torch.compile(lambda x: method.apply(layer, x, None, adapters=ad, batch=batch), fullgraph=True, backend=backend)
    assert call(torch.zeros(m, k).bfloat16()).shape == (m, n) and len(graphs) == 1
    text = graphs[0].print_readable(print_output=False)
    assert ("adapter_linear" if m == 200 and slots == 1 else "adapter_apply") in text and ("adapter_grad" in text) == grad


def _adapters(pkg, slots=3, rank=16, widths=None):
    layer = torch.nn.Module()
    layer.mxl_shape, layer.mxl_format = (128, 256), 0
    layer.weight = torch.nn.Parameter(torch.zeros(1), requires_grad=False)
    if widths:
        layer.logical_widths = widths
    return pkg.LowRankAdapters(layer, slots, rank)


def test_load_of_own_values(pkg):
    """A slot's own values, whole or cut to a smaller rank, and another slot's."""
    ad = _adapters(pkg)
    g = torch.Generator().manual_seed(1)
    a, b = torch.randn(16, 256, generator=g).bfloat16(), torch.randn(128, 16, generator=g).bfloat16()
    ad.load(1, a, b, 0.5)
    ad.load(1, ad.lora_a[1], ad.lora_b[1], 2.0)
    assert torch.equal(ad.lora_a[1], a) and torch.equal(ad.lora_b[1], b) and float(ad.scaling[1]) == 2.0
    ad.load(1, ad.lora_a[1, 4:12], ad.lora_b[1, :, 4:12], 2.0)
    assert torch.equal(ad.lora_a[1, :8], a[4:12]) and torch.equal(ad.lora_b[1, :, :8], b[:, 4:12])
    assert not bool(ad.lora_a[1, 8:].any()) and not bool(ad.lora_b[1, :, 8:].any())
    ad.load(0, ad.lora_a[1], ad.lora_b[1], 1.0)
    assert torch.equal(ad.lora_a[0], ad.lora_a[1]) and torch.equal(ad.lora_b[0], ad.lora_b[1])
    with pytest.raises(ValueError, match="no adapter"):
        ad.load(0, torch.tensor(1.0), b, 1.0)


_QUERIES = '''
import sys
sys.path.insert(0, {root!r})
import __graft_entry__
__graft_entry__.load_package()
from vllm_mach_amd import _lib
huge = [0, -1, 3, 2 ** 31, 2 ** 32, 2 ** 36, 2 ** 62, 2 ** 63 - 1]
for name, good in (("mxl_adapter_tile_count", [4, 2]), ("mxl_adapter_v_elems", [4, 1, 8]),
                   ("mxl_adapter_apply_workspace_bytes", [4, 128, 2, 1, 8]),
                   ("mxl_adapter_linear_supported", [64, 128, 128, 0, 0, 1, 1, 8]),
                   ("mxl_adapter_linear_workspace_bytes", [64, 128, 0, 0]),
                   ("mxl_input_grad_workspace_bytes", [64, 120, 128, 0]), ("mxl_gated_workspace_bytes", [64, 128, 0])):
    flags = {{"mxl_adapter_linear_supported": (3, 4), "mxl_adapter_linear_workspace_bytes": (2, 3),
             "mxl_input_grad_workspace_bytes": (3,), "mxl_gated_workspace_bytes": (2,)}}.get(name, ())
    sizes = [i for i in range(len(good)) if i not in flags]
    for i in sizes:
        for j in sizes:
            for x in huge:
                args = list(good)
                args[i] = args[j] = x
                assert _lib.query(name, *args) >= 0, (name, args)
    if name != "mxl_adapter_apply_workspace_bytes":
        assert _lib.query(name, *good) > 0, name
print("answered")
'''


def test_queries_of_any_size_answer():
    """In a process of its own: a query that divides by zero would end this one."""
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parents[1])
    out = subprocess.run([sys.executable, "-c", _QUERIES.format(root=root)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip().endswith("answered"), (out.returncode, out.stderr[-500:])


def test_one_limit_of_slots(pkg):
    """2048, wherever it is asked."""
    from vllm_mach_amd import _lib
    assert _lib.query("mxl_adapter_tile_count", 4, 2048) == 4 and _lib.query("mxl_adapter_tile_count", 4, 2049) == 0
    with pytest.raises(_lib.MxlError, match="slots <= 2048"):
        _lib.call("mxl_adapter_tiles", 16, 4, 2049, 16, 4, None)
    with pytest.raises(ValueError, match="slots"):
        _adapters(pkg, 2049, 8)
    assert _adapters(pkg, 2048, 8).slots == 2048


def test_plan_names(pkg):
    from vllm_mach_amd import _lib
    name = _lib.tile_plan_name
    assert name("mxl_gated_plan_name", 1, 64, 128, 0, 0) == "gated_tile_kernel<0,4,1,2> (depth 4)"
    assert name("mxl_adapter_linear_plan_name", 35, 64, 128, 0, 1) == "adapter_tile_kernel<0,4,1,true> (depth 4)"
    assert name("mxl_input_grad_plan_name", 1, 640, 128, 4, 0) == "input_grad_kernel<4,128,128,false> + input_grad_join_kernel"
    for fn, *args in (("mxl_gated_plan_name", 0, 64, 128, 0, 0), ("mxl_gated_plan_name", 4, 24, 128, 0, 0),
                      ("mxl_adapter_linear_plan_name", 16, 64, 128, 0, 0), ("mxl_input_grad_plan_name", 4, 64, 64, 0, 0)):
        with pytest.raises(_lib.MxlError, match="bad shape"):
            name(fn, *args)


def test_every_compiled_tile_is_reached():
    """What the build compiled of the tiles is what the GPU tests reach by their plans."""
    import json
    import re
    from pathlib import Path
    import test_gpu_tile_plans as plans
    report = Path(__file__).resolve().parents[1] / "vllm-mach_amd" / "_build" / "kernel_resources.json"
    if not report.exists():
        pytest.skip("no build report (run __graft_entry__.build() first)")
    built = {"gated": set(), "adapter": set(), "input_grad": set()}
    for kernel in re.findall(r'"(_ZN3mxl[^"]*)"', report.read_text()):
        m = re.match(r"_ZN3mxl\d+(gated_tile|adapter_tile|input_grad)_kernelI((?:L[ib]\d+E)+)E", kernel)
        if m:
            built[m[1].removesuffix("_tile")].add(tuple(int(v) for v in re.findall(r"L[ib](\d+)E", m[2])))
    code = plans.CODES
    gated = {(code[f], *c[0], epi) for f, cases in (("mxfp8", plans.GATED_8), ("mxfp6", plans.GATED_8),
                                                    ("mxfp6_e3m2", plans.GATED_8), ("mxfp4", plans.GATED_4))
             for c in cases for epi in (2, 3)}
    adapter = {(code[f], *c[0], int(f == "block"))
               for f, cases in (("mxfp8", plans.ADD_8), ("mxfp6", plans.ADD_8), ("mxfp6_e3m2", plans.ADD_8),
                                ("mxfp4", plans.ADD_4), ("block", plans.ADD_BLOCK)) for c in cases}
    grad = {(code[f], *c[0], int(f == "block")) for f in code for c in (plans.GRAD_BLOCK if f == "block" else plans.GRAD)}
    assert built == {"gated": gated, "adapter": adapter, "input_grad": grad}
    assert len(json.loads(report.read_text())) > 0
