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
