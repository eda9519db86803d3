"""Every tile, ring depth and quarter of the gated blocks, of the products with adapters and of the input gradients, in each
format, at shapes that the library says it runs so."""
import pytest
import torch

import adapters_reference as ref
from test_gpu_adapters import _case, _check_gradients, _ids
from test_gpu_gated import _want

pytestmark = pytest.mark.gpu
CODES = {"mxfp8": 0, "mxfp6": 2, "mxfp6_e3m2": 3, "mxfp4": 4, "block": 0}

# tile (MT, NT), ring depth, quarters: m, output columns, k
GATED = [((16, 4), 2, False, 513, 9216, 128), ((16, 4), 2, True, 2100, 4096, 128), ((8, 4), 3, False, 260, 9216, 128),
         ((8, 4), 3, True, 513, 8192, 128), ((4, 1), 2, False, 65, 9216, 128), ((4, 1), 4, False, 1, 64, 128)]
GATED_8 = GATED + [((8, 2), 4, False, 65, 9216, 640), ((8, 2), 2, True, 200, 9216, 1024), ((8, 1), 4, False, 65, 5120, 2048),
                   ((4, 2), 3, False, 130, 9216, 256), ((4, 2), 4, False, 1, 9216, 384)]
GATED_4 = GATED + [((8, 2), 4, False, 65, 9216, 1152), ((8, 2), 2, True, 200, 9216, 2048), ((8, 1), 4, False, 65, 5120, 4096),
                   ((4, 2), 3, False, 400, 9216, 128), ((4, 2), 4, False, 1, 9216, 640)]
ADD = [((16, 4), 2, False, 1100, 9216, 128), ((16, 4), 2, True, 2100, 8192, 128), ((8, 4), 3, False, 513, 9216, 128),
       ((8, 4), 3, True, 2100, 4096, 128), ((4, 1), 2, False, 200, 9216, 128), ((4, 1), 4, False, 35, 128, 128)]
ADD_8 = ADD + [((8, 2), 4, False, 200, 9216, 640), ((8, 2), 2, True, 513, 8192, 1024), ((8, 1), 4, False, 65, 9216, 2048),
               ((4, 2), 3, False, 513, 5504, 256), ((4, 2), 4, False, 65, 9216, 384)]
ADD_4 = ADD + [((8, 2), 4, False, 200, 9216, 1152), ((8, 2), 2, True, 513, 8192, 2048), ((8, 1), 4, False, 65, 9216, 4096),
               ((4, 2), 3, False, 513, 5504, 384), ((4, 2), 4, False, 65, 9216, 640)]
ADD_BLOCK = [((8, 2), 2, False, 700, 9216, 128), ((8, 2), 2, True, 2100, 4096, 128), ((8, 2), 4, False, 200, 9216, 640),
             ((8, 1), 4, False, 65, 9216, 2048), ((4, 2), 3, False, 513, 9216, 128), ((4, 2), 4, False, 65, 9216, 384),
             ((4, 1), 2, False, 200, 9216, 128), ((4, 1), 4, False, 35, 128, 128)]


def _each(lists):
    return [pytest.param(fmt, *case, id=f"{fmt}-{case[0][0]}x{case[0][1]}-{case[1]}{'q' if case[2] else ''}")
            for fmt, cases in lists.items() for case in cases]


def _name(kernel, fmt, tile, last, depth, quarters):
    return f"{kernel}<{CODES[fmt]},{tile[0]},{tile[1]},{last}> (depth {depth}{', quarters' if quarters else ''})"


def _plan(*args):
    from vllm_mach_amd import _lib
    return _lib.tile_plan_name(*args)


@pytest.mark.parametrize("fmt,tile,depth,quarters,m,i,k",
                         _each({"mxfp8": GATED_8, "mxfp6": GATED_8, "mxfp6_e3m2": GATED_8, "mxfp4": GATED_4}))
def test_gated(pkg, dev, fmt, tile, depth, quarters, m, i, k):
    """The output, and both products' gradients (``gated_grad``)."""
    for grad in (0, 1):
        assert _plan("mxl_gated_plan_name", m, i, k, CODES[fmt], grad) == _name("gated_tile_kernel", fmt, tile, 2 + grad, depth,
                                                                               quarters)
    gen = torch.Generator().manual_seed(m + i)
    method, layer, w = ref.make_layer(pkg, fmt, [i, i], k, dev, gen)
    act = ("silu", "gelu_tanh")[(m + tile[1]) % 2]
    x = torch.randn(m, k, generator=gen).bfloat16().to(dev)
    dh = torch.randn(m, i, generator=gen).bfloat16().to(dev)
    h, bound, g, u, go, uo = _want(fmt, act, x, w)
    ref.check(pkg.gated_linear(x, layer, act), h, bound)
    a, slope = ref.act(act, g)
    d = dh.double().abs()
    dg, du = dh.double() * u * slope, dh.double() * a
    # (second derivatives of both activations are below 1.2; the slope's arithmetic is within 2^-15 of 1 + |g|)
    so = 1.2 * go + 2.0 ** -15 * (1 + g.abs())
    dgo = ref.U * dg.abs() + (1 + ref.U) * d * (uo * (slope.abs() + so) + u.abs() * so) + 1e-30
    duo = ref.U * du.abs() + (1 + ref.U) * d * (1.13 * go + 2.0 ** -16 * g.abs()) + 1e-30
    both = pkg.ops.gated_grad(x, dh, layer.weight, layer.weight_scale, i, CODES[fmt], pkg.linear.ACTIVATIONS[act])
    ref.check(both[:, :i], dg, dgo, "gate")
    ref.check(both[:, i:], du, duo, "up")


@pytest.mark.parametrize("fmt,tile,depth,quarters,m,n,k",
                         _each({"mxfp8": ADD_8, "mxfp6": ADD_8, "mxfp6_e3m2": ADD_8, "mxfp4": ADD_4, "block": ADD_BLOCK}))
def test_products_with_adapters(pkg, dev, fmt, tile, depth, quarters, m, n, k):
    """Tokens of several adapters and none in a tile, a part that ends inside one, with a bias and without."""
    assert _plan("mxl_adapter_linear_plan_name", m, n, k, CODES[fmt], int(fmt == "block")) == \
        _name("adapter_tile_kernel", fmt, tile, "true" if fmt == "block" else "false", depth, quarters)
    slots = min(3, m // 32)
    first = n // 256 * 128 if fmt == "block" else n // 3 // 16 * 16 + 16
    widths = [n] if fmt == "block" and n < 256 else [first, n - first]
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, widths, k, slots, 24, _ids(m, slots, m), m)
    batch = pkg.AdapterBatch(ids, slots)
    base, off = ref.product(ref.quantized(fmt, x), w, scaled=True)
    delta, doff, _ = ref.adapters(x, ad.lora_a, ad.lora_b, ad.scaling, ids, widths, 24)
    want, bound = base + delta, off + doff + 1e-30
    y = method.apply(layer, x, None, adapters=ad, batch=batch)
    ref.check(y, want, ref.U * want.abs() + (1 + ref.U) * bound)
    bias = torch.randn(n, generator=g).bfloat16().to(dev)
    z = method.apply(layer, x, bias, adapters=ad, batch=batch)
    if fmt == "mxfp4":  # (joins the sum)
        want = want + bias.double()
        ref.check(z, want, ref.U * want.abs() + (1 + ref.U) * (bound + want.abs() * 2.0 ** -23))
    else:
        assert torch.equal(z, y + bias)


# tile, split: m, n, k
GRAD = [((128, 128), False, 1, 128, 128), ((128, 128), True, 1, 640, 128), ((256, 128), False, 2100, 128, 2048),
        ((256, 128), True, 130, 2560, 6400), ((256, 256), False, 5000, 128, 2560), ((256, 256), True, 900, 5120, 4224)]
GRAD_BLOCK = [((128, 128), False, 1, 128, 128), ((128, 128), True, 1, 640, 128), ((128, 128), False, 2100, 192, 1152),
              ((128, 128), True, 300, 2560, 1152)]


def _grad_cases():
    return [pytest.param(fmt, *case, id=f"{fmt}-{case[0][0]}x{case[0][1]}{'-split' if case[1] else ''}-{case[2]}")
            for fmt in ref.FORMATS for case in (GRAD_BLOCK if fmt == "block" else GRAD)]


def _grad_plan(fmt, m, n, k):
    return _plan("mxl_input_grad_plan_name", m, n, k, CODES[fmt], int(fmt == "block"))


def _grad_name(fmt, tile, split):
    return (f"input_grad_kernel<{CODES[fmt]},{tile[0]},{tile[1]},{'true' if fmt == 'block' else 'false'}>"
            + (" + input_grad_join_kernel" if split else ""))


@pytest.mark.parametrize("fmt,tile,split,m,n,k", _grad_cases())
def test_input_gradients(pkg, dev, fmt, tile, split, m, n, k):
    assert _grad_plan(fmt, m, n, k) == _grad_name(fmt, tile, split)
    g = torch.Generator().manual_seed(m + n)
    method, layer, w = ref.make_layer(pkg, fmt, [n], k, dev, g)
    dy = torch.randn(m, n, generator=g).bfloat16().to(dev)
    want, off = ref.product(dy.double(), w.t().contiguous())
    ref.check(pkg.ops.input_grad(dy, *pkg.adapters.grad_of(layer)), want, off + ref.U * want.abs() + 1e-30)


@pytest.mark.parametrize("fmt,tile,split,m,n,k", _grad_cases())
def test_gradients_of_adapters(pkg, dev, fmt, tile, split, m, n, k):
    """The adapters' part of dx within those tiles (from 32 rows an adapter on) and apart."""
    assert _grad_plan(fmt, m, n, k) == _grad_name(fmt, tile, split)
    slots = max(1, min(3, m // 32))
    first = n // 256 * 128 if fmt == "block" else n // 3 // 16 * 16 + 16
    widths = [n] if n < 256 else [first, n - first]
    case = _case(pkg, dev, fmt, widths, k, slots, 24, _ids(m, slots, m), m, True)
    _check_gradients(pkg, fmt, *case)


@pytest.mark.parametrize("fmt,tile,depth,quarters,m,n,k", _each({"mxfp8": ADD_8, "mxfp4": ADD_4, "block": ADD_BLOCK}))
def test_an_infinity_stays_with_its_adapter(pkg, dev, fmt, tile, depth, quarters, m, n, k):
    """In B and in A, whichever tile adds them: other rows, columns and parts keep their bits."""
    slots, rank = min(3, m // 32), 24
    first = n // 256 * 128 if fmt == "block" else n // 3 // 16 * 16 + 16
    widths = [n] if fmt == "block" and n < 256 else [first, n - first]
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, widths, k, slots, rank, _ids(m, slots, m), m)
    batch = pkg.AdapterBatch(ids, slots)
    call = lambda: method.apply(layer, x, None, adapters=ad, batch=batch)  # noqa: E731
    y, mine = call(), ids == 0
    cols = torch.arange(n, device=dev)
    for col in sorted({0, widths[0] - 1, n - 1}):
        kept = ad.lora_b.data[0, col, 3].clone()
        ad.lora_b.data[0, col, 3] = float("inf")
        z = call()
        ad.lora_b.data[0, col, 3] = kept
        assert torch.equal(z[~mine], y[~mine]) and torch.equal(z[:, cols != col], y[:, cols != col])
        assert not bool(z[mine, col].isfinite().any())
    for part in range(len(widths)):
        kept = ad.lora_a.data[0, part * rank + 9, 5].clone()
        ad.lora_a.data[0, part * rank + 9, 5] = float("nan")
        z = call()
        ad.lora_a.data[0, part * rank + 9, 5] = kept
        of_part = (cols >= ad.cols[part]) & (cols < ad.cols[part + 1])
        assert torch.equal(z[~mine], y[~mine]) and torch.equal(z[:, ~of_part], y[:, ~of_part])
        assert bool(z[mine][:, of_part].isnan().all())


@pytest.mark.parametrize("fmt,tile,split,m,n,k", _grad_cases())
def test_an_infinity_of_a_stays_in_its_rows(pkg, dev, fmt, tile, split, m, n, k):
    slots = max(1, min(3, m // 32))
    g, method, layer, w, ad, x, ids = _case(pkg, dev, fmt, [n], k, slots, 24, _ids(m, slots, m), m, True)
    batch = pkg.AdapterBatch(ids, slots)
    dy = torch.randn(m, n, generator=g).bfloat16().to(dev)
    x.requires_grad_()

    def gradient():
        return torch.autograd.grad(method.apply(layer, x, None, adapters=ad, batch=batch), x, dy)[0]

    dx, mine, cols = gradient(), ids == 0, torch.arange(k, device=dev)
    for col in (0, k - 1):
        kept = ad.lora_a.data[0, 17, col].clone()
        ad.lora_a.data[0, 17, col] = float("-inf")
        bad = gradient()
        ad.lora_a.data[0, 17, col] = kept
        assert torch.equal(bad[~mine], dx[~mine]) and torch.equal(bad[:, cols != col], dx[:, cols != col])
        assert not bool(bad[mine, col].isfinite().any())
