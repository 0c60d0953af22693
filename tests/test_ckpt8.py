"""8-bit activation checkpoints: codes against the format's definition, activations against 64 bits, the quadratic fit with
its features kept in 8 bits, refusals."""
import math

import pytest
import torch

from customnetworklayers_b200 import _lib, ckpt8
from tests.operators_ref import HALF, TINY, act, act_slope, assert_within, put_away

DT = [torch.float32, torch.float16, torch.bfloat16]


# ---- refusals (no GPU) -------------------------------------------------------------------------------------------
def test_refusals_without_a_gpu():
    x = torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ckpt8.store(x)
    with pytest.raises(RuntimeError, match="int8"):
        ckpt8.activation(x, fmt="int4")
    with pytest.raises(RuntimeError, match="format"):
        ckpt8.activation(x, fmt=None)
    with pytest.raises(RuntimeError, match="gelu"):
        ckpt8.Activation8("relu")
    lib = _lib.load()
    assert lib.cnl_ckpt8_store(1, 1, 1, -1, 0, 1, None) == 2
    assert lib.cnl_ckpt8_store(1, 1, 1, 8, 3, 1, None) == 8
    assert lib.cnl_ckpt8_store(1, 1, 1, 8, 0, 0, None) == 8
    assert lib.cnl_ckpt8_store(None, 1, 1, 8, 0, 1, None) == 7
    assert lib.cnl_ckpt8_restore(1, None, 1, 8, 0, 1, None) == 7
    assert lib.cnl_act8_forward(1, 1, 1, None, 8, 0, 1, 1, None) == 7
    assert lib.cnl_act8_forward(1, 1, 1, 1, 8, 0, 1, 3, None) == 8
    assert lib.cnl_act8_backward(1, 1, None, 1, 8, 0, 1, 1, None) == 7
    assert lib.cnl_ckpt8_store(None, None, None, 0, 0, 1, None) == 0


def test_the_definition_itself():
    x = torch.tensor([127.0, 1.5, 2.5, -0.5] + [0.0] * 28, dtype=torch.float64)
    assert put_away(x, "int8")[:4].tolist() == [127.0, 2.0, 2.0, 0.0]                 # ties to even, unit 1
    x[0] = 127.5
    assert put_away(x, "int8")[:2].tolist() == [128.0, 2.0]                           # would round to 128: unit 2
    assert put_away(torch.tensor([448.0, 17.0, 449.0 * 0], dtype=torch.float64), "e4m3")[:2].tolist() == [448.0, 16.0]
    g = torch.Generator().manual_seed(0)
    y = torch.randn(4096, generator=g, dtype=torch.float64)
    top = y.view(-1, 32).abs().amax(1, keepdim=True).expand(-1, 32).reshape(-1)
    assert ((put_away(y, "int8") - y).abs() <= top / 127).all()                       # half a unit, unit <= top * 2 / 127
    assert ((put_away(y, "e4m3") - y).abs() <= torch.maximum(y.abs() / 16, top * 2.0 ** -17)).all()


# ---- codes -------------------------------------------------------------------------------------------------------
def _values(n, dtype, seed):
    """Ordinary values, ties, values around the borders between two units, and blocks far apart in size."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=g, dtype=torch.float64)
    x *= torch.exp2(torch.randint(-10, 8, (n // 32 + 1,), generator=g).double()).repeat_interleave(32)[:n]
    half = torch.randint(-255, 256, (n,), generator=g).double() / 2                    # n + 1/2: ties of both formats
    pick = torch.rand(n, generator=g)
    x = torch.where(pick < 0.3, half, x)
    x[pick > 0.97] = 0.0
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [1, 3, 31, 32, 33, 255, 1000, 4096, 8192 * 3 + 5])
def test_restored_values_are_the_definitions(n, fmt, dtype):
    x = _values(n, dtype, n)
    stored = ckpt8.store(x.cuda(), fmt)
    assert stored.codes.shape == (n,) and stored.scales.shape == (-(-n // 32),) and stored.nbytes == n + -(-n // 32)
    ref = put_away(x.double(), fmt)
    assert torch.equal(ckpt8.restore(stored, torch.float32).double().cpu(), ref)        # every step is exact
    back = ckpt8.restore(stored)
    assert back.dtype == dtype and torch.equal(back.cpu(), ref.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_a_view_that_starts_at_an_odd_element_gives_the_same_codes(fmt, dtype):
    x = _values(5001, dtype, 3).cuda()
    a, b = ckpt8.store(x[1:], fmt), ckpt8.store(x[1:].clone(), fmt)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    odd = ckpt8.Stored8(torch.empty(5001, dtype=torch.uint8, device="cuda")[1:].copy_(a.codes), a.scales, a.shape, a.dtype, fmt)
    assert torch.equal(ckpt8.restore(odd), ckpt8.restore(a))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_zeros_limits_and_elements_that_are_not_finite(fmt, dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(32 * 7, dtype=dtype)
    x[32] = info.max                                   # saturates: the code next above would be infinite
    x[33] = -info.max
    x[64:67] = torch.tensor([float("inf"), 1.0, 0.25])
    x[96:99] = torch.tensor([float("nan"), -3.0, 2.0])
    x[128:160] = float("-inf")
    x[160:163] = torch.tensor([info.tiny, -info.tiny / 2, info.tiny * 1.5], dtype=torch.float64).to(dtype)
    x[192] = info.smallest_normal * info.eps           # the smallest subnormal
    got = ckpt8.restore(ckpt8.store(x.cuda(), fmt)).cpu()
    ref = put_away(x.double(), fmt).clamp(-info.max, info.max).to(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got[~torch.isnan(ref)], ref[~torch.isnan(ref)])
    assert torch.isnan(got[64]) and got[65] == 1.0 and torch.isnan(got[96]) and got[0] == 0 and torch.isfinite(got[32])


@pytest.mark.gpu
def test_empty_and_large():
    empty = ckpt8.store(torch.empty(0, 5, device="cuda"))
    assert ckpt8.restore(empty).shape == (0, 5)
    n = 2 ** 31 + 39                                    # elements and code bytes past 2^31
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.tensor([3.0, -127.0, 0.5])
    x[2 ** 30] = 5.0
    back = ckpt8.restore(ckpt8.store(x))
    assert back[-3:].tolist() == [3.0, -127.0, 0.0] and back[2 ** 30] == 5.0 and int(back.count_nonzero()) == 3


# ---- activations -------------------------------------------------------------------------------------------------
def _bound(x, ref, dtype):
    """Rounding to the type, and per 32-bit step 2^-24: about ten products, the exponential's argument x^2/2 rounded once
    (error x^2 2^-25 of the result); the 16-bit types take the shorter polynomial, 8.3e-6 of the tail's value."""
    x = x.double()
    tail = 8.3e-6 if dtype != torch.float32 else 1.7e-7
    fp32 = (16 + x * x) * 2.0 ** -24 + tail
    return HALF[dtype] * ref.abs() + TINY[dtype] + fp32 * ref.abs().maximum(x.abs() * torch.exp(-x * x / 2) + 2.0 ** -100)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kind", ["gelu", "silu"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [1, 33, 4096, 10001])
def test_activation_and_its_gradient(n, fmt, kind, dtype):
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(n, generator=g, dtype=torch.float64) * 3).to(dtype)
    dy = torch.randn(n, generator=g, dtype=torch.float64).to(dtype)
    leaf = x.cuda().requires_grad_(True)
    y = ckpt8.activation(leaf, kind, fmt)
    (dx,) = torch.autograd.grad(y, leaf, dy.cuda())
    ref = act(x.double(), kind)
    assert_within(y, ref, _bound(x, ref, dtype), "y")
    back = put_away(x.double(), fmt)
    slope = act_slope(back, kind)
    # dx is a product with dy; slope's fp32 error is a few 2^-24 of its terms (at most 1 + |x| phi)
    tail = 8.3e-6 if dtype != torch.float32 else 1.7e-7
    bound = HALF[dtype] * (slope * dy.double()).abs() + TINY[dtype] + dy.double().abs() * ((24 + back * back) * 2.0 ** -24 + tail) * 1.2
    assert_within(dx, slope * dy.double(), bound, "dx")
    with torch.no_grad():
        assert torch.equal(ckpt8.activation(leaf, kind, fmt), y)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gelu", "silu"])
def test_activation_slope_against_differences(kind):
    # points that 8 bits hold exactly: whole multiples of 1/16 under 8 in a block whose largest is just under 8
    x = (torch.arange(-100, 101).double() / 16)
    x = torch.nn.functional.pad(x, (0, 224 - 201), value=7.9375)
    x = x.view(7, 32)
    x[:, -1] = 7.9375
    x = x.reshape(-1)
    leaf = x.float().cuda().requires_grad_(True)
    y = ckpt8.activation(leaf, kind, "int8")
    (dx,) = torch.autograd.grad(y.sum(), leaf)
    e = 2.0 ** -6
    with torch.no_grad():
        up, down = (ckpt8.activation((x + s * e).float().cuda(), kind, "int8").double().cpu() for s in (1, -1))
    # central difference: e^2 / 6 times the third derivative (under 2), and two fp32 values' errors over 2 e
    assert_within(dx, (up - down) / (2 * e), e * e / 3 + 2.0 ** -20 * 8 / e)


@pytest.mark.gpu
def test_activation_of_a_transposed_and_of_an_infinite_input():
    x = torch.randn(64, 48, device="cuda").t().requires_grad_(True)
    y = ckpt8.activation(x)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(x))
    z = x.detach().contiguous().requires_grad_(True)
    y2 = ckpt8.activation(z)
    (dz,) = torch.autograd.grad(y2, z, torch.ones(48, 1, device="cuda").expand(48, 64))
    assert torch.equal(y, y2) and torch.equal(dx, dz)
    bad = torch.tensor([float("inf"), 1.0, float("nan")], device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(ckpt8.activation(bad).sum(), bad)
    assert torch.isnan(g[0]) and torch.isfinite(g[1]) and torch.isnan(g[2])


@pytest.mark.gpu
def test_input_is_not_kept_and_second_derivatives_are_refused():
    x = torch.randn(1 << 20, device="cuda", requires_grad=True)
    y = ckpt8.activation(x * 1.0)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() > 0
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
def test_refusals_on_the_device():
    x = torch.randn(64, 32, device="cuda")
    with pytest.raises(RuntimeError, match="contiguous"):
        ckpt8.store(x.t())
    with pytest.raises(RuntimeError, match="float32"):
        ckpt8.store(x.double())
    s = ckpt8.store(x)
    with pytest.raises(RuntimeError, match="shape"):
        ckpt8.restore(ckpt8.Stored8(s.codes[:-1], s.scales, s.shape, s.dtype, s.fmt))
    with pytest.raises(RuntimeError, match="dtype"):
        ckpt8.restore(s, torch.int32)


# ---- the quadratic fit keeps its features in 8 bits --------------------------------------------------------------
@pytest.mark.gpu
def test_quadfit_with_features_in_8_bits():
    from customnetworklayers_b200 import QuadFit_cuda_ext
    from customnetworklayers_b200.QuadFitting import QuadFittingFromFlow
    g = torch.Generator(device="cuda").manual_seed(4)
    n, h, w, c = 2, 24, 40, 8
    f0, f1 = (torch.randn(n, h, w, c, generator=g, device="cuda").requires_grad_(True) for _ in range(2))
    flow = torch.rand(n, h, w, 2, generator=g, device="cuda") * 4 - 2
    up = torch.randn(n, h, w, 3, generator=g, device="cuda")
    plain, packed = QuadFittingFromFlow("cuda"), QuadFittingFromFlow("cuda", checkpoint="int8")
    a, b = plain(f0, f1, flow), packed(f0, f1, flow)
    assert torch.equal(a, b)
    got = torch.autograd.grad(b, (f0, f1), up)
    # the gradient is the layer's own at the restored features
    nchw = lambda t: t.detach().permute(0, 3, 1, 2).contiguous()  # noqa: E731
    back = [ckpt8.restore(ckpt8.store(nchw(t))) for t in (f0, f1)]
    want = QuadFit_cuda_ext.backward(nchw(up), *back, nchw(flow))
    assert torch.equal(nchw(got[0]), want[0])
    # the second map's gradient is a sum by atomics: up to 5 * h * w addends a pixel, order free
    assert_within(nchw(got[1]), want[1], 2.0 ** -24 * 64 * want[1].abs().max().double())
    with pytest.raises(RuntimeError, match="int8"):
        QuadFittingFromFlow("cuda", checkpoint="int5")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kind", ["gelu", "silu"])
@pytest.mark.parametrize("n", [8, 5])
def test_activation_at_the_ends_of_the_line(n, kind, dtype):
    """x Phi(x) and x sigmoid(x) at infinities, NaN and the type's largest values, aligned and not."""
    top = torch.finfo(dtype).max
    x = torch.tensor([float("inf"), float("-inf"), float("nan"), top, -top, 0.0, -0.0, 1.0][:n], dtype=dtype)
    ref = act(x.double(), kind)
    assert ref[0] == float("inf") and ref[3] == top and ref[4] == 0
    for at in (0, 1):
        dev = torch.zeros(n + 1, dtype=dtype, device="cuda")[at:at + n].copy_(x)
        with torch.no_grad():
            y = ckpt8.activation(dev, kind)
        y2 = ckpt8.activation(dev.clone().requires_grad_(True), kind, "e4m3").detach()
        for got in (y, y2):
            assert_within(got, ref, 2.0 ** -18 * torch.ones(n, dtype=torch.float64) + HALF[dtype] * ref.abs().nan_to_num(0, 0, 0), "y")


@pytest.mark.gpu
def test_quadfit_puts_nothing_away_where_no_gradient_is_wanted():
    from customnetworklayers_b200.QuadFitting import QuadFittingFromFlow
    g = torch.Generator(device="cuda").manual_seed(5)
    f0, f1 = (torch.randn(1, 12, 20, 4, generator=g, device="cuda") for _ in range(2))
    flow = torch.rand(1, 12, 20, 2, generator=g, device="cuda")
    fit = QuadFittingFromFlow("cuda", checkpoint="int8")
    lib = _lib.load()

    def launches(*maps):
        before = lib.cnl_launch_count()
        sol = fit(*maps)
        return lib.cnl_launch_count() - before, sol

    plain, want = launches(f0, f1, flow)
    with torch.no_grad():
        n, sol = launches(f0.clone().requires_grad_(True), f1, flow)
    assert n == plain == 1 and torch.equal(sol, want)
    n, sol = launches(f0, f1.clone().requires_grad_(True), flow)
    assert n == plain + 2 and torch.equal(sol, want)               # one map's gradient needs both maps


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_what_an_activation_keeps_for_its_backward_pass(fmt):
    n = 1 << 22
    x = torch.randn(n, device="cuda", requires_grad=True)
    y = ckpt8.activation(x * 1.0, "gelu", fmt)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y.detach_()                                            # lets go of the graph and of what it keeps
    kept = before - torch.cuda.memory_allocated()
    assert n * (1 + 1 / 32) <= kept <= n * (1 + 1 / 32) + 512


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gelu", "silu"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_the_two_passes_without_autograd(fmt, kind):
    g = torch.Generator(device="cuda").manual_seed(9)
    x, dy = (torch.randn(3, 77, 9, generator=g, device="cuda").half() for _ in range(2))
    y, stored = ckpt8.forward(x, kind, fmt)
    dx = ckpt8.backward(stored, dy, kind)
    leaf = x.clone().requires_grad_(True)
    want = ckpt8.activation(leaf, kind, fmt)
    assert torch.equal(y, want) and torch.equal(dx, torch.autograd.grad(want, leaf, dy)[0])
    assert torch.equal(stored.codes, ckpt8.store(x, fmt).codes) and stored.shape == x.shape
    with pytest.raises(RuntimeError, match="shape"):
        ckpt8.backward(stored, dy[:1].clone(), kind)
