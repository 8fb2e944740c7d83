"""Gate and up projections with activation and product (gated_linear), forward and backward.

Reference: the formulas in 64 bits. A projection's fp32 sum of k products is at most k / 16 + 8
additions deep, each off by at most 2^-24 of the sum of |products|: bar d = (k / 16 + 8) 2^-24
|x| |W|^T. Through the product act(g) u that is |u act'| d_g + |act| d_u (both slopes are below
1.2, and so is act'' in between), and the result's rounding adds eps / 2 of its value (and half of
float16's smallest subnormal). dg and du are rounded once before their products: eps / 2 of each
enters through |W|, |x|.
"""

from __future__ import annotations

import math

import pytest
import torch

import cuda_force_b200 as cf

pytestmark = pytest.mark.gpu


def activation64(g, name):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g**3))
    return g * (1 + th) / 2, (1 + th) / 2 + g * (1 - th**2) * c * (1 + 3 * 0.044715 * g**2) / 2


def depth(count):
    return (count / 16 + 8) * 2.0**-24


def reference(x, wg, wu, dy, name):
    """name -> (value, bar before the result's rounding), in 64 bits; x and dy are 2-D."""
    half = torch.finfo(x.dtype).eps / 2
    tiny = 2.0**-25 if x.dtype == torch.float16 else 0.0
    x, wg, wu, dy = (t.detach().double() for t in (x, wg, wu, dy))
    k, n = x.shape[1], wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    dg_bar, du_bar = (x.abs() @ w.abs().t() * depth(k) for w in (wg, wu))
    act, slope = activation64(g, name)
    fast = 2.0**-19  # the exponential and the quotient of the activation
    out = {"y": (act * u, 1.2 * u.abs() * dg_bar + (act.abs() + dg_bar) * du_bar
                 + fast * (act * u).abs())}
    dg, du = dy * u * slope, dy * act
    off_g = (dy.abs() * (1.2 * u.abs() * dg_bar + 1.2 * du_bar + fast * u.abs() * 1.2)
             + half * dg.abs() + tiny)
    off_u = dy.abs() * (1.2 * dg_bar + fast * act.abs()) + half * du.abs() + tiny
    mag_x = dg.abs() @ wg.abs() + du.abs() @ wu.abs()
    out["x"] = (dg @ wg + du @ wu,
                off_g @ wg.abs() + off_u @ wu.abs() + depth(2 * n) * mag_x)
    m = x.shape[0]
    for key, d, off in (("w_gate", dg, off_g), ("w_up", du, off_u)):
        out[key] = (d.t() @ x, off.t() @ x.abs() + depth(m) * (d.abs().t() @ x.abs()))
    return out


def check(name, got, ref):
    value, bar = ref
    assert got.shape == value.shape, name
    tol = torch.finfo(got.dtype).eps / 2 * value.abs() * (1 + 2.0**-7) + bar
    if got.dtype == torch.float16:
        tol = tol + 2.0**-25
    worst = ((got.double() - value).abs() - tol).max().item()
    assert worst <= 0, f"{name}: {worst:.3g} over the bar"


def make(m, k, n, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    return (r(m, k).to(dtype), (r(n, k) * k**-0.5).to(dtype), (r(n, k) * k**-0.5).to(dtype),
            r(m, n).to(dtype))


SHAPES = [
    # (m, k, n): one token, streamed and tiled token counts, ends inside tiles and 64-blocks
    (1, 8, 8), (1, 256, 136), (3, 1000, 520), (8, 4096, 2048), (9, 200, 4000), (16, 72, 24),
    (17, 512, 264), (100, 1024, 1000), (128, 64, 128), (129, 320, 384), (300, 1032, 776),
    (1000, 504, 2056), (2500, 1024, 2048),
    # few tiles of dx: clusters of 2, 4 and 8 CTAs share its contraction
    (5, 264, 4104), (130, 1000, 2600), (200, 2048, 1200), (700, 520, 5000),
    # streamed: tiles of two sizes, several to a CTA
    (4, 256, 304), (2, 1000, 9608), (8, 576, 11008),
]


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, dtype, activation, cuda_device):
    x, wg, wu, dy = make(*shape, dtype, cuda_device)
    ref = reference(x, wg, wu, dy, activation)
    y = cf.gated_linear(x, wg, wu, activation)
    assert y.dtype == dtype
    check("y", y, ref["y"])
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    y2 = cf.gated_linear(x, wg, wu, activation)
    check("y", y2, ref["y"])
    grads = torch.autograd.grad(y2, leaves, dy, retain_graph=True)
    for name, grad in zip(("x", "w_gate", "w_up"), grads):
        assert grad.dtype == dtype
        check(name, grad, ref[name])
    again = torch.autograd.grad(y2, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    assert torch.equal(cf.gated_linear(x.detach(), wg.detach(), wu.detach(), activation), y)


@pytest.mark.parametrize("wanted", ["x", "w_gate", "w_up", "x w_up"])
def test_only_the_wanted_gradients(wanted, cuda_device):
    x, wg, wu, dy = make(70, 256, 192, torch.bfloat16, cuda_device)
    ref = reference(x, wg, wu, dy, "silu")
    named = {"x": x, "w_gate": wg, "w_up": wu}
    leaves = {k: named[k].requires_grad_() for k in wanted.split()}
    grads = torch.autograd.grad(cf.gated_linear(x, wg, wu), list(leaves.values()), dy)
    for name, grad in zip(leaves, grads):
        check(name, grad, ref[name])


@pytest.mark.parametrize("shape", [(5, 7, 9), (40, 100, 33), (200, 65, 130)], ids=str)
def test_odd_feature_counts_are_padded(shape, cuda_device):
    x, wg, wu, dy = make(*shape, torch.bfloat16, cuda_device)
    ref = reference(x, wg, wu, dy, "gelu")
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    y = cf.gated_linear(x, wg, wu, "gelu")
    check("y", y.detach(), ref["y"])
    for name, grad in zip(("x", "w_gate", "w_up"), torch.autograd.grad(y, leaves, dy)):
        check(name, grad, ref[name])


def test_gradient_agrees_with_differences(cuda_device):
    # Central differences of a fixed functional of the kernel's float16 output along one direction
    # of each input: with a step h of 2^-3 the quotient is off by the roundings of 2 * 512 outputs
    # (random signs, each 2^-11 of values of order 1, over 2 h: about 0.06) and of the stepped
    # inputs, and by h^2 of a third derivative below 1: 0.1 of a slope of order 10.
    x, wg, wu, dy = make(16, 64, 32, torch.float16, cuda_device, seed=5)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    grads = torch.autograd.grad(cf.gated_linear(x, wg, wu), leaves, dy)
    g = torch.Generator(device=cuda_device).manual_seed(11)
    with torch.no_grad():
        for i, grad in enumerate(grads):
            way = grad.double() + 0.3 * grad.double().norm() / math.sqrt(grad.numel()) * torch.randn(
                grad.shape, generator=g, device=cuda_device, dtype=torch.float64)
            way /= way.norm()
            h = 2.0**-3
            value, at = [], []
            for sign in (1, -1):
                moved = [t.detach() for t in leaves]
                moved[i] = (moved[i].double() + sign * h * way).half()
                at.append(moved[i].double())
                value.append((cf.gated_linear(*moved).double() * dy).sum())
            slope = (value[0] - value[1]).item()
            predicted = (grad.double() * (at[0] - at[1])).sum().item()
            assert abs(slope - predicted) <= 0.1 * abs(predicted) + 0.02


def test_extreme_gates(cuda_device):
    # Saturated gates: act is 0 or the gate itself, its slope 0 or 1, nothing turns into NaN.
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.zeros(4, 64, device=cuda_device, dtype=dtype)
        x[:, 0] = torch.tensor([200.0, -200.0, 3.0e4, -3.0e4])
        x[:, 1] = 1
        w = torch.zeros(64, 64, device=cuda_device, dtype=dtype)
        w[:, 0] = 1
        up = torch.zeros_like(w)
        up[:, 1] = 0.5
        for name in ("silu", "gelu"):
            xs = x.clone().requires_grad_()
            y = cf.gated_linear(xs, w, up, name)
            want = torch.tensor([100.0, 0.0, 1.5e4, 0.0], device=cuda_device)[:, None]
            assert torch.allclose(y.float(), want.expand(4, 64), rtol=2.0**-8, atol=1e-30)
            (dx,) = torch.autograd.grad(y, xs, torch.ones_like(y))
            assert torch.allclose(dx[:, 0].float(), torch.tensor([32.0, 0.0, 32.0, 0.0],
                                                                 device=cuda_device))
            # d x[2, 1] is the sum of 64 products 3e4 * 0.5 = 9.6e5, beyond float16's 65504:
            # infinite there, finite everywhere else.
            bad = ~dx.isfinite()
            assert bad.sum() == (1 if dtype == torch.float16 else 0)
            assert not dx.isnan().any() and (dtype != torch.float16 or bad[2, 1])


@pytest.mark.parametrize("m", [4, 40, 300])
def test_special_values_stay_in_their_row(m, cuda_device):
    x, wg, wu, _ = make(m, 128, 256, torch.bfloat16, cuda_device)
    clean = cf.gated_linear(x, wg, wu)
    x[1, 5] = float("nan")
    x[3] = 0
    y = cf.gated_linear(x, wg, wu)
    assert y[1].isnan().all() and torch.count_nonzero(y[3]) == 0
    keep = [i for i in range(m) if i not in (1, 3)]
    assert torch.equal(y[keep], clean[keep])


def test_layouts_and_empties(cuda_device):
    x, wg, wu, dy = make(24, 256, 96, torch.bfloat16, cuda_device)
    y = cf.gated_linear(x, wg, wu)
    assert torch.equal(cf.gated_linear(x.view(2, 3, 4, 256), wg, wu).view(24, 96), y)
    # transposed storage, a slice off the 16-byte boundary, a strided view
    assert torch.equal(cf.gated_linear(x, wg.t().contiguous().t(), wu), y)
    buf = torch.empty(24 * 256 + 1, device=cuda_device, dtype=torch.bfloat16)
    odd = buf[1:].view(24, 256)
    odd.copy_(x)
    assert torch.equal(cf.gated_linear(odd, wg, wu), y)
    wide = torch.empty(24, 300, device=cuda_device, dtype=torch.bfloat16)
    wide[:, :256] = x
    assert torch.equal(cf.gated_linear(wide[:, :256], wg, wu), y)
    none = x[:0].requires_grad_()
    w = wg.clone().requires_grad_()
    empty = cf.gated_linear(none, w, wu)
    assert empty.shape == (0, 96)
    dx, dw = torch.autograd.grad(empty.sum(), (none, w))
    assert dx.shape == (0, 256) and torch.count_nonzero(dw) == 0 and dw.shape == w.shape
    assert cf.gated_linear(x, wg[:0], wu[:0]).shape == (24, 0)
    flat = cf.gated_linear(x[:, :0], wg[:, :0], wu[:, :0])
    assert flat.shape == (24, 96) and torch.count_nonzero(flat) == 0
    # one weight for both projections, and an expanded incoming gradient
    both = wg.clone().requires_grad_()
    out = cf.gated_linear(x, both, both)
    (d,) = torch.autograd.grad(out, both, torch.ones(1, 1, device=cuda_device,
                                                    dtype=torch.bfloat16).expand(24, 96))
    ref = reference(x, wg, wg, torch.ones(24, 96, device=cuda_device), "silu")
    bar = (ref["w_gate"][1] + ref["w_up"][1]
           + 2.0**-7 * (ref["w_gate"][0].abs() + ref["w_up"][0].abs()))
    # ones in float32 do not carry bfloat16's step: add it for dg, du
    bar = bar + 2.0**-8 * 2 * (x.double().abs().sum(0)[None, :] * 4)
    assert ((d.double() - ref["w_gate"][0] - ref["w_up"][0]).abs() <= bar).all()


def test_a_second_derivative_is_refused(cuda_device):
    x, wg, wu, _ = make(4, 64, 32, torch.bfloat16, cuda_device)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(cf.gated_linear(x, wg, wu).sum(), x, create_graph=True)


def test_rows_behind_the_last_are_left_alone(cuda_device):
    from cuda_force_b200 import _abi
    from tests.helpers import ptr, stream_ptr

    lib = _abi.load()
    for m in (3, 20, 130, 300):
        x, wg, wu, _ = make(m, 64, 136, torch.bfloat16, cuda_device)
        y = torch.full((m + 256, 136), 7.0, device=cuda_device, dtype=torch.bfloat16)
        g = torch.full((m + 256, 136), 7.0, device=cuda_device)
        u = g.clone()
        assert lib.cf_gated_linear(ptr(x), ptr(wg), ptr(wu), ptr(y), ptr(g), ptr(u), m, 64, 136,
                                   _abi.CF_ACT_SILU, _abi.CF_DTYPE_BF16,
                                   stream_ptr()) == _abi.CF_OK
        torch.cuda.synchronize()
        assert (y[m:] == 7).all() and (g[m:] == 7).all() and (u[m:] == 7).all()
        ref = x.double() @ wg.double().t()
        assert torch.allclose(g[:m].double(), ref, rtol=1e-5, atol=1e-5)


def test_side_stream_and_graphs(cuda_device):
    x, wg, wu, dy = make(160, 256, 320, torch.bfloat16, cuda_device)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]

    def step():
        y = cf.gated_linear(x, wg, wu)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    eager = [v.clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, on_side))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    with torch.no_grad():
        x.mul_(0.5)
    changed = step()
    for graph, out in (graphs[1], graphs[0], graphs[1]):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(changed, out))


def test_device_status_is_clean(cuda_device):
    from cuda_force_b200 import _abi

    assert _abi.load().cf_device_status() == _abi.CF_OK
