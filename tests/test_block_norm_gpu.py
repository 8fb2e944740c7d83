"""The norms around a block with gate and residual scale (gated_residual_rmsnorm).

Reference: the formulas in 64 bits. A result is rounded once to its type, which is off by at
most half a step (finfo.eps / 2 of the value); the fp32 arithmetic before that is a chain of
fewer than 64 roundings of 2^-24 relative to the largest term that enters the value, so the bar
is eps / 2 * |value| + 2^-18 * (largest sum of |terms| in the tensor), and half of the smallest
subnormal for float16.
"""

from __future__ import annotations

import pytest
import torch

import cuda_force_b200 as cf

pytestmark = pytest.mark.gpu

EPS = 1e-6


def reference(x, residual, weight, post, gate, scale, dn, dh, eps=EPS):
    """name -> (value, largest sum of |terms|), in 64 bits."""
    shape, cols = x.shape, x.shape[-1]
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    x, residual, weight, post, gate, dn, dh = map(d, (x, residual, weight, post, gate, dn, dh))
    g = torch.ones((), dtype=torch.float64, device=x.device) if gate is None else gate
    mean = lambda t: t.sum(-1, keepdim=True) / cols  # noqa: E731
    q = torch.rsqrt(mean(x * x) + eps) if post is not None else torch.ones_like(x[..., :1])
    w_post = post if post is not None else torch.ones_like(weight)
    xh = x * q
    p = xh * w_post
    h = scale * residual + g * p
    t = torch.rsqrt(mean(h * h) + eps)
    hh = h * t
    h_abs = (scale * residual).abs() + (g * p).abs()
    out = {"normalised": (hh * weight, h_abs * t * weight.abs()), "residual_out": (h, h_abs)}
    if dn is None and dh is None:
        return out
    dn = torch.zeros_like(x) if dn is None else dn
    dh = torch.zeros_like(x) if dh is None else dh
    a = dn * weight
    m1 = mean(a * hh)
    m1_abs = mean((a * hh).abs())
    grad = dh + t * (a - hh * m1)
    grad_abs = dh.abs() + t * (a.abs() + h_abs * t * m1_abs)
    out["residual"] = (scale * grad, abs(scale) * grad_abs)
    rows = tuple(range(x.dim() - 1))
    out["weight"] = ((dn * hh).sum(rows), (dn.abs() * h_abs * t).sum(rows))
    if gate is not None:
        def over(v):
            v = v.reshape(shape)
            if gate.dim() == 1:
                return v.sum(rows)
            return v.sum([i for i in rows if gate.shape[i] == 1], True) if any(
                gate.shape[i] == 1 for i in rows) else v
        out["gate"] = (over(grad * p), over(grad_abs * p.abs()))
    c, c_abs = (grad * g).expand(shape), (grad_abs * g.abs()).expand(shape)
    if post is not None:
        out["post_weight"] = ((c * xh).sum(rows), (c_abs * xh.abs()).sum(rows))
        c, c_abs = c * post, c_abs * post.abs()
        m2, m2_abs = mean(c * xh), mean(c_abs * xh.abs())
        c, c_abs = q * (c - xh * m2), q * (c_abs + xh.abs() * m2_abs)
    out["x"] = (c, c_abs)
    return out


def check(name, got, ref):
    value, mag = ref
    assert got.shape == value.shape, name
    tol = torch.finfo(got.dtype).eps / 2 * value.abs() + 2.0**-18 * mag.max()
    if got.dtype == torch.float16:
        tol = tol + 2.0**-25
    worst = ((got.double() - value).abs() - tol).max().item()
    assert worst <= 0, f"{name}: {worst:.3g} over the bar"


def make(shape, dtype, wdtype, post, gate, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    cols = shape[-1]
    t = {"x": (2 * r(*shape)).to(dtype), "residual": (3 * r(*shape)).to(dtype),
         "weight": (1 + 0.1 * r(cols)).to(wdtype),
         "post_weight": (1 + 0.1 * r(cols)).to(wdtype) if post else None,
         "gate": (0.5 + 0.3 * r(*gate)).to(wdtype) if gate else None}
    return t, r(*shape).to(dtype), r(*shape).to(dtype)


CASES = [
    # one row; warp-per-row form with four rows a CTA and a ragged last CTA
    ((1, 64), torch.bfloat16, torch.bfloat16, True, (64,)),
    ((7, 200), torch.float16, torch.float16, True, (200,)),
    # each width of the register form, 16-byte and element-wise
    ((33, 1024), torch.bfloat16, torch.bfloat16, True, None),
    ((33, 1027), torch.bfloat16, torch.float32, False, (1027,)),
    ((65, 2048), torch.float16, torch.float16, True, (65, 2048)),
    ((2500, 4096), torch.bfloat16, torch.bfloat16, True, (4096,)),
    ((19, 8192), torch.float16, torch.float32, False, None),
    ((9, 8192), torch.float32, torch.float32, True, (8192,)),
    ((40, 4095), torch.float32, torch.float32, True, (40, 4095)),
    # long rows: forward in registers and backward looping, then both looping
    ((5, 12000), torch.bfloat16, torch.bfloat16, True, (12000,)),
    ((3, 20001), torch.float32, torch.float32, True, (3, 20001)),
    ((6, 17000), torch.bfloat16, torch.float32, False, (17000,)),
    # a gate for each sample: groups cut into slots, whole groups in a slot, single tokens
    ((3, 500, 256), torch.bfloat16, torch.bfloat16, True, (3, 1, 256)),
    ((3000, 2, 512), torch.float16, torch.float16, True, (3000, 1, 512)),
    ((5, 333, 1111), torch.float32, torch.float32, False, (5, 1, 1111)),
    ((4, 1, 128), torch.bfloat16, torch.bfloat16, True, (4, 1, 128)),
    ((2, 3, 5, 96), torch.bfloat16, torch.float32, True, (2, 3, 1, 96)),
    ((600, 3, 9001), torch.bfloat16, torch.bfloat16, True, (600, 1, 9001)),
    ((2, 7, 9001), torch.float16, torch.float16, True, (2, 1, 9001)),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}")
def test_forward_and_gradients(case, cuda_device):
    shape, dtype, wdtype, post, gate = case
    t, dn, dh = make(shape, dtype, wdtype, post, gate, cuda_device)
    ref = reference(*t.values(), 0.8, dn, dh)
    names = [k for k, v in t.items() if v is not None]
    n, h = cf.gated_residual_rmsnorm(*t.values(), residual_scale=0.8, eps=EPS)
    assert n.dtype == h.dtype == dtype
    check("normalised", n, ref["normalised"])
    check("residual_out", h, ref["residual_out"])
    for k in names:
        t[k].requires_grad_()
    n2, h2 = cf.gated_residual_rmsnorm(*t.values(), residual_scale=0.8, eps=EPS)
    assert torch.equal(n2, n) and torch.equal(h2, h)
    first = torch.autograd.grad((n2, h2), [t[k] for k in names], (dn, dh), retain_graph=True)
    for k, grad in zip(names, first):
        assert grad.dtype == t[k].dtype
        check(k, grad, ref[k])
    # the same call again gives the same bits
    again = torch.autograd.grad((n2, h2), [t[k] for k in names], (dn, dh))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("which", ["normalised", "residual_out"])
@pytest.mark.parametrize("cols", [512, 9000])
def test_one_gradient_missing(which, cols, cuda_device):
    t, dn, dh = make((11, cols), torch.float32, torch.float32, True, (cols,), cuda_device)
    for v in t.values():
        v.requires_grad_()
    n, h = cf.gated_residual_rmsnorm(*t.values())
    dn, dh = (dn, None) if which == "normalised" else (None, dh)
    ref = reference(*t.values(), 1.0, dn, dh)
    grads = torch.autograd.grad(n if dh is None else h, list(t.values()), dn if dh is None else dh,
                                allow_unused=True)
    for k, grad in zip(t, grads):
        check(k, grad, ref[k])


def test_gradient_agrees_with_differences(cuda_device):
    # Central differences of a fixed functional in 64 bits of the kernel's own fp32 outputs. With
    # step s the quotient is off by rounding, about 2^-22 * |sum of |terms|| / s, and by s^2; at
    # s = 2^-6 and sums of about 300 both are below 0.02 of gradients of order 1.
    t, dn, dh = make((2, 160), torch.float32, torch.float32, True, (160,), cuda_device, seed=3)
    for v in t.values():
        v.requires_grad_()
    grads = torch.autograd.grad(cf.gated_residual_rmsnorm(*t.values()), list(t.values()), (dn, dh))
    g = torch.Generator(device=cuda_device).manual_seed(9)
    with torch.no_grad():
        for k, grad in zip(t, grads):
            way = torch.randn(t[k].shape, generator=g, device=cuda_device)
            way /= way.norm()
            value = []
            for sign in (1, -1):
                moved = {**t, k: t[k] + sign * 2.0**-6 * way}
                n, h = cf.gated_residual_rmsnorm(*moved.values())
                value.append((n.double() * dn).sum() + (h.double() * dh).sum())
            slope = ((value[0] - value[1]) * 2.0**5).item()
            assert abs(slope - (grad.double() * way).sum().item()) <= 0.02 * max(
                1.0, grad.norm().item()), k


def test_plain_form_is_the_residual_norm(cuda_device):
    # Without post-norm, gate and scale: fused_residual_rmsnorm, up to its rounding of the sum.
    x = torch.randn(64, 1024, device=cuda_device)
    r = torch.randn_like(x)
    w = torch.rand(1024, device=cuda_device)
    n, h = cf.gated_residual_rmsnorm(x, r, w)
    n0, h0 = cf.fused_residual_rmsnorm(x, r, w)
    assert torch.equal(h, h0)
    assert torch.allclose(n, n0, rtol=1e-6, atol=1e-7)


def test_strides_offsets_and_broadcast_inputs(cuda_device):
    # Transposed and sliced inputs, a pointer off the 16-byte boundary, an expanded gate.
    base = torch.randn(256, 40, device=cuda_device, dtype=torch.bfloat16)
    x = base.t()
    r = torch.randn(40, 300, device=cuda_device, dtype=torch.bfloat16)[:, 3:259]
    w = torch.rand(257, device=cuda_device, dtype=torch.bfloat16)[1:]
    gate = torch.rand(1, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    dn, dh = torch.randn_like(r), torch.randn_like(r)
    n, h = cf.gated_residual_rmsnorm(x, r, w, None, gate.expand(256))
    ref = reference(x, r, w, None, gate.expand(256), 1.0, dn, dh)
    check("normalised", n, ref["normalised"])
    check("residual_out", h, ref["residual_out"])
    (dgate,) = torch.autograd.grad((n, h), gate, (dn, dh))
    value, mag = ref["gate"]
    # 256 gradients, each rounded to bfloat16, then their sum rounded again.
    bar = 2.0**-8 * (value.abs().sum() + value.sum().abs()) + 2.0**-18 * mag.sum()
    assert (dgate.double() - value.sum()).abs().item() <= bar.item()


def test_special_rows(cuda_device):
    # A row of zeros gives zeros; NaN and infinity stay in their own row.
    x = torch.randn(6, 512, device=cuda_device)
    r = torch.randn_like(x)
    w = torch.ones(512, device=cuda_device)
    clean_n, clean_h = cf.gated_residual_rmsnorm(x, r, w, w)
    x2, r2 = x.clone(), r.clone()
    x2[1] = 0
    r2[1] = 0
    x2[3, 7] = float("nan")
    r2[4, 9] = float("inf")
    n, h = cf.gated_residual_rmsnorm(x2, r2, w, w)
    assert torch.count_nonzero(n[1]) == 0 and torch.count_nonzero(h[1]) == 0
    assert n[3].isnan().all() and h[4, 9].isinf() and n[4, 9].isnan()
    for row in (0, 2, 5):
        assert torch.equal(n[row], clean_n[row]) and torch.equal(h[row], clean_h[row])


def test_a_second_derivative_is_refused(cuda_device):
    x = torch.randn(4, 64, device=cuda_device, requires_grad=True)
    n, _ = cf.gated_residual_rmsnorm(x, x.detach(), torch.ones(64, device=cuda_device))
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(n.sum(), x, create_graph=True)


def test_empty_inputs(cuda_device):
    w = torch.ones(64, device=cuda_device, requires_grad=True)
    x = torch.zeros(0, 64, device=cuda_device, requires_grad=True)
    n, h = cf.gated_residual_rmsnorm(x, x, w, w, w)
    assert n.shape == h.shape == (0, 64)
    (dw,) = torch.autograd.grad(n.sum() + h.sum(), w)
    assert torch.count_nonzero(dw) == 0 and dw.shape == (64,)
    gate = torch.zeros(0, 1, 64, device=cuda_device, requires_grad=True)
    x = torch.zeros(0, 7, 64, device=cuda_device)
    n, h = cf.gated_residual_rmsnorm(x, x, w, None, gate)
    (dg,) = torch.autograd.grad(n.sum() + h.sum(), gate)
    assert n.shape == (0, 7, 64) and dg.shape == gate.shape


def test_side_stream_and_graph(cuda_device):
    t, dn, dh = make((96, 640), torch.bfloat16, torch.bfloat16, True, (640,), cuda_device)
    for v in t.values():
        v.requires_grad_()

    def step():
        n, h = cf.gated_residual_rmsnorm(*t.values())
        grads = torch.autograd.grad((n, h), list(t.values()), (dn, dh))
        return (n.detach(), h.detach(), *grads)

    eager = [v.clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, on_side))
    # Two captured graphs, replayed in turn and with changed inputs.
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for graph, out in (graphs[1], graphs[0], graphs[1]):
        for v in out:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, out))
    with torch.no_grad():
        t["x"].mul_(0.5)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    changed = step()
    assert all(torch.equal(a, b) for a, b in zip(changed, graphs[0][1]))


def test_c_entry_checks_the_workspace(cuda_device):
    from cuda_force_b200 import _abi
    from tests.helpers import ptr, stream_ptr

    lib = _abi.load()
    x = torch.randn(8, 128, device=cuda_device)
    w = torch.ones(128, device=cuda_device)
    stats = torch.ones(8, 2, device=cuda_device)
    need = lib.cf_gated_residual_rmsnorm_backward_workspace_bytes(8, 128, 0, 0, _abi.CF_DTYPE_F32)
    assert need >= 128 * 4
    ws = torch.empty(need, dtype=torch.uint8, device=cuda_device)
    out = [torch.empty_like(x), torch.empty_like(x), torch.empty_like(w)]
    call = lambda bytes_: lib.cf_gated_residual_rmsnorm_backward(  # noqa: E731
        ptr(x), None, ptr(x), ptr(x), ptr(w), None, None, 1, _abi.CF_DTYPE_F32, ptr(stats),
        ptr(out[0]), ptr(out[1]), ptr(out[2]), None, None, 8, 128, 1.0, _abi.CF_DTYPE_F32, ptr(ws),
        bytes_, stream_ptr())
    assert call(need - 1) == _abi.CF_ERR_WORKSPACE
    assert call(need) == _abi.CF_OK
    torch.cuda.synchronize()
