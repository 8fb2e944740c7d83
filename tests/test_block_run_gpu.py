"""The feed-forward block's operators one after another, as a transformer uses them: the norms
around the block, gate and up projections, and the down projection in 16 bits for training or in
8-bit floating point for serving.

Bars. Every tensor handed on is rounded once to bfloat16, off by at most eps / 2 = 2^-8 of each
value; the chains here hand on at most eight tensors forward and eight more backward, and a norm or
a product of independent errors passes a relative error (2-norm over 2-norm) on at most doubled,
so forward 2^-8 * 8 = 2^-5 and gradients 2^-4 bound the relative errors with room for none of them
to cancel. An 8-bit code is off by at most 2^-4 of its value (e4m3), and the down projection's
operands are two of them: 2^-3 on its result, which is half of the residual sum or less.
"""

from __future__ import annotations

import pytest
import torch

import cuda_force_b200 as cf

pytestmark = pytest.mark.gpu

HIDDEN, INNER = 512, 1408


def weights(device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    w = {"gate_proj": r(INNER, HIDDEN) * HIDDEN**-0.5, "up_proj": r(INNER, HIDDEN) * HIDDEN**-0.5,
         "down_proj": r(HIDDEN, INNER) * INNER**-0.5, "pre": 1 + 0.1 * r(HIDDEN),
         "post": 1 + 0.1 * r(HIDDEN), "next": 1 + 0.1 * r(HIDDEN), "layer_gate": 0.5 + 0.1 * r(HIDDEN)}
    return {k: v.bfloat16() for k, v in w.items()}


def norm64(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def block64(attn, stream, w):
    h = stream + attn
    n = norm64(h, w["pre"])
    inner = torch.nn.functional.silu(n @ w["gate_proj"].t()) * (n @ w["up_proj"].t())
    out = inner @ w["down_proj"].t()
    h2 = 0.9 * h + w["layer_gate"] * norm64(out, w["post"])
    return norm64(h2, w["next"]), h2


def block(attn, stream, w, down):
    n, h = cf.gated_residual_rmsnorm(attn, stream, w["pre"])
    inner = cf.gated_linear(n, w["gate_proj"], w["up_proj"])
    return cf.gated_residual_rmsnorm(down(inner), h, w["next"], w["post"], w["layer_gate"],
                                     residual_scale=0.9)


def off(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("shape", [(2, 3), (3, 170)], ids=str)
def test_a_training_step(shape, cuda_device):
    w = weights(cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    attn, stream, dn, dh = (torch.randn(*shape, HIDDEN, generator=g, device=cuda_device).bfloat16()
                            for _ in range(4))
    leaves = {"attn": attn, "stream": stream, **w}
    for t in leaves.values():
        t.requires_grad_()
    n, h = block(attn, stream, w, lambda t: t @ w["down_proj"].t())
    grads = torch.autograd.grad((n, h), list(leaves.values()), (dn, dh))
    exact = {k: t.detach().double().requires_grad_() for k, t in leaves.items()}
    n64, h64 = block64(exact["attn"], exact["stream"], exact)
    assert off(n, n64.detach()) <= 2.0**-5 and off(h, h64.detach()) <= 2.0**-5
    ref = torch.autograd.grad((n64, h64), list(exact.values()), (dn.double(), dh.double()))
    for name, got, want in zip(leaves, grads, ref):
        assert got.shape == want.shape and off(got, want) <= 2.0**-4, name


@pytest.mark.parametrize("tokens", [1, 8, 40, 300])
def test_serving_with_8_bit_down_projection(tokens, cuda_device):
    w = weights(cuda_device)
    codes, scales = cf.quantize_fp8(w["down_proj"], block_rows=cf.FP8_BLOCK_SIZE)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    attn, stream = (torch.randn(tokens, HIDDEN, generator=g, device=cuda_device).bfloat16()
                    for _ in range(2))
    run = lambda: block(attn, stream, w, lambda t: cf.linear_fp8(t, codes, scales))  # noqa: E731
    n, h = run()
    n64, h64 = block64(attn.double(), stream.double(), {k: v.double() for k, v in w.items()})
    assert off(n, n64) <= 2.0**-3 and off(h, h64) <= 2.0**-3
    # captured and replayed with other tokens in place
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    attn.copy_(attn.flip(0) * 0.5)
    stream.copy_(stream.roll(1, 0))
    graph.replay()
    torch.cuda.synchronize()
    again = run()
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


def test_two_streams_at_once(cuda_device):
    # The same block on two streams with inputs of their own: no workspace is shared.
    w = weights(cuda_device)
    codes, scales = cf.quantize_fp8(w["down_proj"], block_rows=cf.FP8_BLOCK_SIZE)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    inputs = [[torch.randn(m, HIDDEN, generator=g, device=cuda_device).bfloat16()
               for _ in range(2)] for m in (64, 500)]
    down = lambda t: cf.linear_fp8(t, codes, scales)  # noqa: E731
    alone = [block(*i, w, down) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    results = [[] for _ in inputs]
    for _ in range(20):
        for i, s, r in zip(inputs, streams, results):
            with torch.cuda.stream(s):
                r.append(block(*i, w, down))
    torch.cuda.synchronize()
    for want, r in zip(alone, results):
        for got in r:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_forward_mode_differentiation_is_refused(cuda_device):
    x = torch.randn(4, 64, device=cuda_device, dtype=torch.bfloat16)
    w = torch.ones(64, device=cuda_device, dtype=torch.bfloat16)
    square = torch.zeros(32, 64, device=cuda_device, dtype=torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        dual_w = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: cf.gated_residual_rmsnorm(x, dual, w),
                     lambda: cf.gated_residual_rmsnorm(x, x, w, None, dual_w),
                     lambda: cf.gated_linear(dual, square, square)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        n, _ = cf.gated_residual_rmsnorm(x, x, w)  # without a tangent nothing changes
    assert torch.equal(n, cf.gated_residual_rmsnorm(x, x, w)[0])
