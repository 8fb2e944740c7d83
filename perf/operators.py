"""Cases for the operators of a transformer's feed-forward block: the norms around it
(``gated_residual_rmsnorm``), its gate and up projections (``gated_linear``) and the 8-bit
floating-point quantiser and linear (``quantize_fp8``, ``linear_fp8``).

``run`` computes a case in plain torch operations in 32 bits, or, where ``own`` is true, through
``cuda_force_b200``; ``exact`` computes it in 64 bits."""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
BLOCK = 128
E4M3_MAX = 448.0


def listed():
    return [
        # One decoding step of eight sequences: post-norm, scaled residual, next pre-norm. Latency.
        {"name": "norm_decode_8x4096_bf16", "op": "norm", "train": False, "batch": 8, "tokens": 1,
         "cols": 4096, "dtype": "bf16", "post": True, "gate": "none", "scale": 1.0},
        # A long prompt through a Llama-7B-sized stream with a learned gate for each channel.
        {"name": "norm_prefill_16384x4096_bf16", "op": "norm", "train": False, "batch": 1,
         "tokens": 16384, "cols": 4096, "dtype": "bf16", "post": True, "gate": "channel",
         "scale": 0.8},
        # A training step of the same stream: forward and every gradient.
        {"name": "norm_train_8192x4096_bf16", "op": "norm", "train": True, "batch": 4,
         "tokens": 2048, "cols": 4096, "dtype": "bf16", "post": True, "gate": "channel",
         "scale": 1.0},
        # Conditioned training with a gate for each sample, fp32 and an odd row length.
        {"name": "norm_train_sample_gate_5x333x1111_f32", "op": "norm", "train": True, "batch": 5,
         "tokens": 333, "cols": 1111, "dtype": "f32", "post": False, "gate": "sample",
         "scale": 0.5},
        # Activations of a down projection, quantised row by row.
        {"name": "quant_rows_8192x11008_bf16", "op": "quant", "rows": 8192, "cols": 11008,
         "block_rows": 1, "dtype": "bf16"},
        # One MLP weight of Llama-7B, quantised in square blocks.
        {"name": "quant_blocks_11008x4096_bf16", "op": "quant", "rows": 11008, "cols": 4096,
         "block_rows": 128, "dtype": "bf16"},
        # One decoding step of eight sequences through an up projection: the weight's bytes.
        {"name": "fp8_decode_8x4096x11008_bf16", "op": "fp8", "m": 8, "k": 4096, "n": 11008,
         "dtype": "bf16"},
        # A short prompt: ragged tokens, half a block at the end of k, features that end in a tile.
        {"name": "fp8_ragged_777x4160x1030_f16", "op": "fp8", "m": 777, "k": 4160, "n": 1030,
         "dtype": "f16"},
        # The Llama-70B MLP projection of the column-sharded benchmark, on one GPU.
        {"name": "fp8_prefill_16384x8192x28672_bf16", "op": "fp8", "m": 16384, "k": 8192,
         "n": 28672, "dtype": "bf16"},
        # One decoding step of four sequences through gate and up.
        {"name": "gated_decode_4x4096x11008_bf16", "op": "gated", "train": False, "m": 4,
         "k": 4096, "n": 11008, "dtype": "bf16", "activation": "silu"},
        # A ragged prompt in half precision with the tanh form of GELU.
        {"name": "gated_prefill_1501x4096x11008_f16", "op": "gated", "train": False, "m": 1501,
         "k": 4096, "n": 11008, "dtype": "f16", "activation": "gelu"},
        # A training step of the Llama-7B gate and up projections: output and all gradients.
        {"name": "gated_train_4096x4096x11008_bf16", "op": "gated", "train": True, "m": 4096,
         "k": 4096, "n": 11008, "dtype": "bf16", "activation": "silu"},
    ]


def _spread(rng, low, high, step=1):
    """A whole number of [low, high], spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(step, int(v / step + 0.5) * step)


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "quant", "fp8", "fp8", "gated", "gated_train"])
    half = rng.choice(["bf16", "f16"])
    if kind.startswith("norm"):
        batch = _spread(rng, 1, 16)
        return {"op": "norm", "train": kind == "norm_train", "batch": batch,
                "tokens": _spread(rng, 1, 16384 // batch),
                "cols": _spread(rng, 64, 8192, rng.choice([1, 8, 64])),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "post": rng.random() < 0.6,
                "gate": rng.choice(["none", "channel", "sample", "full"]),
                "scale": rng.choice([1.0, 0.5, 0.8])}
    if kind == "quant":
        return {"op": "quant", "rows": _spread(rng, 1, 16384), "cols": _spread(rng, 128, 16384, 8),
                "block_rows": rng.choice([1, 128]), "dtype": rng.choice(["bf16", "f16", "f32"])}
    if kind == "fp8":
        return {"op": "fp8", "m": _spread(rng, 1, 16384), "k": _spread(rng, 128, 8192, 16),
                "n": _spread(rng, 64, 28672, rng.choice([1, 8, 128])), "dtype": half}
    train = kind == "gated_train"
    return {"op": "gated", "train": train, "m": _spread(rng, 1, 4096 if train else 8192),
            "k": _spread(rng, 128, 4096, 8), "n": _spread(rng, 128, 11008, 8), "dtype": half,
            "activation": rng.choice(["silu", "gelu"])}


def _lead(case):
    return (case["batch"], case["tokens"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda") * std + mean

    if case["op"] == "norm":
        dt, c, lead = DTYPES[case["dtype"]], case["cols"], _lead(case)
        gate_shape = {"none": None, "channel": (c,), "sample": (case["batch"], 1, c),
                      "full": (*lead, c)}[case["gate"]]
        s = {"case": case, "x": normal(*lead, c, std=2.0).to(dt),
             "residual": normal(*lead, c, std=3.0).to(dt),
             "weight": normal(c, std=0.1, mean=1.0).to(dt),
             "post": normal(c, std=0.1, mean=1.0).to(dt) if case["post"] else None,
             "gate": normal(*gate_shape, std=0.3, mean=0.5).to(dt) if gate_shape else None}
        if case["train"]:
            s["dn"] = normal(*lead, c).to(dt)
            s["dh"] = normal(*lead, c).to(dt)
            for name in ("x", "residual", "weight", "post", "gate"):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    dt = DTYPES[case["dtype"]]
    if case["op"] == "quant":
        rows, cols = case["rows"], case["cols"]
        x = normal(rows, cols, std=0.02 if case["block_rows"] > 1 else 1.0)
        # One entry in a thousand is an outlier, as in trained weights and activations.
        x = torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 1e-3, x * 20.0, x)
        return {"case": case, "x": x.to(dt)}
    m, k, n = case["m"], case["k"], case["n"]
    if case["op"] == "fp8":
        codes, scales = _plain_quantize(normal(n, k, std=0.02), 128)
        return {"case": case, "x": normal(m, k).to(dt), "codes": codes, "scales": scales}
    s = {"case": case, "x": normal(m, k).to(dt), "w_gate": normal(n, k, std=k**-0.5).to(dt),
         "w_up": normal(n, k, std=k**-0.5).to(dt)}
    if case["train"]:
        s["dy"] = normal(m, n).to(dt)
        for name in ("x", "w_gate", "w_up"):
            s[name].requires_grad_()
    return s


def _plain_quantize(x, block_rows):
    """Codes and scales of blocks of block_rows x 128: scale = absmax / 448 (1 where that is 0)."""
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    wide = torch.zeros(rb * block_rows, cb * BLOCK, device=x.device)
    wide[:rows, :cols] = x
    blocks = wide.view(rb, block_rows, cb, BLOCK)
    scales = blocks.abs().amax(dim=(1, 3)) / E4M3_MAX
    scales = torch.where(scales > 0, scales, torch.ones_like(scales))
    codes = (blocks / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.view(rb * block_rows, cb * BLOCK)[:rows, :cols].contiguous(), scales


def _plain_spread(scales, block_rows, rows, cols):
    """Each block's scale at every element of the block."""
    s = scales.repeat_interleave(block_rows, 0)[:rows]
    return s.repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_norm(s):
    case, dt = s["case"], s["x"].dtype
    x, r, w = (s[name].detach().float() for name in ("x", "residual", "weight"))
    q = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xh = x * q
    p = xh * s["post"].detach().float() if case["post"] else x
    gate = s["gate"].detach().float() if s["gate"] is not None else None
    h = case["scale"] * r + (p if gate is None else gate * p)
    t = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    hh = h * t
    out = {"normalised": (hh * w).to(dt), "residual_out": h.to(dt)}
    if not case["train"]:
        return out
    dn, dh = s["dn"].float(), s["dh"].float()
    a = dn * w
    d = dh + t * (a - hh * (a * hh).mean(-1, keepdim=True))
    out["d_residual"] = (case["scale"] * d).to(dt)
    out["d_weight"] = (dn * hh).sum((0, 1)).to(dt)
    dp = d
    if gate is not None:
        dgate = d * p
        out["d_gate"] = {"channel": lambda v: v.sum((0, 1)), "sample": lambda v: v.sum(1, True),
                         "full": lambda v: v}[case["gate"]](dgate).to(dt)
        dp = d * gate
    if case["post"]:
        out["d_post"] = (dp * xh).sum((0, 1)).to(dt)
        c = dp * s["post"].detach().float()
        dp = q * (c - xh * (c * xh).mean(-1, keepdim=True))
    out["d_x"] = dp.to(dt)
    return out


def _own_norm(s):
    import cuda_force_b200 as cf

    case = s["case"]
    n, h = cf.gated_residual_rmsnorm(s["x"], s["residual"], s["weight"], s["post"], s["gate"],
                                     residual_scale=case["scale"], eps=EPS)
    out = {"normalised": n.detach(), "residual_out": h.detach()}
    if case["train"]:
        names = [name for name in ("residual", "weight", "gate", "post", "x")
                 if s[name] is not None]
        grads = torch.autograd.grad((n, h), [s[name] for name in names], (s["dn"], s["dh"]))
        out.update({"d_" + name: grad for name, grad in zip(names, grads)})
    return out


def _plain_activation(g, activation):
    """The activation of g and its derivative."""
    if activation == "silu":
        sig = torch.reciprocal(1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    c = math.sqrt(2.0 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g * g * g))
    slope = c * (1.0 + 3 * 0.044715 * g * g)
    return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * slope


def _plain_gated(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu = (s[name].detach().float() for name in ("x", "w_gate", "w_up"))
    g, u = x @ wg.t(), x @ wu.t()
    act, slope = _plain_activation(g, case["activation"])
    out = {"y": (act * u).to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dg, du = dy * u * slope, dy * act
        out["d_x"] = (dg @ wg + du @ wu).to(dt)
        out["d_w_gate"] = (dg.t() @ x).to(dt)
        out["d_w_up"] = (du.t() @ x).to(dt)
    return out


def _own_gated(s):
    import cuda_force_b200 as cf

    y = cf.gated_linear(s["x"], s["w_gate"], s["w_up"], activation=s["case"]["activation"])
    out = {"y": y.detach()}
    if s["case"]["train"]:
        grads = torch.autograd.grad(y, (s["x"], s["w_gate"], s["w_up"]), s["dy"])
        out.update(zip(("d_x", "d_w_gate", "d_w_up"), grads))
    return out


def _plain_quant(s):
    codes, scales = _plain_quantize(s["x"].float(), s["case"]["block_rows"])
    return {"codes": codes, "scales": scales}


def _own_quant(s):
    import cuda_force_b200 as cf

    codes, scales = cf.quantize_fp8(s["x"], block_rows=s["case"]["block_rows"])
    return {"codes": codes, "scales": scales}


def _plain_fp8(s):
    x, n, k = s["x"], s["case"]["n"], s["case"]["k"]
    codes, scales = _plain_quantize(x.float(), 1)
    a = codes.float() * _plain_spread(scales, 1, *x.shape)
    w = s["codes"].float() * _plain_spread(s["scales"], 128, n, k)
    return {"y": (a @ w.t()).to(x.dtype)}


def _own_fp8(s):
    import cuda_force_b200 as cf

    return {"y": cf.linear_fp8(s["x"], s["codes"], s["scales"])}


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    if case["op"] == "gated":
        return _own_gated(state) if own else _plain_gated(state)
    if case["op"] == "quant":
        return _own_quant(state) if own else _plain_quant(state)
    return _own_fp8(state) if own else _plain_fp8(state)


def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "norm":
        c = case["cols"]
        rows = case["batch"] * case["tokens"]
        gate = {"none": 0, "channel": c, "sample": case["batch"] * c, "full": rows * c}[case["gate"]]
        weights = c * (2 if case["post"] else 1) + gate
        if not case["train"]:
            return {"bytes": size * (4 * rows * c + weights), "flops": 12 * rows * c}
        return {"bytes": size * (8 * rows * c + 2 * weights), "flops": 45 * rows * c}
    if case["op"] == "quant":
        n = case["rows"] * case["cols"]
        scales = -(-case["rows"] // case["block_rows"]) * -(-case["cols"] // BLOCK)
        return {"bytes": n * (size + 1) + 4 * scales, "flops": 3 * n}
    m, k, n = case["m"], case["k"], case["n"]
    if case["op"] == "fp8":
        scales = 4 * -(-n // BLOCK) * -(-k // BLOCK)
        return {"bytes": 2 * m * k + n * k + scales + 2 * m * n, "flops": 2 * m * n * k}
    if case["train"]:
        return {"bytes": 2 * (2 * m * k + 4 * n * k + 2 * m * n), "flops": 12 * m * n * k}
    return {"bytes": 2 * (m * k + 2 * n * k + m * n), "flops": 4 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    v = {name: t.detach().double() for name, t in s.items() if isinstance(t, torch.Tensor)}
    if case["op"] == "norm":
        return _exact_norm(case, v)
    if case["op"] == "gated":
        return _exact_gated(case, v)
    # Block scales are 32-bit numbers by definition: one division, rounded once.
    if case["op"] == "quant":
        scales = _exact_scales(s["x"], case["block_rows"])
        rows = torch.arange(case["rows"], device="cuda") // case["block_rows"]
        cols = torch.arange(case["cols"], device="cuda") // BLOCK
        return {"codes": v["x"] / scales.double()[rows][:, cols], "scales": scales.double()}
    sa = _exact_scales(s["x"], 1)
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    row_block = torch.arange(case["n"], device="cuda") // BLOCK
    for b, k0 in enumerate(range(0, case["k"], BLOCK)):
        part = s["x"][:, k0:k0 + BLOCK].float() / sa[:, b:b + 1]
        a = part.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).double() * sa[:, b:b + 1].double()
        w = v["codes"][:, k0:k0 + BLOCK] * v["scales"][row_block, b][:, None]
        y.addmm_(a, w.t())
    return {"y": y}


def _exact_scales(x, block_rows):
    rows, cols = x.shape
    pad = (0, -cols % BLOCK, 0, -rows % block_rows)
    blocks = torch.nn.functional.pad(x.abs().float(), pad)
    blocks = blocks.unflatten(1, (-1, BLOCK)).amax(2).unflatten(0, (-1, block_rows)).amax(1)
    scales = blocks / E4M3_MAX
    return scales.masked_fill(scales == 0, 1.0)


def _exact_norm(case, v):
    cols = case["cols"]
    x = v["x"].reshape(-1, cols)
    lead = (*_lead(case), cols)
    ones = torch.ones(cols, dtype=torch.float64, device="cuda")
    post = v.get("post", ones)
    gate = v.get("gate", ones).expand(lead).reshape(-1, cols)
    q = ((x * x).sum(1) / cols + EPS) ** -0.5 if case["post"] else torch.ones_like(x[:, 0])
    unit = x * q[:, None]
    h = case["scale"] * v["residual"].reshape(-1, cols) + gate * unit * post
    t = ((h * h).sum(1) / cols + EPS) ** -0.5
    hh = h * t[:, None]
    out = {"normalised": (hh * v["weight"]).reshape(lead), "residual_out": h.reshape(lead)}
    if not case["train"]:
        return out
    dn, dh = v["dn"].reshape(-1, cols), v["dh"].reshape(-1, cols)
    a = dn * v["weight"]
    d = dh + t[:, None] * (a - hh * ((a * hh).sum(1) / cols)[:, None])
    out["d_residual"] = (case["scale"] * d).reshape(lead)
    out["d_weight"] = torch.einsum("rc,rc->c", dn, hh)
    if case["gate"] != "none":
        dgate = (d * unit * post).reshape(lead)
        out["d_gate"] = {"channel": lambda z: z.sum((0, 1)), "sample": lambda z: z.sum(1, True),
                         "full": lambda z: z}[case["gate"]](dgate)
    c = d * gate
    if case["post"]:
        out["d_post"] = torch.einsum("rc,rc->c", c, unit)
        c = c * post
        c = q[:, None] * (c - unit * ((c * unit).sum(1) / cols)[:, None])
    out["d_x"] = c.reshape(lead)
    return out


def _exact_gated(case, v):
    x, wg, wu = v["x"], v["w_gate"], v["w_up"]
    g = torch.einsum("mk,nk->mn", x, wg)
    u = torch.einsum("mk,nk->mn", x, wu)
    if case["activation"] == "silu":
        s = torch.sigmoid(g)
        act, slope = g * s, s + g * s * (1 - s)
    else:
        c = (2 / math.pi) ** 0.5
        th = torch.tanh(c * g * (1 + 0.044715 * g**2))
        act = g * (1 + th) / 2
        slope = (1 + th) / 2 + g * (1 - th**2) * c * (1 + 0.134145 * g**2) / 2
    out = {"y": act * u}
    if case["train"]:
        dg, du = v["dy"] * u * slope, v["dy"] * act
        out["d_x"] = torch.einsum("mn,nk->mk", dg, wg) + torch.einsum("mn,nk->mk", du, wu)
        out["d_w_gate"] = torch.einsum("mn,mk->nk", dg, x)
        out["d_w_up"] = torch.einsum("mn,mk->nk", du, x)
    return out
