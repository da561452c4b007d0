"""Measured cases of the layer operators: GroupNorm with an activation on channels-last maps and the
linear layer with bias, activation and residual, each forward alone and with its gradients.

``run`` computes a case in plain torch operations, or, where ``own`` is set, with the calls a user makes
of ``gaussian_2d_splat_encoder_b200.layers``.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _norm(name, B, h, w, C, groups, dtype, act, first, train):
    return dict(name=name, op="norm", B=B, h=h, w=w, C=C, groups=groups, dtype=dtype, act=act, first=first,
                train=train)


def _linear(name, M, K, N, dtype, act, residual, train):
    return dict(name=name, op="linear", M=M, K=K, N=N, dtype=dtype, act=act, residual=residual, train=train)


def listed():
    return [
        # one 128 x 128 image's stride-8 map in the encoder's order (GELU, then 8 groups): a launch's latency
        _norm("norm_128", 1, 16, 16, 256, 8, "bf16", "gelu", True, False),
        # the same stage at 768 x 768, the released configuration
        _norm("norm_768", 1, 96, 96, 256, 8, "bf16", "gelu", True, False),
        # four images' stride-2 maps, the largest the encoder normalises; norm before the activation
        _norm("norm_stride2_batch", 4, 384, 384, 64, 8, "bf16", "silu", False, False),
        # training the fine decoder's stage on a batch of four at 768 x 768
        _norm("norm_train_batch", 4, 192, 192, 128, 8, "bf16", "gelu", True, True),
        # training on odd crops in single precision: 20 channels per group, sides that no tile divides
        _norm("norm_train_odd", 3, 61, 47, 120, 6, "fp32", "silu", False, True),
        # pooled features of four images into another model's width: a launch's latency
        _linear("linear_pooled", 4, 256, 1024, "fp16", "gelu", False, False),
        # a coarse head's 18 outputs from 257 channels (256 and the image gradient) at 768 x 768
        _linear("linear_head", 9216, 257, 18, "bf16", "none", False, False),
        # the stride-4 latents of a 768 x 768 image widened by four
        _linear("linear_widen", 36864, 128, 512, "bf16", "gelu", False, False),
        # tokens of eight images in a wide model, back onto its residual stream
        _linear("linear_wide", 16384, 4096, 4096, "bf16", "none", True, False),
        # a training step of a residual layer on the stride-4 tokens of one image
        _linear("linear_train", 36864, 256, 1024, "bf16", "gelu", True, True),
        # a training step with every size odd for the hardware: the fine head's 133 channels
        _linear("linear_train_odd", 10007, 133, 75, "fp16", "silu", False, True),
        # the encoder's public maps are single precision: 256 channels kept that way
        _linear("linear_fp32_train", 9216, 256, 256, "fp32", "gelu", False, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    dtype, act = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["none", "gelu", "silu"])
    train = rng.random() < 0.5
    if rng.random() < 0.5:
        most = (16 << 20) if train else (36 << 20)
        while True:
            groups = rng.choice([1, 2, 4, 6, 8, 8, 16, 32])
            per = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 16, 16, 20, 32])
            c = dict(op="norm", B=rng.randint(1, 8), h=_log(rng, 4, 400), w=_log(rng, 4, 400), C=groups * per,
                     groups=groups, dtype=dtype, act=act, first=rng.random() < 0.5, train=train)
            n = c["B"] * c["h"] * c["w"] * c["C"]
            if 2048 <= n <= (most // 2 if dtype == "fp32" else most):
                return c
    most = 2.5e11 / (3 if train else 1) / (4 if dtype == "fp32" else 1)
    while True:
        c = dict(op="linear", M=_log(rng, 1, 150000), K=_log(rng, 3, 4096), N=_log(rng, 3, 4096), dtype=dtype, act=act,
                 residual=rng.random() < 0.4, train=train)
        M, K, N = c["M"], c["K"], c["N"]
        if M * K * N <= most and M * (K + 2 * N) * SIZE[dtype] <= 3e8:
            return c


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    t = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = dict(case)
    if case["op"] == "norm":
        B, h, w, C = case["B"], case["h"], case["w"], case["C"]
        # a convolution's outputs: every channel has a mean and a spread of its own
        x = randn(B, h, w, C) * (0.5 + randn(C).abs()) + randn(C)
        s.update(x=x.to(t), weight=1 + 0.2 * randn(C), bias=0.2 * randn(C))
        if case["train"]:
            s.update(dy=randn(B, h, w, C).to(t))
        leaves = ("x", "weight", "bias")
    else:
        M, K, N = case["M"], case["K"], case["N"]
        s.update(x=randn(M, K).to(t), weight=(randn(N, K) / math.sqrt(K)).to(t), bias=(0.1 * randn(N)).to(t))
        s.update(residual=randn(M, N).to(t) if case["residual"] else None)
        if case["train"]:
            s.update(dy=randn(M, N).to(t))
        leaves = ("x", "weight", "bias") + (("residual",) if case["residual"] else ())
    s.update(leaves=leaves)
    if case["train"]:
        for k in leaves:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------- the plain form
def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_norm(s):
    x = s["x"].detach().float()
    B, G, C = x.shape[0], s["groups"], x.shape[-1]
    weight, bias = s["weight"].detach().float(), s["bias"].detach().float()
    u = _act(x, s["act"]) if s["first"] else x
    u = u.reshape(B, -1, G, C // G)
    mean = u.mean((1, 3), keepdim=True)
    d = u - mean
    rstd = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + EPS)
    xh = d * rstd
    z = xh.reshape(B, -1, C) * weight + bias
    y = z if s["first"] else _act(z, s["act"])
    y = y.reshape(x.shape).to(s["x"].dtype)
    if not s["train"]:
        return y
    dz = s["dy"].float().reshape(B, -1, C)
    if not s["first"]:
        dz = dz * _act_slope(z, s["act"])
    g = (dz * weight).reshape(B, -1, G, C // G)
    du = (g - g.mean((1, 3), keepdim=True) - xh * (g * xh).mean((1, 3), keepdim=True)) * rstd
    dx = du.reshape(x.shape)
    if s["first"]:
        dx = dx * _act_slope(x, s["act"])
    dweight = (dz * xh.reshape(B, -1, C)).sum((0, 1))
    return [y, dx.to(s["x"].dtype), dweight, dz.sum((0, 1))]


def _plain_linear(s):
    x, weight, bias = (s[k].detach().float() for k in ("x", "weight", "bias"))
    t = s["x"].dtype
    z = x @ weight.t() + bias
    y = _act(z, s["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    y = y.to(t)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    dz = dy * _act_slope(z, s["act"])
    out = [y, (dz @ weight).to(t), (dz.t() @ x).to(t), dz.sum(0).to(t)]
    return out + ([s["dy"]] if s["residual"] is not None else [])


def run(state):
    s = state
    if own:
        from gaussian_2d_splat_encoder_b200 import layers

        if s["op"] == "norm":
            y = layers.group_norm_act(s["x"], s["groups"], s["weight"], s["bias"], EPS, act=s["act"],
                                      act_first=s["first"])
        else:
            y = layers.linear_act(s["x"], s["weight"], s["bias"], act=s["act"], residual=s["residual"])
        if not s["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])]
    with torch.no_grad():
        return _plain_norm(s) if s["op"] == "norm" else _plain_linear(s)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, C = case["B"] * case["h"] * case["w"] * case["C"], case["C"]
        # x -> y; a training step also dy -> dx and the two parameter gradients
        return {"bytes": n * size * (4 if case["train"] else 2) + C * 4 * (4 if case["train"] else 2),
                "flops": n * (60 if case["train"] else 25)}
    M, K, N = case["M"], case["K"], case["N"]
    maps = M * K + M * N * (2 if case["residual"] else 1)
    if case["train"]:
        maps += M * K + M * N * (2 if case["residual"] else 1)
    params = (N * K + N) * (2 if case["train"] else 1)
    return {"bytes": (maps + params) * size, "flops": 2 * M * N * K * (3 if case["train"] else 1)}


# --------------------------------------------------------------- the definition in 64 bits, by autograd
def exact(case, seed):
    s = prepare(case, seed)
    F = torch.nn.functional
    named = {"gelu": F.gelu, "silu": F.silu, "none": lambda v: v}[case["act"]]
    leaves = {k: s[k].detach().double().requires_grad_(bool(case["train"])) for k in s["leaves"]}
    with torch.enable_grad():
        if case["op"] == "norm":
            u = leaves["x"].movedim(-1, 1)
            args = (case["groups"], None, None, EPS)
            wide = (-1, 1, 1)
            if case["first"]:
                y = F.group_norm(named(u), *args) * leaves["weight"].view(wide) + leaves["bias"].view(wide)
            else:
                y = named(F.group_norm(u, *args) * leaves["weight"].view(wide) + leaves["bias"].view(wide))
            y = y.movedim(1, -1)
        else:
            y = named(F.linear(leaves["x"], leaves["weight"], leaves["bias"]))
            if case["residual"]:
                y = y + leaves["residual"]
        if not case["train"]:
            return y.detach().contiguous()
        grads = torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
    return [y.detach().contiguous(), *(g.contiguous() for g in grads)]
