"""Definitions of the layer operators in float64 and the rounding bounds their kernels are held to.

A rounding to type t is off by at most h = finfo(t).eps / 2 of the value; u = 2^-24 is that of fp32, in
which the kernels compute.  Bounds are elementwise and built from the magnitudes that enter a result."""

import torch
import torch.nn.functional as F

U = 2.0 ** -24
ACTS = {"none": lambda v: v, "gelu": F.gelu, "silu": F.silu}
# a fp32 activation or slope is off by 7e-7 < 12 u absolutely (the kernels' erf and ex2 / rcp forms), its
# own argument's error passes with a slope of at most 1.13
ACT_U = 12.0


def half(t):
    return torch.finfo(t).eps / 2


def least(t):
    """Half the spacing of t's subnormals: below finfo(t).smallest_normal a rounding is off by up to this,
    whatever the value (fp16 2^-25; nothing that matters in bf16 and fp32)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def rand(*shape, seed, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def leaf64(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def norm_ref(x, G, w, b, eps, act, first):
    """(y, xh) in x's precision."""
    f = ACTS[act]
    u = f(x) if first else x
    B, C = x.shape[0], x.shape[-1]
    g = u.reshape(B, -1, G, C // G)
    m = g.mean((1, 3), keepdim=True)
    v = (g - m).square().mean((1, 3), keepdim=True)
    xh = ((g - m) / torch.sqrt(v + eps)).reshape(x.shape)
    z = xh if w is None else xh * w
    z = z if b is None else z + b
    return (z if first else f(z)), xh


def close(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} for {tuple(ref.shape)}"
    bad = ~((got - ref).abs() <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                                 f"{float(((got - ref).abs() / bound.clamp_min(1e-300)).max()):.3g} of it")


def check_norm(got, grads, x, G, w, b, eps, act, first, dy):
    """got = y; grads = (dx, dw, db) or None, of inputs x, w, b (any may lack a gradient)."""
    lo = 1e-30 + least(x.dtype)
    X, W, Bi = leaf64(x), leaf64(w), leaf64(b)
    y, xh = norm_ref(X, G, W, Bi, eps, act, first)
    B, C = x.shape[0], x.shape[-1]
    with torch.no_grad():
        u = ACTS[act](X) if first else X
        g = u.reshape(B, -1, G, C // G)
        m = g.mean((1, 3), keepdim=True)
        rs = 1 / torch.sqrt((g - m).square().mean((1, 3), keepdim=True) + eps)
        wa = torch.ones(C, dtype=torch.float64, device=x.device) if W is None else W.abs()
        ba = torch.zeros_like(wa) if Bi is None else Bi.abs()
        # errors of u, of the slice means and of their join are a few u of the largest |u| of the group
        big = g.abs().amax((1, 3), keepdim=True) + (1.0 if first else 0.0)
        exh = 32 * U * (big * rs * torch.ones_like(g)).reshape(x.shape) + 32 * U * xh.abs()
        ez = exh * wa + 4 * U * (xh.abs() * wa + ba)
        ey = ez if first else 1.13 * ez + ACT_U * U * (1 + y.abs())
    close(got, y.detach(), half(got.dtype) * y.abs() + ey + lo, "y")
    if grads is None:
        return
    leaves = [t for t in (X, W, Bi) if t is not None]
    ref = dict(zip([i for i, t in enumerate((X, W, Bi)) if t is not None], torch.autograd.grad(y, leaves, dy.double())))
    with torch.no_grad():
        D = dy.double()
        Z = leaf64(xh * (1 if W is None else W) + (0 if Bi is None else Bi))
    if first:
        dz, edz = D, torch.zeros_like(D)
    else:
        (s,) = torch.autograd.grad(ACTS[act](Z).sum(), Z)
        dz, edz = D * s, D.abs() * (ACT_U * U * (1 + Z.abs()) + ez)  # second derivatives stay below 1
    dz, xh = dz.detach(), xh.detach()
    # a sum in fp32 is off by at most its longest chain (<= 512 terms here and in the trees above it) times u
    # of the terms' magnitudes, besides the terms' own errors
    L = 512 * U
    eterm = edz * xh.abs() + dz.abs() * exh
    over = tuple(range(x.dim() - 1))
    if 1 in ref and grads[1] is not None:
        e = (eterm + L * (dz * xh).abs()).sum(over)
        close(grads[1], ref[1], half(grads[1].dtype) * ref[1].abs() + e + lo, "dweight")
    if 2 in ref and grads[2] is not None:
        e = (edz + L * dz.abs()).sum(over)
        close(grads[2], ref[2], half(grads[2].dtype) * ref[2].abs() + e + lo, "dbias")
    if grads[0] is not None:
        def mean(t):
            return t.reshape(g.shape).mean((1, 3), keepdim=True).expand(g.shape).reshape(x.shape)

        gw = dz.abs() * wa
        egw = edz * wa
        m0, m1 = mean(gw), mean(gw * xh.abs())
        em0, em1 = mean(egw) + L * m0, mean(eterm * wa) + L * m1
        rsx = (rs * torch.ones_like(g)).reshape(x.shape)
        mag = gw + m0 + xh.abs() * m1
        e = rsx * (egw + em0 + xh.abs() * em1 + exh * m1 + 64 * U * mag)
        if first and act != "none":
            # the slope is below 1.13, off by ACT_U u
            e = 1.13 * e + rsx * mag * ACT_U * U * (1 + X.detach().abs())
        close(grads[0], ref[0], half(grads[0].dtype) * ref[0].abs() + e + lo, "dx")


def check_linear(got, grads, x, w, b, r, act, dy):
    """got = y; grads = (dx, dw, db, dr) or None."""
    K, N = x.shape[-1], w.shape[0]
    X, W, Bi, R = (leaf64(t) for t in (x.reshape(-1, K), w, b, None if r is None else r.reshape(-1, N)))
    z = X @ W.t() + (0 if Bi is None else Bi)
    y = ACTS[act](z) + (0 if R is None else R)
    h, lo = half(x.dtype), 1e-30 + least(x.dtype)

    def chain(n):
        # a sum of n products: the tensor cores add 16 at a time and may cut instead of rounding (2 u); fp32
        # operands enter as three bf16 terms, six products in place of one
        return 2 * U * (n / 2 + 32)

    with torch.no_grad():
        ez = chain(K) * (X.abs() @ W.abs().t() + (0 if Bi is None else Bi.abs()))
        ey = (1.13 * ez if act != "none" else ez) + (ACT_U * U * (1 + z.abs()) if act != "none" else 0)
        close(got.reshape(-1, N), y, h * y.abs() + ey + 2 * U * y.abs() + lo, "y")
    if grads is None:
        return
    D = dy.reshape(-1, N).double()
    leaves = [t for t in (X, W, Bi, R) if t is not None]
    ref = dict(zip([i for i, t in enumerate((X, W, Bi, R)) if t is not None], torch.autograd.grad(y, leaves, D)))
    with torch.no_grad():
        Zl = leaf64(z)
    (s,) = torch.autograd.grad(ACTS[act](Zl).sum(), Zl)
    with torch.no_grad():
        dz = D * s
        # the slope is kept in steps of 1 / 49152 for 16-bit types and dz enters the products in x's type; second
        # derivatives stay below 1
        step = 0 if x.dtype == torch.float32 else 0.5 / 49152
        edz = 0 if act == "none" else (step + ez + ACT_U * U * (1 + z.abs())) * D.abs() + h * dz.abs() + lo
        M = X.shape[0]
        if grads[0] is not None:
            e = edz @ W.abs() if act != "none" else 0
            e = e + chain(N) * (dz.abs() @ W.abs())
            close(grads[0].reshape(-1, K), ref[0], h * ref[0].abs() + e + lo, "dx")
        if grads[1] is not None:
            e = edz.t() @ X.abs() if act != "none" else 0
            e = e + chain(M) * (dz.abs().t() @ X.abs())
            close(grads[1], ref[1], h * ref[1].abs() + e + lo, "dweight")
        if b is not None and grads[2] is not None:
            e = edz.sum(0) if act != "none" else 0
            close(grads[2], ref[2], h * ref[2].abs() + e + chain(M) * dz.abs().sum(0) + lo, "dbias")
        if r is not None and grads[3] is not None:
            assert torch.equal(grads[3].reshape(-1, N).double(), D), "dresidual"
