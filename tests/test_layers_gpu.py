"""Layer operators (group_norm_act, linear_act) against their definitions in float64, forward and gradients,
over types, group layouts, odd sizes and strides."""

import pytest
import torch

from layers_util import check_linear, check_norm, half, rand

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
MODES = [("none", False), ("gelu", False), ("silu", False), ("gelu", True), ("silu", True)]


@pytest.fixture(scope="module")
def ops(lib):
    from gaussian_2d_splat_encoder_b200 import layers

    return layers


def norm_case(ops, x, G, w, b, act, first, dy, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], G, leaves[1], leaves[2], eps, act=act, act_first=first)
    live = [t for t in leaves if t is not None]
    got = iter(torch.autograd.grad(y, live, dy))
    grads = [None if t is None else next(got) for t in leaves]
    assert y.is_contiguous() and y.dtype == x.dtype
    with torch.no_grad():
        assert torch.equal(ops.group_norm_act(x, G, w, b, eps, act=act, act_first=first), y)
    check_norm(y.detach(), grads, x, G, w, b, eps, act, first, dy)


NORM_SHAPES = [((1, 16, 16, 256), 8), ((2, 7, 5, 24), 3), ((3, 61, 47, 120), 6), ((1, 1, 8), 8), ((1, 1, 1), 1),
               ((2, 3, 33), 11), ((1, 40, 2048), 1), ((1, 100, 512), 512), ((5, 1, 1, 64), 8), ((3, 64), 4),
               ((70, 9, 16), 16), ((1, 3001, 7), 7), ((1, 33, 1000), 40), ((2, 50, 2047), 23), ((1, 2500, 2), 1),
               ((2, 30, 72), 9), ((1, 5000, 40), 5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,G", NORM_SHAPES)
def test_norm_shapes(ops, shape, G, dtype):
    act, first = MODES[(sum(shape) + G) % 5]
    x = rand(*shape, seed=1, dtype=dtype, scale=1.5, shift=0.3)
    w, b = rand(shape[-1], seed=2, shift=1.0), rand(shape[-1], seed=3)
    norm_case(ops, x, G, w, b, act, first, rand(*shape, seed=4, dtype=dtype))


@pytest.mark.parametrize("act,first", MODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("affine", ["both", "typed", "weight", "bias", "none"])
def test_norm_modes(ops, act, first, dtype, affine):
    x = rand(2, 19, 23, 48, seed=5, dtype=dtype)
    pt = dtype if affine == "typed" else torch.float32
    w = rand(48, seed=6, dtype=pt, shift=1.0) if affine in ("both", "typed", "weight") else None
    b = rand(48, seed=7, dtype=pt) if affine in ("both", "typed", "bias") else None
    norm_case(ops, x, 6, w, b, act, first, rand(2, 19, 23, 48, seed=8, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_strides(ops, dtype):
    """Channel slices, an NCHW map in channels_last, offsets that break 16-byte alignment, rows and images
    out of order, expanded inputs and an expanded gradient."""
    wide = rand(2, 9, 11, 96, seed=9, dtype=dtype)
    w, b = rand(32, seed=10, shift=1.0), rand(32, seed=11)
    dyw = rand(2, 9, 11, 100, seed=12, dtype=dtype)
    nchw = rand(2, 32, 9, 11, seed=13, dtype=dtype).to(memory_format=torch.channels_last)
    views = [wide[..., 32:64], wide[..., 5:37], wide[:, ::2, :, :32], wide[1:, :, 3:, 64:], nchw.permute(0, 2, 3, 1),
             wide.transpose(1, 2)[..., :32], wide[:, :1, :1, :32].expand(2, 9, 11, 32), wide[:1, ..., :32].expand(3, 9, 11, 32)]
    for k, x in enumerate(views):
        dy = rand(*x.shape, seed=20 + k, dtype=dtype)
        if x.shape == (2, 9, 11, 32):
            dy = dyw[..., 1 + k:33 + k]
        norm_case(ops, x, 4, w, b, "silu", bool(k & 1), dy)
    x = wide[..., :32]
    norm_case(ops, x, 4, w, b, "gelu", True, torch.ones((), dtype=dtype, device="cuda").expand(x.shape))


def test_norm_far_mean(ops):
    """A mean far from zero and a first pixel far from the rest: the variance is not a difference of squares."""
    x = rand(2, 5000, 16, seed=14, shift=1000.0)
    norm_case(ops, x, 2, None, None, "none", False, rand(2, 5000, 16, seed=15))
    x = rand(1, 5000, 16, seed=16)
    x[0, 0] = 1e4
    norm_case(ops, x, 4, None, None, "none", False, rand(1, 5000, 16, seed=17))
    x = torch.full((1, 77, 8), 3.25, device="cuda")
    norm_case(ops, x, 2, None, None, "none", False, rand(1, 77, 8, seed=18))


def test_norm_nan_stays_in_its_group(ops):
    x = rand(2, 40, 32, seed=19)
    ref = ops.group_norm_act(x, 4, act="gelu")
    x[1, 7, 9] = float("nan")
    y = ops.group_norm_act(x, 4, act="gelu")
    assert bool(y[1, :, 8:16].isnan().all())
    keep = torch.ones(2, 40, 32, dtype=torch.bool, device="cuda")
    keep[1, :, 8:16] = False
    assert torch.equal(y[keep], ref[keep])


def test_norm_partial_gradients(ops):
    x, w, b = rand(2, 30, 24, seed=20), rand(24, seed=21, shift=1.0), rand(24, seed=22)
    dy = rand(2, 30, 24, seed=23)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ref = torch.autograd.grad(ops.group_norm_act(full[0], 3, full[1], full[2], act="silu"), full, dy)
    for mask in range(1, 7):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        live = [i for i in range(3) if mask >> i & 1]
        got = torch.autograd.grad(ops.group_norm_act(ts[0], 3, ts[1], ts[2], act="silu"), [ts[i] for i in live], dy)
        for i, g in zip(live, got):
            assert torch.equal(g, ref[i])


def test_norm_empty(ops):
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = ops.group_norm_act(x, 2, w, act="gelu")
        assert y.shape == shape
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert gx.shape == shape and not bool(gw.any())


def test_norm_gradient_by_differences(ops):
    """The directional derivative against central differences in fp32: the step's truncation (t^2) and the
    forward's rounding (u sum|y| / t) stay below 2e-3 of the gradient's scale."""
    x, w, b = rand(1, 12, 10, 16, seed=24), rand(16, seed=25, shift=1.0), rand(16, seed=26)
    dy = rand(1, 12, 10, 16, seed=27)
    for act, first in MODES:
        ts = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(ops.group_norm_act(ts[0], 4, ts[1], ts[2], act=act, act_first=first), ts, dy)
        for i in range(3):
            v = rand(*ts[i].shape, seed=30 + i)
            t, f = 1e-2, []
            for s in (t, -t):
                a = [p.detach() + (s * v if j == i else 0) for j, p in enumerate(ts)]
                f.append(float((ops.group_norm_act(a[0], 4, a[1], a[2], act=act, act_first=first).double() * dy).sum()))
            num, ana = (f[0] - f[1]) / (2 * t), float((grads[i].double() * v).sum())
            assert abs(num - ana) <= 2e-3 * float(grads[i].double().norm() * v.double().norm()), (act, first, i)


# ------------------------------------------------------------------------------------------ linear
def linear_case(ops, x, w, b, r, act, dy):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y = ops.linear_act(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3])
    live = [t for t in leaves if t is not None]
    got = iter(torch.autograd.grad(y, live, dy))
    grads = [None if t is None else next(got) for t in leaves]
    assert y.is_contiguous() and y.dtype == x.dtype and y.shape == x.shape[:-1] + (w.shape[0],)
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, act=act, residual=r), y)
    check_linear(y.detach(), grads, x, w, b, r, act, dy)


LINEAR_SIZES = [(1, 1, 1), (1, 256, 1024), (4, 256, 1024), (2, 4097, 3), (16, 512, 96), (17, 40, 264), (100, 257, 18),
                (129, 64, 64), (128, 128, 128), (300, 133, 75), (1000, 8, 1000), (2500, 384, 128), (777, 1000, 520),
                (5000, 3, 5), (9216, 257, 18), (20000, 64, 32), (64, 4096, 256), (513, 72, 2056)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", LINEAR_SIZES)
def test_linear_sizes(ops, M, K, N, dtype):
    act = ("none", "gelu", "silu")[(M + N) % 3]
    x, w, b = rand(M, K, seed=40, dtype=dtype), rand(N, K, seed=41, dtype=dtype, scale=K ** -0.5), rand(N, seed=42, dtype=dtype)
    r = rand(M, N, seed=43, dtype=dtype) if M % 2 else None
    linear_case(ops, x, w, b, r, act, rand(M, N, seed=44, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("with_bias,with_residual", [(True, True), (True, False), (False, True), (False, False)])
def test_linear_modes(ops, dtype, act, with_bias, with_residual):
    for M in (3, 333):
        x, w = rand(M, 3, 80, seed=45, dtype=dtype), rand(56, 80, seed=46, dtype=dtype, scale=0.11)
        b = rand(56, seed=47, dtype=dtype) if with_bias else None
        r = rand(M, 3, 56, seed=48, dtype=dtype) if with_residual else None
        linear_case(ops, x, w, b, r, act, rand(M, 3, 56, seed=49, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_strides(ops, dtype):
    """Channel slices with and without 16-byte alignment, a strided weight, residual and gradient, transposed
    and expanded tensors."""
    wide = rand(250, 200, seed=50, dtype=dtype)
    wt = rand(150, 120, seed=51, dtype=dtype, scale=0.1)
    ro = rand(250, 100, seed=52, dtype=dtype)
    for k, (x, w) in enumerate([(wide[:, 64:144], wt[:72, 8:88]), (wide[:, 3:83], wt[::2, 1:81]),
                                (wide[::3, :80], wt.t()[:, 70:]), (rand(80, 250, seed=53, dtype=dtype).t(), wt[3:60, :80]),
                                (wide[:1, :80].expand(250, 80), wt[:64, :80]), (wide[7:8, :80], wt[:1, 40:])]):
        M, N = x.shape[0], w.shape[0]
        r = ro[:M, 5:5 + N] if N <= 90 else None
        dy = rand(M, N + 3, seed=54 + k, dtype=dtype)[:, 1:N + 1]
        linear_case(ops, x, w, rand(N, seed=55, dtype=dtype), r, "silu", dy)
    x, w = wide[:, :80], wt[:64, :80]
    linear_case(ops, x, w, None, None, "gelu", torch.ones((), dtype=dtype, device="cuda").expand(250, 64))


def test_linear_long_sums(ops):
    """dweight and dbias sum over all rows: many, in every type."""
    for dtype in TYPES:
        x, w = rand(70001, 24, seed=56, dtype=dtype), rand(20, 24, seed=57, dtype=dtype, scale=0.2)
        linear_case(ops, x, w, rand(20, seed=58, dtype=dtype), None, "gelu", rand(70001, 20, seed=59, dtype=dtype, shift=0.1))


@pytest.mark.parametrize("M,K,N", [(70000, 200, 300), (300, 4096, 130), (600, 150, 4096)])
def test_linear_fp32_keeps_fp32_accuracy(ops, M, K, N):
    """Long sums in each of the three products: in norm within 2e-6, 32 roundings' worth (u = 2^-24), however
    long the sum."""
    x, w, b = rand(M, K, seed=300), rand(N, K, seed=301, scale=K ** -0.5), rand(N, seed=302)
    dy = rand(M, N, seed=303)
    ts = [t.requires_grad_(True) for t in (x, w, b)]
    y = ops.linear_act(*ts, act="gelu")
    grads = torch.autograd.grad(y, ts, dy)
    ds = [t.detach().double().requires_grad_(True) for t in ts]
    Y = torch.nn.functional.gelu(ds[0] @ ds[1].t() + ds[2])
    ref = torch.autograd.grad(Y, ds, dy.double())
    for name, a, e in zip(("y", "dx", "dw", "db"), (y.detach(), *grads), (Y.detach(), *ref)):
        rel = float((a.double() - e).norm() / e.norm())
        assert rel <= 2e-6, (name, rel)


def test_linear_nan_stays_in_its_row(ops):
    for dtype in TYPES:
        x, w, b = rand(300, 72, seed=60, dtype=dtype), rand(40, 72, seed=61, dtype=dtype), rand(40, seed=62, dtype=dtype)
        ref = ops.linear_act(x, w, b, act="gelu")
        x[37, 5], x[200, 71] = float("nan"), float("inf")
        y = ops.linear_act(x, w, b, act="gelu")
        keep = torch.ones(300, dtype=torch.bool, device="cuda")
        keep[[37, 200]] = False
        assert torch.equal(y[keep], ref[keep])
        assert bool(y[37].isnan().all()) and not bool(y[200].isfinite().all())


def test_linear_empty(ops):
    x = torch.empty(0, 5, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, b = (rand(*s, seed=63, dtype=torch.bfloat16).requires_grad_(True) for s in ((8, 16), (8,)))
    y = ops.linear_act(x, w, b, act="gelu")
    assert y.shape == (0, 5, 8)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert gx.shape == x.shape and not bool(gw.any()) and not bool(gb.any())


def test_linear_partial_gradients(ops):
    x, w, b, r = rand(200, 48, seed=64), rand(40, 48, seed=65), rand(40, seed=66), rand(200, 40, seed=67)
    dy = rand(200, 40, seed=68)
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    ref = torch.autograd.grad(ops.linear_act(full[0], full[1], full[2], act="silu", residual=full[3]), full, dy)
    for mask in range(1, 15):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b, r))]
        live = [i for i in range(4) if mask >> i & 1]
        y = ops.linear_act(ts[0], ts[1], ts[2], act="silu", residual=ts[3])
        for i, g in zip(live, torch.autograd.grad(y, [ts[i] for i in live], dy)):
            assert torch.equal(g, ref[i])


def test_linear_gradient_by_differences(ops):
    """As test_norm_gradient_by_differences."""
    x, w, b = rand(30, 24, seed=70), rand(20, 24, seed=71, scale=0.2), rand(20, seed=72)
    dy = rand(30, 20, seed=73)
    for act in ("none", "gelu", "silu"):
        ts = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(ops.linear_act(ts[0], ts[1], ts[2], act=act), ts, dy)
        for i in range(3):
            v = rand(*ts[i].shape, seed=74 + i)
            t, f = 1e-2, []
            for s in (t, -t):
                a = [p.detach() + (s * v if j == i else 0) for j, p in enumerate(ts)]
                f.append(float((ops.linear_act(a[0], a[1], a[2], act=act).double() * dy).sum()))
            num, ana = (f[0] - f[1]) / (2 * t), float((grads[i].double() * v).sum())
            assert abs(num - ana) <= 2e-3 * float(grads[i].double().norm() * v.double().norm()), (act, i)


# ----------------------------------------------------------------------------------- both together
def _block(ops, x, p):
    """A fine-decoder stage's tail and a residual layer on it, then a head: GELU -> GroupNorm, widen, back
    with a residual, 18 outputs."""
    h = ops.group_norm_act(x, 8, p["gw"], p["gb"], act="gelu", act_first=True)
    t = ops.linear_act(h, p["w1"], p["b1"], act="silu")
    t = ops.linear_act(t, p["w2"], p["b2"], residual=h)
    t = ops.group_norm_act(t, 4, p["gw"], p["gb"], act="silu")
    return ops.linear_act(t, p["w3"], p["b3"])


def _block_params(dtype, C=64, seed=80):
    p = dict(gw=rand(C, seed=seed, shift=1.0, scale=0.2), gb=rand(C, seed=seed + 1, scale=0.2),
             w1=rand(4 * C, C, seed=seed + 2, scale=C ** -0.5, dtype=dtype), b1=rand(4 * C, seed=seed + 3, dtype=dtype),
             w2=rand(C, 4 * C, seed=seed + 4, scale=(4 * C) ** -0.5, dtype=dtype), b2=rand(C, seed=seed + 5, dtype=dtype),
             w3=rand(18, C, seed=seed + 6, scale=C ** -0.5, dtype=dtype), b3=rand(18, seed=seed + 7, dtype=dtype))
    return {k: v.requires_grad_(True) for k, v in p.items()}


@pytest.mark.parametrize("dtype", TYPES)
def test_block_trains(ops, dtype):
    """The operators one after another, as a trained stage and head use them: outputs and all gradients against
    the same block in float64.  Every operator rounds once to its type (h), so each of the five layers adds
    about h of its values' norm forward and again backward: at most 16 h in norm, and 1e-5 in fp32."""
    from layers_util import ACTS, norm_ref

    x = rand(2, 24, 20, 64, seed=79, dtype=dtype).requires_grad_(True)
    p = _block_params(dtype)
    y = _block(ops, x, p)
    dy = rand(*y.shape, seed=78, dtype=dtype)
    grads = torch.autograd.grad(y, [x, *p.values()], dy)
    X = x.detach().double().requires_grad_(True)
    P = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    h = norm_ref(X, 8, P["gw"], P["gb"], 1e-5, "gelu", True)[0]
    t = ACTS["silu"](h @ P["w1"].t() + P["b1"])
    t = t @ P["w2"].t() + P["b2"] + h
    t = norm_ref(t, 4, P["gw"], P["gb"], 1e-5, "silu", False)[0]
    Y = t @ P["w3"].t() + P["b3"]
    ref = torch.autograd.grad(Y, [X, *P.values()], dy.double())
    tol = max(16 * half(dtype), 1e-5)
    for name, a, e in zip(["y", "x", *p], [y, *grads], [Y, *ref]):
        rel = float((a.detach().double() - e.detach()).norm() / e.detach().norm())
        assert rel <= tol, f"{name}: {rel:.3g} against {tol:.3g}"


def test_same_bits_again(ops):
    x = rand(2, 40, 44, 64, seed=81, dtype=torch.bfloat16).requires_grad_(True)
    p = _block_params(torch.bfloat16)

    def once():
        y = _block(ops, x, p)
        return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], torch.ones_like(y))]

    a = once()
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(a, once()))


def test_other_stream_and_two_at_once(ops):
    """Two streams run the block at the same time on their own inputs; each gets what it gets alone."""
    p = _block_params(torch.float16)
    xs = [rand(2, 64, 64, 64, seed=82 + k, dtype=torch.float16).requires_grad_(True) for k in range(2)]

    def once(x):
        y = _block(ops, x, p)
        return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], torch.ones_like(y))]

    alone = [once(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(once(xs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(u, v) for u, v in zip(g, alone[k]))


def test_captured_and_replayed(ops):
    """A training step of the block in a CUDA graph: replays on new inputs match eager calls, two graphs replayed
    on two streams at once do not disturb each other."""
    graphs = []
    for k in range(2):
        x = rand(1, 48, 40, 64, seed=84 + k, dtype=torch.bfloat16).requires_grad_(True)
        p = _block_params(torch.bfloat16, seed=90 + 10 * k)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                y = _block(ops, x, p)
                torch.autograd.grad(y, [x, *p.values()], torch.ones_like(y))
        torch.cuda.current_stream().wait_stream(s)
        del y
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = _block(ops, x, p)
            out = [y.detach(), *torch.autograd.grad(y, [x, *p.values()], torch.ones_like(y))]
        graphs.append((g, x, p, out, torch.cuda.Stream()))
    for step in range(3):
        for k, (g, x, p, out, s) in enumerate(graphs):
            with torch.no_grad():
                x.copy_(rand(*x.shape, seed=100 + 2 * step + k, dtype=x.dtype))
        torch.cuda.synchronize()
        for g, x, p, out, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, x, p, out, s in graphs:
            y = _block(ops, x, p)
            ref = [y.detach(), *torch.autograd.grad(y, [x, *p.values()], torch.ones_like(y))]
            assert all(torch.equal(u, v) for u, v in zip(out, ref))


def test_offsets_past_32_bits(ops):
    """Maps of more than 2^31 elements: the last rows against a call on those rows alone (both within one bf16
    rounding of the same value, so at most a step of 2^-7 apart)."""
    x = torch.empty(3, 1 << 20, 704, device="cuda", dtype=torch.bfloat16)
    x[:2].fill_(0.5)
    x[2] = rand(1 << 20, 704, seed=120, dtype=torch.bfloat16)
    w = rand(704, seed=121, shift=1.0)
    xr = x.requires_grad_(True)
    y = ops.group_norm_act(xr, 8, w, act="gelu")
    (dx,) = torch.autograd.grad(y, xr, y.detach())
    tail = x.detach()[2:].clone().requires_grad_(True)
    yt = ops.group_norm_act(tail, 8, w, act="gelu")
    (dt,) = torch.autograd.grad(yt, tail, yt.detach())
    for a, e in ((y[2, -99999:], yt[0, -99999:]), (dx[2, -99999:], dt[0, -99999:])):
        assert torch.allclose(a.float(), e.float(), rtol=2 ** -6, atol=2 ** -6)
    del y, dx, yt, dt, tail, xr, x
    torch.cuda.empty_cache()
    M = (1 << 21) + 77
    x, w = rand(M, 16, seed=122, dtype=torch.bfloat16), rand(1048, 16, seed=123, dtype=torch.bfloat16)
    xr = x.requires_grad_(True)
    y = ops.linear_act(xr, w, act="silu")
    (dx,) = torch.autograd.grad(y, xr, y.detach())
    tail = x.detach()[-1000:].clone().requires_grad_(True)
    yt = ops.linear_act(tail, w, act="silu")
    (dt,) = torch.autograd.grad(yt, tail, yt.detach())
    assert torch.equal(y[-1000:], yt)
    # the same rounded dz in both; fp32 sums of 1048 terms of some 10 in another order, then one rounding each
    assert torch.allclose(dx[-1000:].float(), dt.float(), rtol=2 ** -6, atol=0.05)
    del y, dx, x, xr
    torch.cuda.empty_cache()


def test_refusals_on_the_device(ops):
    x = rand(2, 4, 16, seed=110)
    with pytest.raises(ValueError, match="divide"):
        ops.group_norm_act(x, 3)
    with pytest.raises(ValueError, match="act must be"):
        ops.group_norm_act(x, 4, act="relu")
    with pytest.raises(ValueError, match="float32 or"):
        ops.group_norm_act(x.bfloat16(), 4, torch.ones(16, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="weight must be"):
        ops.group_norm_act(x, 4, torch.ones(15, device="cuda"))
    with pytest.raises(ValueError, match="one type"):
        ops.group_norm_act(x.half(), 4, torch.ones(16, device="cuda"), torch.ones(16, device="cuda").half())
    with pytest.raises(ValueError, match="2048"):
        ops.group_norm_act(torch.ones(1, 2, 2056, device="cuda"), 8)
    with pytest.raises(ValueError, match="float32, bfloat16"):
        ops.group_norm_act(x.double(), 4)
    w = rand(8, 16, seed=111)
    with pytest.raises(ValueError, match="like x"):
        ops.linear_act(x, w.half())
    with pytest.raises(ValueError, match="weight"):
        ops.linear_act(x, w.t())
    with pytest.raises(ValueError, match="residual"):
        ops.linear_act(x, w, residual=rand(4, 8, seed=112))
    with pytest.raises(ValueError, match="bias"):
        ops.linear_act(x, w, torch.ones(7, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.linear_act(x, w.cpu())
    y = ops.linear_act(x.requires_grad_(True), w, act="gelu")
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_no_wait_gave_up(ops, lib):
    """No bounded device wait of the linear kernels ran out in this process."""
    import ctypes as C

    flag = C.c_int(-1)
    torch.cuda.synchronize()
    assert lib.gs_linear_error_flag(C.byref(flag)) == 0 and flag.value == 0
