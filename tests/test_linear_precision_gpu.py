"""What linear_act's backward keeps of the activation's slope and of dz, at sizes and scales where a rounding to
fewer bits than the result's would show."""

import pytest
import torch

from layers_util import ACT_U, ACTS, U, half, least, leaf64, rand

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops(lib):
    from gaussian_2d_splat_encoder_b200 import layers

    return layers


@torch.enable_grad()
def slope64(z, act):
    z = z.detach().requires_grad_(True)
    return torch.autograd.grad(ACTS[act](z).sum(), z)[0]


def inside(got, ref, bound, what):
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                                 f"{float(((got.double() - ref).abs() / bound).max()):.3g} of it")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("M,K,N", [(1, 8, 4096), (1, 4096, 1000), (1, 8, 4095), (300, 8, 1024), (300, 8, 1023)])
def test_slopes_far_below_zero(ops, act, dtype, M, K, N):
    """x = 0, so z is the bias and dbias sums M times dy act'(bias): every slope by itself, from the one-launch
    and the split product, by whole rows and element by element.  SiLU's fp32 slope s + z s (1 - s) is good to some 64
    u of each of its two terms (the exponent's argument is rounded: |z| u <= 30 u; they cancel near z = -1.28, so
    u of the slope itself would not do), GELU's to ACT_U u (1 + |z|); the sum of M equal terms adds at most M u of
    itself."""
    x = torch.zeros(M, K, dtype=dtype, device="cuda")
    w = rand(N, K, seed=1, dtype=dtype)
    b = torch.linspace(-30, 10, N, device="cuda").to(dtype).requires_grad_(True)
    (db,) = torch.autograd.grad(ops.linear_act(x, w, b, act=act), b, torch.full((M, N), 2.0, dtype=dtype, device="cuda"))
    s = slope64(b.double(), act)
    ref = 2.0 * M * s
    z = b.detach().double()
    own = ACT_U * U * (1 + z.abs()) if act == "gelu" else 64 * U * torch.sigmoid(z) * (1 + z.abs())
    inside(db, ref, (half(dtype) + (4 + M) * U) * ref.abs() + own * 2 * M + least(dtype) + 1e-30, "dbias")


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_gradients_of_saturated_units(ops, dtype):
    """Every unit between -16 and -10 of SiLU (slopes of 1e-6 to 5e-4): dx and dweight against 64 bits, elementwise,
    with dz off by at most its own rounding."""
    M, K, N = 300, 40, 264
    x, w = rand(M, K, seed=2, dtype=dtype), rand(N, K, seed=3, dtype=dtype, scale=K ** -0.5)
    b = torch.full((N,), -13.0, dtype=dtype, device="cuda")
    dy = rand(M, N, seed=4, dtype=dtype, scale=512.0)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(ops.linear_act(xs, ws, b, act="silu"), (xs, ws), dy)
    X, W = leaf64(x), leaf64(w)
    gx, gw = torch.autograd.grad(ACTS["silu"](X @ W.t() + b.double()), (X, W), dy.double())
    with torch.no_grad():
        dz = dy.double() * slope64(X @ W.t() + b.double(), "silu")
        # z is off by at most 64 u of its terms (below 20 in all), which changes a slope by as much of itself; the
        # slope's two terms do not cancel here: their magnitudes sum to less than 1.3 of it
        edz = (half(dtype) + (64 * 1.3 + 64 * 20) * U) * dz.abs() + least(dtype)
        sums = 2 * U * (max(M, N) / 2 + 32)
        inside(dx, gx, half(dtype) * gx.abs() + (edz + sums * dz.abs()) @ W.abs() + least(dtype), "dx")
        inside(dw, gw, half(dtype) * gw.abs() + (edz + sums * dz.abs()).t() @ X.abs() + least(dtype), "dweight")


def few_bits(*shape, seed, dtype, scale):
    """Multiples of scale / 8 up to scale: short sums of their products are exact in fp32, so z is."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(-8, 9, shape, generator=g, device="cuda") * (scale / 8)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("M,K,N,dy_scale", [(20, 16, 16, 1.0), (4096, 16, 16, 1.0), (4097, 16, 16, 1.0), (16, 16, 4096, 1.0),
                                            (16, 16, 4104, 1.0), (16, 24, 5003, 1.0), (4999, 24, 19, 1.0),
                                            (333, 24, 40, 2.0 ** -20)])
def test_dz_is_not_rounded_to_the_type(ops, act, dtype, M, K, N, dy_scale):
    """z exact, so the gradients' errors are dz's in the products and the results' own rounding.  dz keeps two terms of
    x's type (h^2 of it; fp16's second term has 11 bits below fp16's smallest step), however many rows there are:
    rounded once (h) it would break the bound of dx where N is small and of dweight where M is.  dbias sums dz itself."""
    x, w = few_bits(M, K, seed=10, dtype=dtype, scale=1.0), few_bits(N, K, seed=11, dtype=dtype, scale=0.5)
    b, dy = few_bits(N, seed=12, dtype=dtype, scale=1.0), rand(M, N, seed=13, dtype=dtype, scale=dy_scale)
    ts = [t.clone().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.linear_act(*ts, act=act), ts, dy)
    X, W, B = x.double(), w.double(), b.double()
    z, D, h = X @ W.t() + B, dy.double(), half(dtype)
    dz = D * slope64(z, act)
    slope = (ACT_U * U * (1 + z.abs()) if act == "gelu" else 64 * U * torch.sigmoid(z) * (1 + z.abs())) * D.abs() + U * dz.abs()
    edz = slope + (2 ** -21 if dtype == torch.float32 else h * h) * dz.abs() + (least(dtype) * 2.0 ** -11 if dtype != torch.float32 else 0)

    def sums(n):  # as check_linear's: the tensor cores add 16 at a time and may cut instead of rounding
        return 2 * U * (n / 2 + 32)

    lo = least(dtype) + 1e-30
    inside(dx, dz @ W, h * (dz @ W).abs() + (edz + sums(N) * dz.abs()) @ W.abs() + lo, "dx")
    inside(dw, dz.t() @ X, h * (dz.t() @ X).abs() + (edz + sums(M) * dz.abs()).t() @ X.abs() + lo, "dweight")
    inside(db, dz.sum(0), h * dz.sum(0).abs() + (slope + (M / 2 + 32) * U * dz.abs()).sum(0) + lo, "dbias")


def test_fp32_infinities_and_the_largest_numbers(ops):
    """fp32 operands enter as bf16 terms: an infinity has the formula's result (64 bits' is the same), and numbers
    above bf16's largest are numbers.  Sizes of a padded row, of whole rows, of split sums."""
    for M, K, N in ((40, 33, 20), (300, 64, 72), (5, 2000, 24)):
        x, w, dy = rand(M, K, seed=20), rand(N, K, seed=21), rand(M, N, seed=22)
        w[3, 5], x[2, 5], dy[4, 1] = 0.0, 1.0, 0.5
        for at in ("x", "w", "dy"):
            a = dict(x=x.clone(), w=w.clone(), dy=dy.clone())
            a[at][1, 7], a[at][4, 9] = float("inf"), -float("inf")
            X, W = a["x"].requires_grad_(True), a["w"].requires_grad_(True)
            y = ops.linear_act(X, W)
            got = [y.detach(), *torch.autograd.grad(y, (X, W), a["dy"])]
            Xd, Wd, D = (a[k].detach().double() for k in ("x", "w", "dy"))
            for g, r in zip(got, (Xd @ Wd.t(), D @ Wd, D.t() @ Xd)):
                assert torch.equal(g.isnan(), r.isnan()) and torch.equal(g.isinf(), r.isinf())
                assert torch.equal(g[g.isinf()].double(), r[r.isinf()])
        x[1, 7], x[2, 5] = 3.4e38, -3.402823e38
        y = ops.linear_act(x, w * 2.0 ** -20)
        ref = x.double() @ (w * 2.0 ** -20).double().t()
        e = 2 * U * (K / 2 + 32) * (x.double().abs() @ (w * 2.0 ** -20).double().abs().t())
        inside(y, ref, e + 1e-30, "largest")


@pytest.mark.parametrize("M,K,N", [(8300, 1024, 4096), (8300, 1022, 4099)])
def test_fp32_parts_in_panels_and_groups(ops, M, K, N):
    """More parts than the workspace holds at once in each of the three products (17 of 16 MB for dweight): a forward
    and dx over panels of rows, the last of them short, dweight over groups of parts."""
    from layers_util import check_linear

    x, w, b = rand(M, K, seed=30), rand(N, K, seed=31, scale=K ** -0.5), rand(N, seed=32)
    r, dy = rand(M, N, seed=33), rand(M, N, seed=34)
    ts = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = ops.linear_act(ts[0], ts[1], ts[2], act="silu", residual=ts[3])
    grads = torch.autograd.grad(y, ts, dy)
    check_linear(y.detach(), grads, x, w, b, r, "silu", dy)
    ds = [t.double().requires_grad_(True) for t in (x, w, b)]
    Y = ACTS["silu"](ds[0] @ ds[1].t() + ds[2]) + r.double()
    for name, a, e in zip(("y", "dx", "dw", "db"), (y.detach(), *grads), (Y.detach(), *torch.autograd.grad(Y, ds, dy.double()))):
        rel = float((a.double() - e).norm() / e.norm())
        assert rel <= 2e-6, (name, rel)
    # parameters one by one: dbias folds beside whichever product is last
    for live in ((0, 2), (1, 2), (2,)):
        y = ops.linear_act(*[t if i in live else t.detach() for i, t in enumerate(ts[:3])], act="silu", residual=r)
        got = torch.autograd.grad(y, [ts[i] for i in live], dy)
        assert all(torch.equal(g, grads[i]) for g, i in zip(got, live))


def test_long_sums_of_one_sign(ops):
    """Sums of 2^18 positive terms with no tile to spare for splitting: an accumulator that cuts (2 u a step of 16
    terms) may run over 16384 terms, 1024 steps, so a result is within h + 2048 u + 64 u of itself; one run over them
    all loses 1.4e-3, three times fp16's h."""
    dtype, L = torch.float16, 1 << 18
    for M, K, N in ((L, 2048, 2048), (1024, L, 2304), (1024, 200, L // 2)):
        x = rand(M, K, seed=40).abs().add_(0.5).to(dtype)
        if K == L:  # forward
            w = (rand(N, K, seed=41).abs_() + 0.5).mul_(1.0 / K).to(dtype)
            y, ref = ops.linear_act(x, w), torch.zeros(M, N, dtype=torch.float64, device="cuda")
            for i in range(0, K, 1 << 15):
                ref += x[:, i:i + (1 << 15)].double() @ w[:, i:i + (1 << 15)].double().t()
        else:  # dweight over the rows, dx over the outputs
            w = torch.full((N, K), 2.0 ** -10, dtype=dtype, device="cuda").requires_grad_(True)
            dy = (rand(M, N, seed=42).abs_() + 0.5).mul_(2.0 ** -10).to(dtype)
            leaf = w if M == L else x.requires_grad_(True)
            (y,) = torch.autograd.grad(ops.linear_act(x, w), leaf, dy)
            if M == L:
                ref = torch.zeros(N, K, dtype=torch.float64, device="cuda")
                for i in range(0, M, 1 << 15):
                    ref += dy[i:i + (1 << 15)].double().t() @ x.detach()[i:i + (1 << 15)].double()
            else:
                ref = dy.double() @ w.detach().double()
        inside(y, ref, (half(dtype) + 2112 * U) * ref, (M, K, N))
        del x, w, y, ref


@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "gelu"), (torch.float16, "silu")])
@pytest.mark.parametrize("N", [4096, 4100])
def test_16_bit_parts_in_panels(ops, N, dtype, act):
    """A forward over 16448 terms has two parts, of more rows than the workspace holds at once: two panels, the second
    short, by whole rows and element by element, with bias, residual and the kept slope."""
    from layers_util import check_linear

    M, K = 9000, 16448
    x, w, b = rand(M, K, seed=50, dtype=dtype), rand(N, K, seed=51, dtype=dtype, scale=K ** -0.5), rand(N, seed=52, dtype=dtype)
    r, dy = rand(M, N, seed=53, dtype=dtype), rand(M, N, seed=54, dtype=dtype)
    ts = [t.clone().requires_grad_(True) for t in (x, b)]
    y = ops.linear_act(ts[0], w, ts[1], act=act, residual=r)
    dx, db = torch.autograd.grad(y, ts, dy)
    check_linear(y.detach(), (dx, None, db, dy), x, w, b, r, act, dy)
    Z = (x.double() @ w.double().t() + b.double()).requires_grad_(True)
    Y = ACTS[act](Z)
    (dz,) = torch.autograd.grad(Y, Z, dy.double())
    for name, a, e in (("y", y, Y + r.double()), ("dx", dx, dz @ w.double()), ("db", db, dz.sum(0))):
        rel = float((a.detach().double() - e.detach()).norm() / e.detach().norm())
        assert rel <= half(dtype) + 2e-5, (name, rel)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_16_bit_parts_in_groups(ops, act, dtype):
    """dweight over 70000 rows has five parts of 64 MB, one more than the workspace holds at once."""
    M, K, N = 70000, 4096, 4096
    x, w, dy = rand(M, K, seed=55, dtype=dtype), rand(N, K, seed=56, dtype=dtype, scale=K ** -0.5), rand(M, N, seed=57, dtype=dtype)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(ops.linear_act(x, w, act=act), w, dy)
    ref = torch.zeros(N, K, dtype=torch.float64, device="cuda")
    with torch.no_grad():
        W = w.double()
        for i in range(0, M, 10000):
            X, D = x[i:i + 10000].double(), dy[i:i + 10000].double()
            ref += (D if act == "none" else D * slope64(X @ W.t(), act)).t() @ X
    rel = float((dw.double() - ref).norm() / ref.norm())
    assert rel <= half(dtype) + 2e-5, rel
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,K,N", [(300, 24, 40), (4000, 256, 1030)])
def test_fp16_dz_beyond_its_range(ops, M, K, N):
    """Gradients near fp16's largest number times a slope of up to 1.13 pass it; dx and dweight, whose factors are small,
    do not."""
    dtype, h = torch.float16, half(torch.float16)
    x, w = few_bits(M, K, seed=60, dtype=dtype, scale=2.0 ** -6), few_bits(N, K, seed=61, dtype=dtype, scale=2.0 ** -6)
    b = torch.full((N,), 1.5, dtype=dtype, device="cuda")
    dy = (65504 - 4096 * rand(M, N, seed=62).abs()).to(dtype) * torch.where(rand(M, N, seed=63) > 0, 1.0, -1.0).to(dtype)
    ts = [t.clone().requires_grad_(True) for t in (x, w)]
    dx, dw = torch.autograd.grad(ops.linear_act(ts[0], ts[1], b, act="gelu"), ts, dy)
    X, W, D = x.double(), w.double(), dy.double()
    z = X @ W.t() + b.double()
    dz = D * slope64(z, "gelu")
    assert bool((dz.abs() > 65504).any())
    edz = ACT_U * U * (1 + z.abs()) * D.abs() + (U + h * h) * dz.abs()
    sums = [2 * U * (n / 2 + 32) for n in (N, M)]
    for got, ref, bound, what in ((dx, dz @ W, (edz + sums[0] * dz.abs()) @ W.abs(), "dx"),
                                  (dw, dz.t() @ X, (edz + sums[1] * dz.abs()).t() @ X.abs(), "dweight")):
        # long sums pass fp16's range themselves here and there (4000 terms of some 7e4 2^-7: 4e4 in the mean, one in
        # eight beyond 65520, from where on their rounding is infinite)
        over = (ref.abs() + bound >= 65504) & got.isinf()
        assert torch.equal(got[over].sign().double(), ref[over].sign()) and over.float().mean() < 0.25
        inside(torch.where(over, 0, got), torch.where(over, 0, ref), h * ref.abs() + bound + least(dtype), what)
