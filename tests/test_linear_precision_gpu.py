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
