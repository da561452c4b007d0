"""linear_act in 16-bit types on each of its tiles: pairs of CTAs and single ones, whole and split sums, whole and ragged
rows, with and without a residual, against 64 bits by element and in norm."""

import pytest
import torch

from layers_util import ACTS, check_linear, half, rand
from linear_tiles import SIZES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib):
    from gaussian_2d_splat_encoder_b200 import layers

    return layers


@pytest.mark.parametrize("act,residual", [("none", True), ("gelu", False), ("silu", True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_tiles(ops, M, K, N, dtype, act, residual):
    """In norm a result is off by its rounding, at most h, and by what the sums and dz lose: less than 2e-5 (a sum over
    16384 terms of either sign loses below 1e-5 of its norm, dz h^2, z's errors pass with slopes of about 1).  A lost
    part, row block or residual is some percent."""
    x, w = rand(M, K, seed=1, dtype=dtype), rand(N, K, seed=2, dtype=dtype, scale=K ** -0.5)
    b = rand(N, seed=3, dtype=dtype)
    r = rand(M, N, seed=4, dtype=dtype) if residual else None
    dy = rand(M, N, seed=5, dtype=dtype)
    ts = [t.clone().requires_grad_(True) for t in (x, w, b)]
    rs = None if r is None else r.clone().requires_grad_(True)
    y = ops.linear_act(*ts, act=act, residual=rs)
    grads = list(torch.autograd.grad(y, ts + ([] if r is None else [rs]), dy)) + ([None] if r is None else [])
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, act=act, residual=r), y)
    check_linear(y.detach(), grads, x, w, b, r, act, dy)
    ds = [t.double().requires_grad_(True) for t in (x, w, b)]
    Y = ACTS[act](ds[0] @ ds[1].t() + ds[2]) + (0 if r is None else r.double())
    for name, a, e in zip(("y", "dx", "dw", "db"), (y.detach(), *grads), (Y.detach(), *torch.autograd.grad(Y, ds, dy.double()))):
        rel = float((a.double() - e).norm() / e.norm())
        assert rel <= half(dtype) + 2e-5, (name, rel)
