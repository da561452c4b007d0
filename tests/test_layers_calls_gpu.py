"""Calls of the layer operators that torch allows around them: hooks on saved tensors, checkpoints."""

import pytest
import torch

from layers_util import rand

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops(lib):
    from gaussian_2d_splat_encoder_b200 import layers

    return layers


def both_ways(run, leaves, dy, around):
    """Gradients of run(*leaves) plainly and inside `around`."""
    plain = torch.autograd.grad(run(*leaves), leaves, dy)
    with around:
        y = run(*leaves)
    return plain, torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("view", ["slice", "unaligned", "images", "expanded"])
def test_saved_on_cpu(ops, view, dtype):
    """Saved tensors that come back compact: the same gradients, to the bit, as the layout changes no sum."""
    wide, w, b = rand(3, 50, 96, seed=1, dtype=dtype), rand(32, seed=2, shift=1.0), rand(32, seed=3)
    x = {"slice": wide[..., 32:64], "unaligned": wide[..., 5:37], "images": wide[:, ::2, :32],
         "expanded": wide[:1, :1, :32].expand(3, 50, 32)}[view].detach().requires_grad_(True)
    leaves = [x, w.requires_grad_(True), b.requires_grad_(True)]
    for act, first in (("gelu", True), ("silu", False)):
        plain, hooked = both_ways(lambda *t: ops.group_norm_act(t[0], 4, t[1], t[2], act=act, act_first=first), leaves,
                                  rand(*x.shape, seed=4, dtype=dtype), torch.autograd.graph.save_on_cpu())
        assert all(torch.equal(p, h) for p, h in zip(plain, hooked))
    wt = rand(80, 64, seed=5, dtype=dtype, scale=0.2)
    wl = (wt[::2, 32:] if view == "images" else wt[:, 3:35] if view == "unaligned" else wt[:, :32]).detach().requires_grad_(True)
    bl = rand(wl.shape[0], seed=6, dtype=dtype).requires_grad_(True)
    for act in ("none", "gelu"):
        plain, hooked = both_ways(lambda *t: ops.linear_act(*t, act=act), [x, wl, bl],
                                  rand(*x.shape[:-1], wl.shape[0], seed=7, dtype=dtype), torch.autograd.graph.save_on_cpu())
        assert all(torch.equal(p, h) for p, h in zip(plain, hooked))


def test_checkpointed(ops):
    from torch.utils.checkpoint import checkpoint

    wide, w = rand(2, 40, 96, seed=8, dtype=torch.bfloat16), rand(48, 32, seed=9, dtype=torch.bfloat16, scale=0.2)
    x = wide[..., 32:64].detach().requires_grad_(True)
    w.requires_grad_(True)

    def block(x, w):
        return ops.linear_act(ops.group_norm_act(x, 4, act="gelu", act_first=True), w, act="silu")

    dy = rand(2, 40, 48, seed=10, dtype=torch.bfloat16)
    plain = torch.autograd.grad(block(x, w), (x, w), dy)
    for reentrant in (False, True):
        y = checkpoint(block, x, w, use_reentrant=reentrant)
        if reentrant:  # (runs its own backward inside, so by .backward())
            y.backward(dy)
            got = (x.grad, w.grad)
        else:
            got = torch.autograd.grad(y, (x, w), dy)
        assert all(torch.equal(p, g) for p, g in zip(plain, got))


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_parameters_only_off_eight_channels(ops, dtype):
    """Strides on eight and twelve channels, dx not wanted: the parameters' gradients are those of the full backward
    (one pixel's row expanded over the map ends its memory at the twelfth channel)."""
    w, b = rand(12, seed=11, shift=1.0).requires_grad_(True), rand(12, seed=12).requires_grad_(True)
    wide = rand(1, 50, 16, seed=13, dtype=dtype)
    for x, dy in ((wide[..., :12], wide[..., :12]),
                  (rand(1, 1, 12, seed=14, dtype=dtype).expand(1, 50, 12), rand(1, 1, 12, seed=15, dtype=dtype).expand(1, 50, 12))):
        got = torch.autograd.grad(ops.group_norm_act(x, 3, w, b, act="silu"), (w, b), dy)
        xs = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
        ref = torch.autograd.grad(ops.group_norm_act(xs, 3, w, b, act="silu"), (xs, w, b), dy.contiguous())
        assert all(torch.equal(g, r) for g, r in zip(got, ref[1:]))


def test_a_wait_that_gave_up_is_reported(ops, lib):
    """The next call raises, once; the check function waits and raises; nothing is left behind."""
    x, w = rand(20, 16, seed=16), rand(8, 16, seed=17).requires_grad_(True)
    ref = ops.linear_act(x, w, act="silu")
    ops.check_linear_waits()
    assert lib.gs_linear_debug_wait(1025, None) == 2
    assert lib.gs_linear_debug_wait(16, None) == 0
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="gave up"):
        ops.linear_act(x, w, act="silu")
    y = ops.linear_act(x, w, act="silu")
    assert torch.equal(y, ref)
    assert lib.gs_linear_debug_wait(16, None) == 0
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="gave up"):
        torch.autograd.grad(y, w, ref.detach(), retain_graph=True)
    torch.autograd.grad(y, w, ref.detach())
    assert lib.gs_linear_debug_wait(16, None) == 0
    with pytest.raises(RuntimeError, match="gave up"):
        ops.check_linear_waits()
    ops.check_linear_waits()


def test_a_new_threads_first_call(ops):
    """Each call is the first of its thread that touches the device: a forward, and a backward of the product alone."""
    import threading

    x, w = rand(64, 32, seed=18, dtype=torch.bfloat16), rand(16, 32, seed=19, dtype=torch.bfloat16).requires_grad_(True)
    z = rand(1, 64, 32, seed=24, dtype=torch.bfloat16)
    dy = rand(64, 16, seed=23, dtype=torch.bfloat16)
    ref = [ops.linear_act(x, w), ops.group_norm_act(z, 4)]
    torch.cuda.synchronize()
    calls = [lambda: ops.linear_act(x, w), lambda: ops.group_norm_act(z, 4)]
    for call, r in zip(calls, ref):
        got = []
        t = threading.Thread(target=lambda: got.append(call()))
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert len(got) == 1 and torch.equal(got[0], r)
    (dw,) = torch.autograd.grad(ref[0], w, dy)
    assert bool(dw.isfinite().all())
