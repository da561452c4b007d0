"""What the layer operators hand to the library, seen on the CPU: autograd runs in earnest, the launches are recorded
instead of made."""

import ctypes as C

import pytest
import torch


class Recorder:
    """The library with the four launching entries replaced by a list of (name, descriptor's fields, arguments)."""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        if not name.endswith(("_fwd", "_bwd")):
            return getattr(self.lib, name)

        def call(desc, *args):
            d = desc._obj
            self.calls.append((name, {f: getattr(d, f) for f, _ in d._fields_}, args))
            return 0

        return call


@pytest.fixture
def ops(lib, monkeypatch):
    from gaussian_2d_splat_encoder_b200 import _lib, layers

    rec = Recorder(lib)
    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(layers, "_elsewhere", lambda dev: False)
    monkeypatch.setattr(layers, "_raw_stream", lambda index: 0)
    layers._norm_plan.cache_clear()
    layers._linear_plan.cache_clear()
    layers.rec = rec
    yield layers
    layers._norm_plan.cache_clear()
    layers._linear_plan.cache_clear()
    del layers.rec


def compact_copies():
    """Saved tensors come back as copies of their own, as torch.autograd.graph.save_on_cpu hands them back."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format),
                                                    lambda t: t)


@pytest.mark.parametrize("view", ["slice", "expanded", "images"])
def test_norm_backward_takes_the_layout_of_what_it_reads(ops, view):
    wide = torch.randn(2, 5, 96)
    x = {"slice": wide[..., 32:64], "expanded": wide[:1, :1, :32].expand(2, 5, 32), "images": wide[:, ::2, :32]}[view]
    x = x.detach().requires_grad_(True)
    with compact_copies():
        y = ops.group_norm_act(x, 4, act="gelu")
    torch.autograd.grad(y, x, torch.zeros_like(y))
    (_, fwd, _), (_, bwd, _) = ops.rec.calls
    assert (fwd["x_row"], fwd["x_img"]) == {"slice": (96, 480), "expanded": (0, 0), "images": (192, 480)}[view]
    assert (bwd["x_row"], bwd["x_img"]) == (32, 32 * x.shape[1])


@pytest.mark.parametrize("offset", [0, 3])
def test_linear_backward_takes_the_layout_of_what_it_reads(ops, offset):
    wide, wt = torch.randn(9, 200), torch.randn(50, 120)
    x = wide[:, offset:offset + 80].detach().requires_grad_(True)
    w = wt[::2, offset:offset + 80].detach().requires_grad_(True)
    with compact_copies():
        y = ops.linear_act(x, w, act="silu")
    torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    (_, fwd, _), (_, bwd, args) = ops.rec.calls
    assert (fwd["ldx"], fwd["ldw"]) == (200, 240) and bool(fwd["unaligned"] & 3) == bool(offset)
    assert (bwd["ldx"], bwd["ldw"]) == (80, 80)
    assert bwd["unaligned"] == sum(bit << k for k, bit in enumerate([args[0] & 15 != 0, args[1] & 15 != 0, args[3] & 15 != 0]))


def test_plain_backward_keeps_the_forward_layout(ops):
    x = torch.randn(2, 5, 96)[..., 32:64].requires_grad_(True)
    y = ops.group_norm_act(x, 4)
    torch.autograd.grad(y, x, torch.zeros_like(y))
    assert all((d["x_row"], d["x_img"]) == (96, 480) for _, d, _ in ops.rec.calls)


@pytest.mark.parametrize("change", [lambda t: t.double(), lambda t: t[..., :1], lambda t: t.to("meta")])
def test_changed_saved_tensors_are_refused(ops, change):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        for y in (ops.group_norm_act(torch.randn(2, 5, 32, requires_grad=True), 4),
                  ops.linear_act(torch.randn(5, 32, requires_grad=True), torch.randn(8, 32))):
            with pytest.raises(RuntimeError, match="saved tensor came back"):
                y.sum().backward()
    assert [n for n, _, _ in ops.rec.calls] == ["gs_group_norm_act_fwd", "gs_linear_act_fwd"]


@pytest.mark.parametrize("which", range(4))
def test_dual_tensors_are_refused(ops, which):
    from torch.autograd import forward_ad

    ts = [torch.randn(5, 32), torch.randn(8, 32), torch.randn(8), torch.randn(5, 8)]
    with forward_ad.dual_level():
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.linear_act(ts[0], ts[1], ts[2], act="gelu", residual=ts[3])
        ns = [torch.randn(2, 5, 8), torch.randn(8), torch.randn(8)]
        if which < 3:
            ns[which] = forward_ad.make_dual(ns[which], torch.ones_like(ns[which]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.group_norm_act(ns[0], 4, ns[1], ns[2])
    assert not ops.rec.calls
    # without a tangent a dual level changes nothing
    with forward_ad.dual_level():
        ops.linear_act(torch.randn(5, 32), torch.randn(8, 32))
        ops.group_norm_act(torch.randn(2, 5, 8), 4)
    assert len(ops.rec.calls) == 2


def test_dual_gradients_are_refused(ops):
    from torch.autograd import forward_ad

    for y, x in ((ops.group_norm_act(x, 4), x) if k else (ops.linear_act(x, torch.randn(8, 32)), x)
                 for k, x in enumerate(torch.randn(2, 5, 32, requires_grad=True) for _ in range(2))):
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, forward_ad.make_dual(torch.zeros_like(y), torch.ones_like(y)))
    assert all(n.endswith("_fwd") for n, _, _ in ops.rec.calls)


def test_function_transforms_are_refused(ops):
    x, w = torch.randn(2, 5, 8), torch.randn(3, 8)
    for f in (lambda t: ops.group_norm_act(t, 4).sum(), lambda t: ops.linear_act(t, w).sum()):
        for transform in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.grad(f)(x),
                          lambda: torch.func.vmap(f)(x.unsqueeze(1))):
            with pytest.raises(RuntimeError):
                transform()
    assert not ops.rec.calls


@pytest.mark.parametrize("images", [(1 << 30) + 1, (1 << 32) + 4])
def test_more_images_than_the_descriptor_holds(ops, images):
    with pytest.raises(ValueError, match="unsupported sizes"):
        ops.group_norm_act(torch.ones(1, 1, 1).expand(images, 1, 1), 1)
    assert not ops.rec.calls


def test_pending_signs_are_applied(ops, monkeypatch):
    """Real views of conjugates (z.conj().imag) carry a sign that is not in memory yet."""
    seen = []

    def reader(name):
        def call(desc, *args):
            def first(p):
                return C.cast(p, C.POINTER(C.c_float))[0]

            # x, weight, bias (and the residual, where the linear forward has it)
            seen.append([first(p) for p in args[:4 if "linear" in name else 3]])
            return 0

        return call

    for name in ("gs_group_norm_act_fwd", "gs_linear_act_fwd"):
        setattr(ops.rec, name, reader(name))
    for view in (torch._neg_view, lambda t: torch.complex(torch.zeros_like(t), t).conj().imag):
        x, p = view(torch.full((2, 5, 1), 3.0)), view(torch.full((1,), 5.0))
        assert x.is_neg() and p.is_neg()
        ops.group_norm_act(x, 1, p, p)
        ops.linear_act(x, p.view(1, 1), p, residual=x)
    assert seen == [[-3, -5, -5], [-3, -5, -5, -3]] * 2


def test_linear_workspace_is_bounded(lib, ops):
    """fp32 sums of many parts: beside the operands' terms (6 bytes an element) the workspace holds at most 256 MiB of
    parts, or 256 rows' or two of them, and the column sums; it does not grow with M N K."""
    size, up8 = lib.gs_linear_act_workspace_size, lambda n: (n + 7) // 8 * 8
    for M, K, N in ((16384, 4096, 4096), (589824, 1024, 1024), (65536, 4096, 4096), (4 << 20, 512, 300), (1 << 20, 2048, 130),
                    (300, 1 << 17, 4096), (5, 4096, 1 << 17)):
        d = ops._LinearDesc(M=M, N=N, K=K, dtype=0, act=1, ldx=K, ldw=K, ldr=N, ldy=N)
        terms = [6 * M * up8(K), 6 * N * up8(K), 6 * M * up8(N)]

        def most(rows, cols, k):  # of a product [rows][cols] over k
            part = up8(cols) * 4
            return max(256 << 20, 256 * part * (k // 512 + 1), 2 * rows * part if rows == N else 0)

        fwd = terms[0] + terms[1] + most(M, N, K)
        bwd = sum(terms) + max(most(M, K, N), most(N, K, 1)) + 600 * N * 4
        assert 0 < size(C.byref(d), 0) <= fwd + 4096 and 0 < size(C.byref(d), 1) <= bwd + 4096, (M, K, N)


def test_linear_sizes_take_the_tiles_they_test(lib, ops):
    """The GPU tests of these sizes cover pairs and single CTAs, whole and split sums only while the sizes take them."""
    from linear_tiles import SIZES

    out = (C.c_int64 * 4)()
    for (M, K, N), want in SIZES.items():
        for dtype in (1, 2):
            d = ops._LinearDesc(M=M, N=N, K=K, dtype=dtype, act=1, ldx=K, ldw=K, ldr=N, ldy=N)
            for product, w in enumerate(want):
                assert lib.gs_linear_act_debug_tiles(C.byref(d), product, out) == 0
                assert (out[0], out[1] > 1) == w, ((M, K, N), product, list(out))
    assert lib.gs_linear_act_debug_tiles(C.byref(d), 3, out) == 2 and lib.gs_linear_act_debug_tiles(C.byref(d), 0, None) == 2


def test_norm_statistics_are_read_on_their_alignment(ops):
    """A hook that keeps tensors in an arena hands the saved bytes back at any address."""
    def at_odd_address(t):
        return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)

    x = torch.randn(2, 5, 32, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, at_odd_address):
        y = ops.group_norm_act(x, 4)
    torch.autograd.grad(y, x, torch.zeros_like(y))
    (_, _, args) = ops.rec.calls[-1]
    assert args[0] % 16 == 4 and args[3] % 8 == 0  # x as it came back, the statistics moved
