"""Layer operators without a GPU: argument checks, the C ABI's refusals and workspace queries, and the
definitions the GPU tests use against torch's own layers."""

import ctypes as C

import pytest
import torch
import torch.nn.functional as F


@pytest.fixture(scope="module")
def ops(lib):
    from gaussian_2d_splat_encoder_b200 import layers

    return layers


def norm_desc(ops, **kw):
    d = dict(B=2, C=64, groups=8, dtype=1, param_dtype=0, act=1, act_first=1, eps=1e-5, rows=100, x_row=64, x_img=6400,
             dy_row=64, dy_img=6400)
    d.update(kw)
    return ops._NormDesc(**d)


def linear_desc(ops, **kw):
    d = dict(M=100, N=32, K=64, dtype=1, act=1, ldx=64, ldw=64, ldr=32, ldy=32)
    d.update(kw)
    return ops._LinearDesc(**d)


def test_no_cpu_fallback(ops):
    x = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.group_norm_act(x, 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.linear_act(x, torch.zeros(4, 8))


def test_norm_workspace_and_refusals(lib, ops):
    size = lib.gs_group_norm_act_workspace_size
    assert 0 < size(C.byref(norm_desc(ops)), 0) < size(C.byref(norm_desc(ops)), 1) < 1 << 24
    for bad in (dict(B=-1), dict(C=0), dict(groups=0), dict(groups=7), dict(dtype=3), dict(param_dtype=2), dict(act=3),
                dict(act=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(rows=-1), dict(C=2056), dict(rows=(1 << 30) + 1)):
        d = norm_desc(ops, **bad)
        assert size(C.byref(d), 0) == 0, bad
        assert lib.gs_group_norm_act_fwd(C.byref(d), *[None] * 6, 0, None) == 2, bad
        assert lib.gs_group_norm_act_bwd(C.byref(d), *[None] * 9, 0, None) == 2, bad
    d = norm_desc(ops)
    assert lib.gs_group_norm_act_fwd(C.byref(d), *[None] * 6, 0, None) == 2
    assert lib.gs_group_norm_act_bwd(C.byref(d), *[None] * 9, 0, None) == 2
    p = C.c_void_p(256)  # never read: the workspace is refused first
    assert lib.gs_group_norm_act_fwd(C.byref(d), p, None, None, p, None, p, 16, None) == 5
    assert lib.gs_group_norm_act_bwd(C.byref(d), p, None, None, p, p, p, None, None, p, 16, None) == 5
    assert lib.gs_group_norm_act_fwd(C.byref(norm_desc(ops, rows=0)), *[None] * 6, 0, None) == 0


def test_linear_workspace_and_refusals(lib, ops):
    size = lib.gs_linear_act_workspace_size
    assert 0 < size(C.byref(linear_desc(ops)), 0) <= size(C.byref(linear_desc(ops)), 1)
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(dtype=3), dict(dtype=-1), dict(act=3), dict(N=(1 << 20) + 1)):
        d = linear_desc(ops, **bad)
        assert size(C.byref(d), 0) == 0, bad
        assert lib.gs_linear_act_fwd(C.byref(d), *[None] * 7, 0, None) == 2, bad
        assert lib.gs_linear_act_bwd(C.byref(d), *[None] * 8, 0, None) == 2, bad
    p = C.c_void_p(256)
    for bad in (dict(ldx=63), dict(ldw=63), dict(ldr=31), dict(unaligned=8), dict(M=(1 << 30) + 1), dict(ldx=1 << 37)):
        d = linear_desc(ops, **bad)
        assert lib.gs_linear_act_fwd(C.byref(d), p, p, None, p, p, None, p, 1 << 30, None) == 2, bad
    assert lib.gs_linear_act_bwd(C.byref(linear_desc(ops, ldy=31)), p, p, p, p, p, p, p, p, 1 << 30, None) == 2
    d = linear_desc(ops)
    need = linear_desc(ops, K=63, ldx=63)  # x is kept padded
    assert size(C.byref(d), 0) == 256 < size(C.byref(need), 0)
    assert lib.gs_linear_act_fwd(C.byref(need), p, p, None, None, p, None, p, 16, None) == 5
    assert lib.gs_linear_act_fwd(C.byref(need), p, p, None, None, p, None, None, 1 << 30, None) == 5
    assert lib.gs_linear_act_bwd(C.byref(d), p, p, p, p, p, p, p, p, 16, None) == 5
    q = C.c_void_p(264)  # off 16 bytes, without the descriptor's bit
    assert lib.gs_linear_act_fwd(C.byref(d), q, p, None, None, p, None, p, 1 << 40, None) == 2
    assert lib.gs_linear_act_fwd(C.byref(d), p, q, None, None, p, None, p, 1 << 40, None) == 2
    assert lib.gs_linear_act_bwd(C.byref(d), p, p, p, q, p, p, p, p, 1 << 40, None) == 2
    # the backward of an activation needs the kept slope
    assert lib.gs_linear_act_bwd(C.byref(d), p, p, None, p, p, p, p, p, 1 << 40, None) == 2
    assert size(C.byref(linear_desc(ops, M=0)), 0) > 0 and size(C.byref(linear_desc(ops, M=0)), 1) > 0
    assert lib.gs_linear_act_fwd(C.byref(linear_desc(ops, M=0)), *[None] * 7, 0, None) == 0


def test_row_strides(ops):
    t = torch.zeros(4, 5, 6, 32)
    assert ops._rows_of(t, 1) == 32 and ops._rows_of(t[..., :8], 0) == 32
    assert ops._rows_of(t[:, ::2, :, :8], 1) is None and ops._rows_of(t[:, :, ::2, :8], 1) == 64
    assert ops._rows_of(t.transpose(1, 2), 1) is None
    assert ops._rows_of(t[:, :1, 2:3], 1) == 32
    assert ops._image_layout(t[:1, :, :, 4:12])[1:] == (32, 0)
    assert ops._row_layout(t[:, :, :, :8].expand(4, 5, 6, 8))[1] == 32
    assert ops._row_layout(torch.zeros(1, 8).expand(9, 8))[0].is_contiguous()


@pytest.mark.parametrize("act,first", [("none", False), ("gelu", True), ("silu", False)])
def test_definition_is_torchs(act, first):
    from layers_util import ACTS, norm_ref

    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 5, 7, 24, generator=g, dtype=torch.float64)
    w, b = torch.randn(24, generator=g, dtype=torch.float64), torch.randn(24, generator=g, dtype=torch.float64)
    u = ACTS[act](x) if first else x
    ref = F.group_norm(u.permute(0, 3, 1, 2), 4, w, b, 1e-5).permute(0, 2, 3, 1)
    ref = ref if first else ACTS[act](ref)
    assert torch.allclose(norm_ref(x, 4, w, b, 1e-5, act, first)[0], ref, rtol=1e-12, atol=1e-12)
