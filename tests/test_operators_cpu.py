"""What the head norm with rotation and the paged cache's operators refuse, and
how they trace, without a GPU: argument checks on fake CUDA tensors, and the
C ABI's own checks, which return before anything is launched."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import smooth_attn as sa
from smooth_attn import _lib


@pytest.fixture
def fake():
    with FakeTensorMode() as m:
        yield m


def _t(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", dtype=dtype)


def _targets(fn, *args):
    return [str(n.target) for n in make_fx(fn, tracing_mode="fake")(*args).graph.nodes if n.op == "call_function"]


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


# ------------------------------------------------------------------ head norm and rotation


def test_qk_norm_rope_refuses(fake):
    q, k, c = _t(2, 4, 8, 64), _t(2, 2, 8, 64), _t(8, 32, dtype=torch.float32)
    f = sa.qk_norm_rope
    with pytest.raises(AssertionError):
        f(q[0], k[0])
    with pytest.raises(AssertionError):
        f(q, _t(2, 2, 9, 64))
    with pytest.raises(ValueError, match="dtype"):
        f(q, k.float())
    with pytest.raises(ValueError, match="dtype"):
        f(q.double(), k.double())
    with pytest.raises(ValueError, match="head dim"):
        f(_t(1, 1, 1, 24), _t(1, 1, 1, 24))
    with pytest.raises(ValueError, match="head dim"):
        f(_t(1, 1, 1, 272), _t(1, 1, 1, 272))
    with pytest.raises(ValueError, match="both"):
        f(q, k, c)
    with pytest.raises(ValueError, match="tables"):
        f(q, k, c, c[:, :16])
    with pytest.raises(ValueError, match="rotate"):
        f(q, k, _t(8, 4, dtype=torch.float32), _t(8, 4, dtype=torch.float32))
    with pytest.raises(ValueError, match="rotate"):
        f(q, k, _t(8, 40, dtype=torch.float32), _t(8, 40, dtype=torch.float32))
    with pytest.raises(ValueError, match="positions for"):
        f(q, k, c[:7], c[:7])
    with pytest.raises(ValueError, match="int32"):
        f(q, k, c, c, positions=torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError, match="shape"):
        f(q, k, c, c, positions=torch.zeros(7, device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError, match="device"):
        f(q, k, c, c, positions=torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError, match="shape"):
        f(q, k, q_weight=_t(32))
    with pytest.raises(ValueError, match="CUDA"):
        f(q, k, q_weight=torch.ones(64))
    with pytest.raises(ValueError, match="eps"):
        f(q, k, eps=-1.0)
    with pytest.raises(ValueError, match="no weights"):
        f(q, k, eps=None, q_weight=_t(64))
    with pytest.raises(ValueError, match="head dim"):
        sa.sp2norm_qk_norm_rope_flash_attention(_t(1, 1, 8, 80), _t(1, 1, 8, 80), _t(1, 1, 8, 80), c, c)
    with pytest.raises(AssertionError):
        sa.sp2norm_qk_norm_rope_flash_attention(q, k, q, c, c)


def test_qk_norm_rope_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        sa.qk_norm_rope(torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 1, 64))


def test_qk_norm_rope_traces(fake):
    q, k, c = _t(2, 4, 8, 64), _t(2, 2, 8, 64), _t(8, 32, dtype=torch.float32)
    w = _t(64, dtype=torch.float32)

    def f(q, k, w):
        a, b = sa.qk_norm_rope(q, k, c, c, q_weight=w)
        # (the autograd engine itself needs a device: its op is called as the backward calls it)
        return (a, b) + torch.ops.smooth_attn_b200.qk_norm_rope_bwd(q, k, a, b, w, None, c, c, None, 1e-6, True)

    t = _targets(f, q, k, w)
    assert "smooth_attn_b200.qk_norm_rope.default" in t and "smooth_attn_b200.qk_norm_rope_bwd.default" in t
    a, b, dq, dk, gw, none = f(q, k, w)
    assert a.shape == dq.shape == q.shape and b.shape == dk.shape == k.shape and a.is_contiguous()
    assert gw.shape == (64,) and gw.dtype == torch.float32 and none.numel() == 0
    o = sa.sp2norm_qk_norm_rope_flash_attention(q, k, k, c, c, q_weight=w)
    assert o.shape == q.shape


def test_c_abi_refuses_rope_arguments_before_launch():
    lib = _lib.load()
    s = _s(64 * 4, 64, 64, 1)

    def fwd(D=64, R=0, dtype=_lib.SA_F32, p=16, strides=s, B=1, w=None, w_dtype=0, eps=1e-6, tables=None, rows=0,
            cs=0, pos=None, pos_bytes=0):
        return lib.sa_qk_norm_rope(p, p, p, p, w, None, w_dtype, tables, tables, cs, pos, pos_bytes, 0, rows,
                                   B, 1, 1, 4, D, R, strides, strides, strides, strides, eps, 1, dtype, None)

    assert fwd(D=24) == _lib.SA_ERR_UNSUPPORTED and fwd(D=272) == _lib.SA_ERR_UNSUPPORTED
    assert fwd(dtype=9) == _lib.SA_ERR_UNSUPPORTED and fwd(B=-1) == _lib.SA_ERR_ARG
    assert fwd(R=24) == _lib.SA_ERR_UNSUPPORTED and fwd(R=80) == _lib.SA_ERR_UNSUPPORTED
    assert fwd(R=64) == _lib.SA_ERR_ARG  # no tables
    assert fwd(R=64, tables=16, rows=3) == _lib.SA_ERR_ARG  # fewer rows than tokens
    assert fwd(R=64, tables=8, rows=4) == _lib.SA_ERR_ALIGN
    assert fwd(R=64, tables=16, rows=4, cs=5) == _lib.SA_ERR_UNSUPPORTED
    assert fwd(R=64, tables=16, rows=4, pos_bytes=4) == _lib.SA_ERR_ARG
    assert fwd(R=64, tables=16, rows=4, pos=16, pos_bytes=2) == _lib.SA_ERR_UNSUPPORTED
    assert fwd(eps=-1.0) == _lib.SA_ERR_ARG and fwd(eps=float("nan")) == _lib.SA_ERR_ARG
    assert fwd(w=16, w_dtype=7) == _lib.SA_ERR_UNSUPPORTED and fwd(w=8) == _lib.SA_ERR_ALIGN
    assert fwd(p=None) == _lib.SA_ERR_ARG and fwd(p=8) == _lib.SA_ERR_ALIGN
    assert fwd(strides=_s(256, 64, 66, 1)) == _lib.SA_ERR_ALIGN
    assert fwd(strides=_s(256, 64, 64, 2)) == _lib.SA_ERR_ALIGN
    assert fwd(B=0, p=None) == _lib.SA_OK  # nothing to do
    assert lib.sa_qk_norm_rope_bwd_workspace_size(128) > 0
    assert lib.sa_qk_norm_rope_bwd_workspace_size(512) == _lib.SA_ERR_UNSUPPORTED

    def bwd(dw=None, w=None, norm=1, ws=16, nbytes=1 << 30):
        return lib.sa_qk_norm_rope_bwd(16, 16, 16, 16, 16, 16, w, None, 0, dw, None, None, None, 0, None, 0, 0, 0,
                                       ws, nbytes, 1, 1, 1, 4, 64, 0, s, s, s, s, s, _s(1, 1, 1, 2), 1e-6, norm,
                                       0, None)

    assert bwd(dw=16) == _lib.SA_ERR_ARG  # a gradient without its weight
    assert bwd(dw=16, w=16, norm=0) == _lib.SA_ERR_ARG
    assert bwd(dw=16, w=16, ws=None) == _lib.SA_ERR_ARG and bwd(dw=16, w=16, nbytes=8) == _lib.SA_ERR_ARG
    assert bwd() == _lib.SA_ERR_ALIGN  # dk's channel stride
