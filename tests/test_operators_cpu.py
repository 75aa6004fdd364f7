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


# ------------------------------------------------------------------ paged cache


def _i(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def test_paged_slots_refuse(fake):
    f = sa.paged_assign_slots
    t, n, p, h = _i(3, 4), _i(3), _i(9), _i(1)
    for bad in (_i(3), _i(3, 4, dtype=torch.int64), _i(4, 3).T, _i(3, 0), torch.zeros(3, 4, dtype=torch.int32)):
        with pytest.raises(ValueError):
            f(bad, n, n, p, h, 3)
    with pytest.raises(TypeError):
        f([[1]], n, n, p, h, 3)
    with pytest.raises(TypeError):
        f(t, [1, 2, 3], n, p, h, 3)
    for ctx, new, pool, head, N in ((_i(2), n, p, h, 3), (n, _i(4), p, h, 3), (n, n, _i(3, 3), h, 3),
                                    (n, n, p, _i(2), 3), (n, n, p, h, -1), (n, n, p, h, 2 ** 31),
                                    (n, _i(3, dtype=torch.float32), p, h, 3), (n.cpu(), n, p, h, 3)):
        with pytest.raises(ValueError):
            f(t, ctx, new, pool, head, N)
    with pytest.raises(ValueError, match="block_size"):
        f(t, n, n, p, h, 3, block_size=0)
    with pytest.raises(ValueError, match="16384"):
        f(_i(16385, 2), _i(16385), _i(16385), p, h, 3)
    r, d = sa.paged_release_pages, torch.zeros(3, dtype=torch.bool, device="cuda")
    for done, pool in ((n, p), (d[:2], p), (d, _i(9, dtype=torch.int64)), (d, _i(18)[::2]), (d, _i(3, 3)),
                       (d.cpu(), p)):
        with pytest.raises(ValueError):
            r(t, n, done, pool, h)
    s = f(t, n, n, p, h, 7)
    assert [tuple(x.shape) for x in s] == [(7,), (7,), (4,), (3,), (1,)] and s.slot_mapping.dtype == torch.int64
    ctx, head = r(t, n, d, p, h)
    assert ctx.shape == (3,) and head.shape == (1,)


def test_paged_append_refuses(fake):
    f = sa.qk_norm_rope_paged_append
    q, k, c = _t(5, 4, 64), _t(5, 2, 64), _t(6, 2, 16, 64)
    s, cs, pos = _i(5, dtype=torch.int64), _t(9, 32, dtype=torch.float32), _i(5)
    with pytest.raises(AssertionError):
        f(q, k, _t(5, 3, 64), c, c, s)
    with pytest.raises(AssertionError):
        f(q[:4], k, k, c, c, s)
    for args in ((q.float(), k.float(), k.float(), c, c, s), (q, k.half(), k, c, c, s), (q, k, k, c.half(), c.half(), s),
                 (q, k, k, c, c[:5], s), (q, k, k, _t(6, 3, 16, 64), _t(6, 3, 16, 64), s),
                 (q, k, k, c.transpose(1, 2), c, s), (q, k, k, c[0], c[0], s), (q, k, k, c, c, s.int()),
                 (q, k, k, c, c, s[:4]), (q, k, k, c, c, s.cpu()), (q, k, k, c, c, s, cs, cs)):
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(ValueError):
        f(q, k, k, c, c, s, cs, cs, positions=_i(4))
    with pytest.raises(ValueError, match="backward"):
        f(q.clone().requires_grad_(True), k, k, c, c, s)
    with pytest.raises(ValueError, match="CUDA"):
        f(*(torch.zeros(1, 1, 64, dtype=torch.bfloat16),) * 3, c, c, s)
    assert f(q, k, k, c, c, s, cs, cs, positions=pos).shape == q.shape


def test_page_choice_refuses(fake):
    q, m, c, bt, cl = _t(2, 4, 1, 64), _t(6, 2, 64), _t(6, 2, 16, 64), _i(2, 3), _i(2)
    f = sa.sp2norm_sparse_paged_attention
    with pytest.raises(AssertionError):
        f(q[:, :, 0], c, c, m, bt, cl, 2)
    with pytest.raises(AssertionError):
        f(_t(2, 3, 1, 64), c, c, m, bt, cl, 2)
    for args in ((q.float(), c, c, m, bt, cl, 2), (q, c, c, m, bt, cl, 0), (q, c, c, m.half(), bt, cl, 2),
                 (q, c, c[:5], m, bt, cl, 2), (q, c, c, _t(6, 2, 32), bt, cl, 2), (q, c, c, m[:, 0], bt, cl, 2),
                 (q, c, c, m, bt[:1], cl, 2), (q, c, c, m, bt, cl[:1], 2), (q, c, c, m, bt[0], cl, 2),
                 (q, c.transpose(1, 2), c, m, bt, cl, 2), (q, c, c, m, bt.cpu(), cl, 2),
                 (_t(2, 4, 1, 96), c, c, m, bt, cl, 2)):
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(ValueError, match="block_size"):
        f(q, c, c, m, bt, cl, 2, block_size=8)
    out, pages = f(q, c, c, m, bt, cl, 9, return_pages=True)
    assert out.shape == (2, 4, 64) and pages.shape == (2, 2, 3)
    assert sa.sp2norm_paged_select(q, m, bt, cl, 2)[0].shape == (2, 2, 2)
    g = sa.paged_key_means
    for args in ((m, c.float(), bt, cl), (m[:5], c, bt, cl), (m.half(), c, bt, cl), (m, c[0], bt, cl),
                 (m, c, bt[0], cl), (m, c, bt, cl[:1]), (m, c.transpose(1, 2), bt, cl)):
        with pytest.raises(ValueError):
            g(*args)
    with pytest.raises(ValueError):
        g(m, c, bt, cl, start_lens=_i(3))
    assert g(m, c, bt, cl, start_lens=cl) is m


def test_paged_operators_trace(fake):
    q, k, c, m = _t(2, 4, 64), _t(2, 2, 64), _t(6, 2, 16, 64), _t(6, 2, 64)
    bt, cl, p, h, d = _i(2, 3), _i(2), _i(9), _i(1), torch.zeros(2, dtype=torch.bool, device="cuda")

    def f(q, k, c, v, m, bt, cl, p, h, d):
        cl, h = sa.paged_release_pages(bt, cl, d, p, h)
        s = sa.paged_assign_slots(bt, cl, torch.ones_like(cl), p, h, 2)
        q = sa.qk_norm_rope_paged_append(q, k, k, c, v, s.slot_mapping)
        sa.paged_key_means(m, c, bt, s.context_lens, start_lens=cl)
        pages, _ = sa.sp2norm_paged_select(q[:, :, None], m, bt, s.context_lens, 2)
        return sa.sp2norm_sparse_paged_attention(q[:, :, None], c, v, m, bt, s.context_lens, 2), pages

    t = _targets(f, q, k, c, c.clone(), m, bt, cl, p, h, d)
    for op in ("paged_release_pages", "paged_assign_slots", "qk_norm_rope_paged_append", "paged_key_means",
               "paged_select", "sparse_paged_decode"):
        assert t.count(f"smooth_attn_b200.{op}.default") == 1, op


def test_c_abi_refuses_paged_arguments_before_launch():
    lib = _lib.load()
    A, U, L, OK = _lib.SA_ERR_ARG, _lib.SA_ERR_UNSUPPORTED, _lib.SA_ERR_ALIGN, _lib.SA_OK

    def assign(B=2, N=2, mb=4, bs=16, ld=4, free=8, p=16, head=16):
        return lib.sa_paged_assign_slots(p, ld, p, p, p, free, head, p, p, p, p, p, B, N, mb, bs, None)

    assert assign(B=-1) == A and assign(mb=0) == A and assign(bs=0) == A and assign(ld=3) == A and assign(free=-1) == A
    assert assign(B=16385) == U and assign(bs=1 << 17) == U and assign(mb=1 << 28, ld=1 << 28) == U
    assert assign(N=-1) == A and assign(N=2 ** 31) == U and assign(p=None) == A and assign(head=None) == A
    rel = lambda B=2, mb=4, ld=4, p=16, head=16: lib.sa_paged_release_pages(  # noqa: E731
        p, ld, p, p, p, 8, head, p, p, B, mb, 16, None)
    assert rel(B=-1) == A and rel(ld=3) == A and rel(B=16385) == U and rel(p=None) == A and rel(head=None) == A
    s3 = _s(128, 64, 1)

    def append(N=2, Hq=2, Hkv=2, D=64, dtype=_lib.SA_BF16, p=16, s=s3, bs=16, slots=16, nb=3):
        return lib.sa_qk_norm_rope_paged_append(p, p, p, p, p, p, slots, None, None, 0, None, None, 0, None, 0, 0, N, Hq,
                                                Hkv, D, 0, nb, bs, s, s, s, 1e-6, 1, dtype, None)

    assert append(N=-1) == A and append(Hkv=0) == A and append(bs=0) == A and append(nb=-1) == A
    assert append(dtype=_lib.SA_F32) == U and append(D=24) == U and append(p=None) == A and append(slots=None) == A
    assert append(p=8) == L and append(s=_s(128, 60, 1)) == L and append(s=_s(128, 64, 2)) == L
    assert append(N=0, p=None) == OK

    def means(B=1, Hkv=2, nb=3, bs=16, mb=4, D=64, dtype=_lib.SA_BF16, p=16):
        return lib.sa_paged_key_means(p, p, p, p, None, B, Hkv, nb, bs, mb, D, dtype, None)

    assert means(B=-1) == A and means(nb=0) == A and means(mb=0) == A and means(p=None) == A and means(p=8) == L
    assert means(D=48) == U and means(dtype=0) == U and means(B=65535) == U and means(nb=2 ** 31) == U
    assert means(B=0, p=None) == OK

    def sparse(B=1, Hq=4, Hkv=2, nb=3, bs=16, mb=4, K=2, D=64, scale=0.1, dtype=_lib.SA_BF16, p=16, ws=256,
               nbytes=1 << 30):
        a = lib.sa_paged_select(p, p, p, p, p, p, ws, nbytes, B, Hq, Hkv, nb, bs, mb, K, D, scale, dtype, None)
        b = lib.sa_sparse_paged_decode(p, p, p, p, p, p, p, None, ws, nbytes, B, Hq, Hkv, nb, bs, mb, K, D, scale, dtype,
                                       None)
        assert a == b
        return a

    assert sparse(K=0) == A and sparse(K=5) == A and sparse(Hq=3) == A and sparse(Hq=0) == A
    assert sparse(scale=float("nan")) == A and sparse(D=48) == U and sparse(dtype=0) == U and sparse(B=65536) == U
    assert sparse(p=None) == A and sparse(ws=None) == A and sparse(nbytes=16) == A and sparse(p=8) == L
    assert sparse(ws=128) == L and sparse(B=0, p=None) == OK
    assert lib.sa_paged_select_workspace_size(2, 8, 512) == 2 * 8 * 512 * 8
    assert lib.sa_paged_select_workspace_size(65536, 1, 1) == U
    assert lib.sa_sparse_paged_decode_workspace_size(2, 32, 8, 512, 64, 16, 128, _lib.SA_BF16) > 2 * 8 * 512 * 8
    assert lib.sa_sparse_paged_decode_workspace_size(2, 32, 8, 512, 0, 16, 128, _lib.SA_BF16) == A


def test_forward_mode_derivatives_are_refused(fake):
    q, k, c, w = _t(5, 4, 64), _t(5, 2, 64), _t(6, 2, 16, 64), _t(64)
    s = _i(5, dtype=torch.int64)
    fw = torch.autograd.forward_ad
    with fw.dual_level(), torch.no_grad():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        f = sa.qk_norm_rope_paged_append
        for args, kw in (((dual(q), k, k), {}), ((q, dual(k), k), {}), ((q, k, dual(k)), {}),
                         ((q, k, k), dict(q_weight=dual(w))), ((q, k, k), dict(k_weight=dual(w)))):
            with pytest.raises(ValueError, match="derivative"):
                f(*args, c, c, s, **kw)
        assert f(q, k, k, c, c, s, q_weight=w).shape == q.shape
        x = q[None].transpose(1, 2)
        with pytest.raises(NotImplementedError, match="jvp"):
            sa.qk_norm_rope(dual(x), k[None].transpose(1, 2))
        assert sa.qk_norm_rope(x, k[None].transpose(1, 2))[0].shape == x.shape


def test_c_abi_refuses_narrowing_arguments_before_launch():
    lib = _lib.load()
    for args in ((16, 16, -1), (None, 16, 1), (16, None, 1)):
        assert lib.sa_narrow_i64(*args, None) == _lib.SA_ERR_ARG
    assert lib.sa_narrow_i64(None, None, 0, None) == _lib.SA_OK
