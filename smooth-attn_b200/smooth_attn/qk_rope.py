"""Head norms of queries and keys with the position rotation in one pass, with
its backward, and the attention that trains through it.

The reference rotates inside a forward-only attention kernel and has no head
norm (``src/smooth_attn/kernels.py:2104-2430``); here both are one operator
(``sa_qk_norm_rope``) in front of ``sp2norm_flash_attention``, so a model with
rotated (and normalised) queries and keys trains on the fused path.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import kernels as K

QK_MAX_HEAD_DIM = 256  # the rows are split over at most 16 lanes of 16 channels
_POS_BYTES = {torch.int32: 4, torch.int64: 8}


def _check_weight(w, name, D, like):
    if w is None:
        return
    K._validate_cuda_tensor(w, name=name)
    if w.shape != (D,):
        raise ValueError(f"{name} must have shape ({D},), got {tuple(w.shape)}")
    if w.device != like.device:
        raise ValueError(f"{name} and the rows must live on the same CUDA device")


def _check_tables(cos, sin, D, like):
    """cos / sin: [positions, R/2] tables, both or neither; R a multiple of 16, at most D."""
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together: pass both or neither")
    if cos is None:
        return 0, 0
    if cos.ndim != 2 or cos.shape != sin.shape:
        raise ValueError(f"cos and sin must be two [positions, R/2] tables, got {tuple(cos.shape)}/{tuple(sin.shape)}")
    if not cos.is_cuda or cos.device != like.device or sin.device != like.device:
        raise ValueError("cos, sin and the rows must live on the same CUDA device")
    R = 2 * cos.shape[1]
    if R == 0 or R % 16 or R > D:
        raise ValueError(f"the tables rotate {R} channels: a multiple of 16, 16 to the head dim {D}, is supported")
    return R, cos.shape[0]


def _check_positions(positions, shapes, like):
    if positions is None:
        return
    if not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be a torch.Tensor")
    if positions.dtype not in _POS_BYTES:
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if tuple(positions.shape) not in shapes:
        raise ValueError(f"positions must have a shape of {shapes}, got {tuple(positions.shape)}")
    if positions.device != like.device:
        raise ValueError("positions and the rows must live on the same CUDA device")


def _check_norm(eps, q_weight, k_weight):
    if eps is None:
        if q_weight is not None or k_weight is not None:
            raise ValueError("eps=None leaves the norm out: it takes no weights")
    elif not eps >= 0:
        raise ValueError(f"eps must be at least 0 (or None for no norm), got {eps}")


def _copied(t):
    return torch.empty(t.shape, device=t.device, dtype=t.dtype).copy_(t)


def _dense(t):
    """t contiguous on a 16-byte boundary (a contiguous view may start off one)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else _copied(t)


def _strides(t):
    """t's strides as the C ABI takes them; a dim of one element has none (torch leaves any number there)."""
    return (ctypes.c_int64 * t.ndim)(*(s if n > 1 else 0 for n, s in zip(t.shape[:-1], t.stride())), 1)


def _rows(t):
    """t with rows that 16-byte loads can take: unit channel stride, base and other strides multiples of 16 bytes."""
    es = t.element_size()
    ok = (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
          and all(n <= 1 or (s * es) % 16 == 0 for n, s in zip(t.shape[:-1], t.stride())))
    return t if ok else _copied(t)


def _weights(q_weight, k_weight):
    """Both weights dense and of one type (the C ABI takes one): fp32 where they differ."""
    wq, wk = (None if w is None else _dense(w) for w in (q_weight, k_weight))
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        wq, wk = wq.float(), wk.float()
    some = wq if wq is not None else wk
    return wq, wk, K._DTYPE_CODE[some.dtype] if some is not None else _lib.SA_F32


def _tables(cos, sin):
    if cos is None:
        return None, None, _lib.SA_F32
    if cos.dtype not in K._DTYPE_CODE or sin.dtype != cos.dtype:
        cos, sin = cos.float(), sin.float()
    return _dense(cos), _dense(sin), K._DTYPE_CODE[cos.dtype]


def _positions(positions, T):
    """(tensor, bytes of an entry, stride between batches)."""
    if positions is None:
        return None, 0, 0
    positions = positions.contiguous()
    return positions, _POS_BYTES[positions.dtype], T if positions.ndim == 2 and positions.shape[0] > 1 else 0


def _check_qk(q, k, cos, sin, q_weight, k_weight, eps, positions):
    assert q.ndim == 4 and k.ndim == 4
    B, _, T, D = q.shape
    assert k.shape[0] == B and k.shape[2] == T and k.shape[3] == D, "q and k differ in more than their heads"
    for name, t in (("q", q), ("k", k)):
        K._validate_cuda_tensor(t, name=name)
    if k.dtype != q.dtype or k.device != q.device:
        raise ValueError(f"q and k must share one dtype and device, got {q.dtype}/{k.dtype}, {q.device}/{k.device}")
    if D % 16 or not 16 <= D <= QK_MAX_HEAD_DIM:
        raise ValueError(f"head dim {D} not supported (a multiple of 16, 16 to {QK_MAX_HEAD_DIM})")
    _check_norm(eps, q_weight, k_weight)
    _check_weight(q_weight, "q_weight", D, q)
    _check_weight(k_weight, "k_weight", D, q)
    R, rows = _check_tables(cos, sin, D, q)
    _check_positions(positions, ((T,), (1, T), (B, T)), q)
    if R and positions is None and rows < T:
        raise ValueError(f"the tables have {rows} positions for {T} tokens")


def _fwd_direct(q, k, q_weight, k_weight, cos, sin, positions, eps):
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    q_out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    k_out = torch.empty(k.shape, device=k.device, dtype=k.dtype)
    if q.numel() + k.numel() == 0:
        return q_out, k_out
    q, k = _rows(q), _rows(k)
    wq, wk, w_code = _weights(q_weight, k_weight)
    cos, sin, cs_code = _tables(cos, sin)
    pos, pos_bytes, pos_sb = _positions(positions, T)
    with K._on(q.device):
        st = _lib.load().sa_qk_norm_rope(
            q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), K._ptr(wq), K._ptr(wk), w_code,
            K._ptr(cos), K._ptr(sin), cs_code, K._ptr(pos), pos_bytes, pos_sb, 0 if cos is None else cos.shape[0],
            B, Hq, Hkv, T, D, 0 if cos is None else 2 * cos.shape[1], _strides(q), _strides(k),
            _strides(q_out), _strides(k_out), 0.0 if eps is None else float(eps), int(eps is not None),
            K._DTYPE_CODE[q.dtype], K._stream(q))
    _lib.check(st, "sa_qk_norm_rope")
    return q_out, k_out


def _bwd_direct(q, k, dq_out, dk_out, q_weight, k_weight, cos, sin, positions, eps, need_dw):
    """(dq, dk, dq_weight, dk_weight); the last two None without a weight or when not needed."""
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    dk = torch.empty(k.shape, device=k.device, dtype=k.dtype)
    q, k, dq_out, dk_out = (_rows(t) for t in (q, k, dq_out, dk_out))
    wq, wk, w_code = _weights(q_weight, k_weight)
    cos, sin, cs_code = _tables(cos, sin)
    pos, pos_bytes, pos_sb = _positions(positions, T)
    dwq = torch.empty_like(wq) if need_dw and wq is not None else None
    dwk = torch.empty_like(wk) if need_dw and wk is not None else None
    lib = _lib.load()
    with K._on(q.device):
        nbytes, ws = 0, None
        if dwq is not None or dwk is not None:
            nbytes = int(lib.sa_qk_norm_rope_bwd_workspace_size(D))
            ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
        st = lib.sa_qk_norm_rope_bwd(
            K._ptr(q), K._ptr(k), K._ptr(dq_out), K._ptr(dk_out), K._ptr(dq), K._ptr(dk), K._ptr(wq), K._ptr(wk),
            w_code, K._ptr(dwq), K._ptr(dwk), K._ptr(cos), K._ptr(sin), cs_code, K._ptr(pos), pos_bytes, pos_sb,
            0 if cos is None else cos.shape[0], K._ptr(ws), nbytes, B, Hq, Hkv, T, D,
            0 if cos is None else 2 * cos.shape[1], _strides(q), _strides(k), _strides(dq_out),
            _strides(dk_out), _strides(dq), _strides(dk), 0.0 if eps is None else float(eps),
            int(eps is not None), K._DTYPE_CODE[q.dtype], K._stream(q))
    _lib.check(st, "sa_qk_norm_rope_bwd")
    if dwq is not None and dwq.dtype != q_weight.dtype:
        dwq = dwq.to(q_weight.dtype)
    if dwk is not None and dwk.dtype != k_weight.dtype:
        dwk = dwk.to(k_weight.dtype)
    return dq, dk, dwq, dwk


def _fwd(q, k, q_weight, k_weight, cos, sin, positions, eps):
    if K._tracing(q, k):
        return K._ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)
    return _fwd_direct(q, k, q_weight, k_weight, cos, sin, positions, eps)


class _QkNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps = eps
        return _fwd(q, k, q_weight, k_weight, cos, sin, positions, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        need_dw = any(ctx.needs_input_grad[2:4])
        if K._tracing(q, k, dq_out, dk_out):
            dq, dk, dwq, dwk = K._ops().qk_norm_rope_bwd(q, k, dq_out, dk_out, wq, wk, cos, sin, positions, ctx.eps,
                                                         need_dw)
        else:
            dq, dk, dwq, dwk = _bwd_direct(q, k, dq_out, dk_out, wq, wk, cos, sin, positions, ctx.eps, need_dw)
        need = ctx.needs_input_grad
        return (dq, dk, dwq if need[2] else None, dwk if need[3] else None, None, None, None, None)


def qk_norm_rope(q, k, cos=None, sin=None, *, q_weight=None, k_weight=None, eps=1e-6, positions=None):
    """Root-mean-square norm of every query and key head, then the rotation of
    its position, in one pass; returns (q, k), contiguous, in q's dtype.

    q: [B, H_q, T, D], k: [B, H_kv, T, D], fp32, fp16 or bf16, any strides, D a
    multiple of 16 up to 256.  Per head row x, in fp32 with one rounding at the end::

        n = x / sqrt(mean(x^2) + eps) * weight
        y = n with its first R channels rotated (rotate-half form, as ``sp2norm_rope_flash_attention``)

    cos / sin: [positions, R/2] tables (``precompute_rope_cos_sin(R, ...)``), R a multiple of
    16 up to D; None leaves the rotation out.  positions: int32 or int64 [T] or [B, T], the
    table row of each token (None: 0 .. T-1).  A position outside the tables is read as 0 and
    reported by ``sa_device_status``.  q_weight / k_weight: [D], None for 1.  eps=None leaves
    the norm out.  Differentiable once in q, k and the weights; the gradients of the weights are
    summed in fp32 in a fixed order, bitwise the same from run to run.  No gradient for cos / sin.
    """
    _check_qk(q, k, cos, sin, q_weight, k_weight, eps, positions)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRopeFn.apply(q, k, q_weight, k_weight, cos, sin, positions, eps)
    return _fwd(q, k, q_weight, k_weight, cos, sin, positions, eps)


def sp2norm_qk_norm_rope_flash_attention(q, k, v, cos, sin, *, q_weight=None, k_weight=None, eps=1e-6,
                                         positions=None, scale=None, window_size=0, exact_math=False,
                                         deterministic=None):
    """``sp2norm_flash_attention`` on normalised and rotated queries and keys, with autograd.

    q, k, cos, sin, q_weight, k_weight, eps, positions as ``qk_norm_rope`` (eps=None: the rotation
    alone, the trainable form of ``sp2norm_rope_flash_attention``); v and the rest as
    ``sp2norm_flash_attention``.  Causality goes by the order along T, not by positions.
    """
    assert q.ndim == 4 and k.ndim == 4 and v.ndim == 4
    B, H_q, T, D = q.shape
    H_kv = k.shape[1]
    assert k.shape == (B, H_kv, T, D) and v.shape == (B, H_kv, T, D)
    assert H_q % H_kv == 0, f"H_q ({H_q}) must be divisible by H_kv ({H_kv})"
    K._flash_check(q, k, v)
    q, k = qk_norm_rope(q, k, cos, sin, q_weight=q_weight, k_weight=k_weight, eps=eps, positions=positions)
    return K.sp2norm_flash_attention(q, k, v, scale=1.0 / math.sqrt(D) if scale is None else scale,
                                     window_size=window_size, exact_math=exact_math, deterministic=deterministic)
