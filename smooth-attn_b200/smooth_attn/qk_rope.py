"""Head norms of queries and keys with the position rotation in one pass, with
its backward, and the attention that trains through it.

The reference rotates inside a forward-only attention kernel and has no head
norm (``src/smooth_attn/kernels.py:2104-2430``); here both are one operator
(``sa_qk_norm_rope``) in front of ``sp2norm_flash_attention``, so a model with
rotated (and normalised) queries and keys trains on the fused path.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad as _fwd_ad
from torch.autograd.function import once_differentiable

from . import _lib
from . import kernels as K

QK_MAX_HEAD_DIM = 256  # the rows are split over at most 16 lanes of 16 channels
_POS_BYTES = {torch.int32: 4, torch.int64: 8}


def _traced(t):
    """Whether a call runs under a tracer (``K._tracing`` of its first tensor, without a generator per call)."""
    return (torch.compiler.is_compiling() or K._get_proxy_mode() is not None or isinstance(t, K._TRACED_TYPES))


def _has_tangent(*tensors):
    """Whether one of them carries a forward-mode derivative, which no kernel here computes."""
    return _fwd_ad._current_level >= 0 and any(t is not None and _fwd_ad.unpack_dual(t).tangent is not None
                                               for t in tensors)


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


def _like(t):
    """An empty tensor in t's own order of dims where the rows can be written so, else contiguous."""
    o = torch.empty_like(t)
    return o if _stride_ok(o) else torch.empty(t.shape, device=t.device, dtype=t.dtype)


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


# ---- plans --------------------------------------------------------------------
#
# A decode step's rows are few: the host's time per call, not the kernel's,
# paces it.  All checks and every argument but the pointers follow from the
# tensors' types, shapes and strides, so they are worked out once per such
# signature and kept as a plan (never by a tensor's address or contents).  A
# call that needs a copy or a conversion has no plan and takes the checked path.
# The arguments are kept as ctypes objects: 28 of them cost a call a quarter less
# than Python numbers.
# (Eight new tokens through the API: 45 us without plans, 19 us with them, on a
# host whose torch.empty costs 3.5 us and a bare kernel launch 4.)

_PLANS: dict = {}
_MAX_PLANS = 1024


def _sig(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _keep(plans, key, plan):
    if len(plans) >= _MAX_PLANS:
        plans.clear()
    plans[key] = plan
    return plan


def _stride_ok(t):
    es = t.element_size()
    return t.stride(-1) == 1 and all(n <= 1 or (s * es) % 16 == 0 for n, s in zip(t.shape[:-1], t.stride()))


def _plain(cos, sin, q_weight, k_weight, positions):
    """Tables, weights and positions as the C ABI takes them, without a copy (alignment aside)."""
    tables = cos is None or (cos.dtype in K._DTYPE_CODE and sin.dtype == cos.dtype and cos.is_contiguous()
                             and sin.is_contiguous())
    ws = [w for w in (q_weight, k_weight) if w is not None]
    weights = all(w.is_contiguous() and w.dtype == ws[0].dtype for w in ws)
    return tables and weights and (positions is None or positions.is_contiguous())


def _row_args(cos, sin, q_weight, k_weight, positions, T):
    """(weight code, table code, position bytes, position stride, table rows) of _plain arguments."""
    some = q_weight if q_weight is not None else k_weight
    pos_sb = T if positions is not None and positions.ndim == 2 and positions.shape[0] > 1 else 0
    return (K._DTYPE_CODE[some.dtype] if some is not None else _lib.SA_F32,
            K._DTYPE_CODE[cos.dtype] if cos is not None else _lib.SA_F32,
            0 if positions is None else _POS_BYTES[positions.dtype], pos_sb, 0 if cos is None else cos.shape[0])


def _key_of(q, k, cos, sin, q_weight, k_weight, eps, positions):
    return (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), _sig(cos),
            _sig(sin), _sig(q_weight), _sig(k_weight), eps, _sig(positions))


def _held(function, at, *values):
    """A C function's arguments from number ``at`` on as ctypes objects: converted once, not at every call."""
    return tuple(t(v) if isinstance(v, (int, float)) else v
                 for t, v in zip(_lib.SIGNATURES[function][1][at:], values))


class _Plan:
    """qk_norm_rope of one signature."""

    def __init__(self, key, q, k, cos, sin, q_weight, k_weight, eps, positions):
        self.key = key
        B, Hq, T, D = q.shape
        w, cs, *table = _row_args(cos, sin, q_weight, k_weight, positions, T)
        out = tuple(_strides(torch.empty_like(t)) for t in (q, k))
        dims = (B, Hq, k.shape[1], T, D, 0 if cos is None else 2 * cos.shape[1])
        ins = (_strides(q), _strides(k))
        flags = (0.0 if eps is None else float(eps), int(eps is not None), K._DTYPE_CODE[q.dtype])
        (self.w,) = _held("sa_qk_norm_rope", 6, w)
        (self.cs,) = _held("sa_qk_norm_rope", 9, cs)
        self.fwd = _held("sa_qk_norm_rope", 11, *table, *dims, *ins, *out, *flags)
        self.table = _held("sa_qk_norm_rope_bwd", 15, *table)
        self.ins = _held("sa_qk_norm_rope_bwd", 20, *dims, *ins)
        self.out = _held("sa_qk_norm_rope_bwd", 30, *out, *flags)
        self.device, self.D = q.get_device(), D
        self.bwd = {}  # by the strides of the two incoming gradients: theirs as the C ABI takes them
        self.ws_bytes = None

    def run(self, q, k, cos, sin, q_weight, k_weight, positions):
        """(q_out, k_out), or None where a base is off a 16-byte boundary."""
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        st = _lib.load().sa_qk_norm_rope(
            q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), self.w,
            None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(), self.cs,
            None if positions is None else positions.data_ptr(), *self.fwd,
            torch._C._cuda_getCurrentRawStream(self.device))
        if st != _lib.SA_OK:
            if st == _lib.SA_ERR_ALIGN:
                return None
            _lib.check(st, "sa_qk_norm_rope")
        return q_out, k_out


    def run_bwd(self, q, k, dq_out, dk_out, q_weight, k_weight, cos, sin, positions, need_dw):
        """_bwd_direct, or None where a gradient needs a copy or a base is off a 16-byte boundary."""
        key = (dq_out.stride(), dk_out.stride())
        strides = self.bwd.get(key)
        if strides is None:
            if not (_stride_ok(dq_out) and _stride_ok(dk_out)):
                return None
            strides = _keep(self.bwd, key, (_strides(dq_out), _strides(dk_out)))
        dq, dk = torch.empty_like(q), torch.empty_like(k)
        dwq = torch.empty_like(q_weight) if need_dw and q_weight is not None else None
        dwk = torch.empty_like(k_weight) if need_dw and k_weight is not None else None
        ws, nbytes = None, 0
        if dwq is not None or dwk is not None:
            nbytes = _bwd_workspace(self.D, self.device)
            ws = q.new_empty(nbytes, dtype=torch.uint8)
        st = _lib.load().sa_qk_norm_rope_bwd(
            q.data_ptr(), k.data_ptr(), dq_out.data_ptr(), dk_out.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), self.w,
            None if dwq is None else dwq.data_ptr(), None if dwk is None else dwk.data_ptr(),
            None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(), self.cs,
            None if positions is None else positions.data_ptr(), *self.table,
            None if ws is None else ws.data_ptr(), nbytes, *self.ins, *strides, *self.out,
            torch._C._cuda_getCurrentRawStream(self.device))
        if st != _lib.SA_OK:
            if st == _lib.SA_ERR_ALIGN:
                return None
            _lib.check(st, "sa_qk_norm_rope_bwd")
        return dq, dk, dwq, dwk


def _plan_of(q, k, cos, sin, q_weight, k_weight, eps, positions):
    """The plan of a checked call, or None if it needs a copy, another device or has nothing to do."""
    try:
        key = _key_of(q, k, cos, sin, q_weight, k_weight, eps, positions)
        plan = _PLANS.get(key)
    except (AttributeError, TypeError):  # not tensors: the checks say so
        key = plan = None
    if plan is None:
        _check_qk(q, k, cos, sin, q_weight, k_weight, eps, positions)
        if (key is None or q.numel() + k.numel() == 0 or not _stride_ok(q) or not _stride_ok(k)
                or not _stride_ok(torch.empty_like(q)) or not _stride_ok(torch.empty_like(k))
                or not _plain(cos, sin, q_weight, k_weight, positions)):
            return None
        plan = _keep(_PLANS, key, _Plan(key, q, k, cos, sin, q_weight, k_weight, eps, positions))
    return plan if plan.device == torch._C._cuda_getDevice() else None


def _fwd_direct(q, k, q_weight, k_weight, cos, sin, positions, eps):
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    q_out, k_out = _like(q), _like(k)
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


@functools.lru_cache(maxsize=None)
def _bwd_workspace(D, device_index):
    """Bytes of the weight gradients' partial sums: by the head dim and the device's SM count."""
    n = int(_lib.load().sa_qk_norm_rope_bwd_workspace_size(D))
    if n < 0:
        _lib.check(n, "sa_qk_norm_rope_bwd_workspace_size")
    return n


def _bwd_direct(q, k, dq_out, dk_out, q_weight, k_weight, cos, sin, positions, eps, need_dw):
    """(dq, dk, dq_weight, dk_weight); the last two None without a weight or when not needed."""
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    dq, dk = _like(q), _like(k)
    q, k, dq_out, dk_out = (_rows(t) for t in (q, k, dq_out, dk_out))
    wq, wk, w_code = _weights(q_weight, k_weight)
    cos, sin, cs_code = _tables(cos, sin)
    pos, pos_bytes, pos_sb = _positions(positions, T)
    dwq = torch.empty_like(wq) if need_dw and wq is not None else None
    dwk = torch.empty_like(wk) if need_dw and wk is not None else None
    with K._on(q.device):
        nbytes, ws = 0, None
        if dwq is not None or dwk is not None:
            nbytes = _bwd_workspace(D, q.device.index)
            ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
        st = _lib.load().sa_qk_norm_rope_bwd(
            K._ptr(q), K._ptr(k), K._ptr(dq_out), K._ptr(dk_out), K._ptr(dq), K._ptr(dk), K._ptr(wq), K._ptr(wk),
            w_code, K._ptr(dwq), K._ptr(dwk), K._ptr(cos), K._ptr(sin), cs_code, K._ptr(pos), pos_bytes, pos_sb,
            0 if cos is None else cos.shape[0], K._ptr(ws), nbytes, B, Hq, Hkv, T, D,
            0 if cos is None else 2 * cos.shape[1], _strides(q), _strides(k), _strides(dq_out), _strides(dk_out),
            _strides(dq), _strides(dk), 0.0 if eps is None else float(eps), int(eps is not None),
            K._DTYPE_CODE[q.dtype], K._stream(q))
    _lib.check(st, "sa_qk_norm_rope_bwd")
    if dwq is not None and dwq.dtype != q_weight.dtype:
        dwq = dwq.to(q_weight.dtype)
    if dwk is not None and dwk.dtype != k_weight.dtype:
        dwk = dwk.to(k_weight.dtype)
    return dq, dk, dwq, dwk


class _QkNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, plan):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps = eps
        res = None if plan is None else plan.run(q, k, cos, sin, q_weight, k_weight, positions)
        ctx.plan = plan if res is not None else None
        if res is not None:
            return res
        if _traced(q):
            return K._ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)
        return _fwd_direct(q, k, q_weight, k_weight, cos, sin, positions, eps)

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        # (the wrapper costs microseconds and matters only where a graph of the gradient is being built)
        if torch.is_grad_enabled():
            return _grads_once(ctx, dq_out, dk_out)
        return _QkNormRopeFn._grads(ctx, dq_out, dk_out)

    @staticmethod
    def _grads(ctx, dq_out, dk_out):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        need = ctx.needs_input_grad
        need_dw = need[2] or need[3]
        if _traced(dq_out):
            dq, dk, dwq, dwk = K._ops().qk_norm_rope_bwd(q, k, dq_out, dk_out, wq, wk, cos, sin, positions, ctx.eps,
                                                         need_dw)
        else:
            res, plan = None, ctx.plan
            # (a hook on saved tensors may hand back others than the forward's)
            if (plan is not None and plan.device == torch._C._cuda_getDevice()
                    and plan.key == _key_of(q, k, cos, sin, wq, wk, ctx.eps, positions)):
                res = plan.run_bwd(q, k, dq_out, dk_out, wq, wk, cos, sin, positions, need_dw)
            dq, dk, dwq, dwk = res if res is not None else _bwd_direct(q, k, dq_out, dk_out, wq, wk, cos, sin,
                                                                      positions, ctx.eps, need_dw)
        return (dq, dk, dwq if need[2] else None, dwk if need[3] else None, None, None, None, None, None)


_grads_once = once_differentiable(_QkNormRopeFn._grads)


def qk_norm_rope(q, k, cos=None, sin=None, *, q_weight=None, k_weight=None, eps=1e-6, positions=None):
    """Root-mean-square norm of every query and key head, then the rotation of
    its position, in one pass; returns (q, k) in their own dtype and order of dims.

    q: [B, H_q, T, D], k: [B, H_kv, T, D], fp32, fp16 or bf16, any strides (outputs and
    gradients keep the order of dims: transposed views of a [B, T, H, D] projection give such
    views again), D a multiple of 16 up to 256.  Per head row x, in fp32 with one rounding at the end::

        n = x / sqrt(mean(x^2) + eps) * weight
        y = n with its first R channels rotated (rotate-half form, as ``sp2norm_rope_flash_attention``)

    cos / sin: [positions, R/2] tables (``precompute_rope_cos_sin(R, ...)``), R a multiple of
    16 up to D; None leaves the rotation out.  positions: int32 or int64 [T] or [B, T], the
    table row of each token (None: 0 .. T-1).  A position outside the tables is read as 0 and
    reported by ``sa_device_status``.  q_weight / k_weight: [D], None for 1.  eps=None leaves
    the norm out.  Differentiable once in q, k and the weights; the gradients of the weights are
    summed in fp32 in a fixed order, bitwise the same from run to run.  No gradient for cos / sin;
    forward-mode derivatives are refused.
    To capture a training step in a CUDA graph, let no eager graph of the same leaves live on
    (``torch.cuda.make_graphed_callables`` sees to it): torch ends such a capture with an error.
    """
    eps = None if eps is None else float(eps)
    traced = _traced(q)
    if traced:
        _check_qk(q, k, cos, sin, q_weight, k_weight, eps, positions)
        plan = None
    else:
        plan = _plan_of(q, k, cos, sin, q_weight, k_weight, eps, positions)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad
                                     or (q_weight is not None and q_weight.requires_grad)
                                     or (k_weight is not None and k_weight.requires_grad))
            or _has_tangent(q, k, q_weight, k_weight, cos, sin)):  # (the function refuses those)
        if traced:  # a traced autograd function drops a gradient of one tensor passed twice: k's as views are others
            k = k.view_as(k)
            k_weight = None if k_weight is None else k_weight.view_as(k_weight)
        return _QkNormRopeFn.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, plan)
    if traced:
        return K._ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)
    res = None if plan is None else plan.run(q, k, cos, sin, q_weight, k_weight, positions)
    return res if res is not None else _fwd_direct(q, k, q_weight, k_weight, cos, sin, positions, eps)


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
