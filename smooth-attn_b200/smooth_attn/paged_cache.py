"""The paged key-value cache around ``sp2norm_paged_attention``: block tables
and slots from request lengths, the append of new tokens, and the decode over
pages chosen by a cheap score.

The reference's decode (``src/smooth_attn/kernels.py:2681-2829``) is handed a
filled cache and a table built on the host.  Here a serving step stays on the
device, in one stream and one CUDA graph if wanted::

    s = paged_assign_slots(block_table, context_lens, new_lens, free_pages, free_head, N)
    q = qk_norm_rope_paged_append(q, k, v, k_cache, v_cache, s.slot_mapping, cos, sin, positions=s.positions)
    paged_key_means(key_means, k_cache, block_table, s.context_lens, start_lens=context_lens)
    o = sp2norm_sparse_paged_attention(q[:, :, None], k_cache, v_cache, key_means, block_table, s.context_lens, 64)

Lengths, slots and positions are new tensors; the block table, the caches, the
mean keys and (on release) the list of free pages are updated in place.
"""

from __future__ import annotations

import math
import os
from typing import NamedTuple

import torch

from . import _lib
from . import kernels as K
from . import qk_rope as R

MAX_REQUESTS = 16384  # one block scans all requests' lengths in shared memory
_WIDER = (torch.int64, torch.uint32, torch.uint64)


class PagedSlots(NamedTuple):
    """What ``paged_assign_slots`` gives, for N tokens of B requests."""

    slot_mapping: torch.Tensor  # int64 [N]: page * block_size + offset, -1 for a token without a place
    positions: torch.Tensor  # int32 [N]: the token's position in its sequence (0 without a place)
    cu_seqlens: torch.Tensor  # int32 [B + 1]: request b's tokens are cu_seqlens[b] .. cu_seqlens[b + 1]
    context_lens: torch.Tensor  # int32 [B]: cached tokens after this step
    free_head: torch.Tensor  # int32 [1]: the list's first page that is still free


# Checked calls by the signature of their tensors, with the arguments that follow from it (as in qk_rope.py).
_PLANS: dict = {}


def _plan(what, rest, tensors):
    """(key, plan) of a call; (None, None) where an argument is no tensor (the checks then say so)."""
    try:
        key = (what, rest, *[None if t is None else (t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors])
        return key, _PLANS.get(key)
    except (AttributeError, TypeError):
        return None, None


def _same_device(like, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != like.device:
            raise ValueError(f"{name} must live on {like.device}, got {t.device}")


def _int32(name, t, shape, like, exact=False):
    """t as a contiguous int32 tensor of that shape; exact: it is read or written in place and never copied."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} must live on {like.device}, got {t.device}")
    if t.dtype is torch.int32 and t.is_contiguous():
        return t
    if exact or t.dtype.is_floating_point or t.dtype.is_complex:
        raise ValueError(f"{name} must be a contiguous int32 tensor, got {t.dtype} with strides {t.stride()}")
    if t.dtype in _WIDER:  # what 32 bits do not hold stays as far out as it is (-1 and 2^31 - 1 are out everywhere)
        t = t.to(torch.int64).contiguous()
        if not t.is_cuda or R._traced(t):
            return t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
        out = torch.empty(shape, dtype=torch.int32, device=t.device)
        with K._on(t.device):
            _lib.check(_lib.load().sa_narrow_i64(t.data_ptr(), out.data_ptr(), t.numel(), K._stream(t)), "sa_narrow_i64")
        return out
    return t.to(torch.int32).contiguous()


def _table_of(block_table, block_size):
    """Checks a block table that is updated in place; returns (B, max_blocks)."""
    if not isinstance(block_table, torch.Tensor):
        raise TypeError("block_table must be a torch.Tensor")
    if not block_table.is_cuda:
        raise ValueError("block_table must be a CUDA tensor")
    if block_table.ndim != 2 or block_table.dtype is not torch.int32:
        raise ValueError(f"block_table must be int32 [B, max_blocks], got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    B, max_blocks = block_table.shape
    if max_blocks and (block_table.stride(1) != 1 or (B > 1 and block_table.stride(0) < max_blocks)):
        raise ValueError("block_table is updated in place: its rows must be contiguous and apart")
    if max_blocks == 0:
        raise ValueError("block_table needs at least one column")
    if block_size < 1 or max_blocks * block_size > 1 << 30:
        raise ValueError(f"block_size {block_size} with {max_blocks} pages a row is not supported")
    if B > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests a call, got {B}")
    return B, max_blocks


def _ld(block_table):
    return max(block_table.stride(0), block_table.shape[1])


def paged_assign_slots(block_table, context_lens, new_lens, free_pages, free_head, num_tokens, *, block_size=16):
    """Places the next tokens of a batch of requests in a paged cache, on the device.

    Request b holds context_lens[b] tokens (pages block_table[b, :ceil(context_lens[b] / block_size)])
    and brings new_lens[b] more; together they are the first sum(new_lens) of ``num_tokens`` flat
    tokens, in request order.  Pages are taken from free_pages[free_head:] in that order and written
    into block_table (int32 [B, max_blocks], in place).  Returns ``PagedSlots``; context_lens and
    free_head are not changed, their successors are in it.

    A token for which there is no room (its table row is full, the pool is empty, num_tokens is too
    small) gets slot -1 and is not counted in ``PagedSlots.context_lens``; so do the tokens behind the
    last request.  Negative lengths count as 0.  A page below 0, in the list or in the held part of
    a row, gives its tokens slot -1 too and is reported by ``sa_device_status``.  free_pages: int32
    [P]; free_head: int32 [1]; context_lens, new_lens: [B], at most 16384 requests.  One launch, no
    host synchronisation.
    """
    num_tokens, block_size = int(num_tokens), int(block_size)
    traced = R._traced(block_table)
    key = None
    if not traced:
        key, plan = _plan("slots", (num_tokens, block_size), (block_table, context_lens, new_lens, free_pages, free_head))
        if plan is not None and plan[0] == torch._C._cuda_getDevice():
            return _assign_call(plan, block_table, context_lens, new_lens, free_pages, free_head)
    given = (context_lens, new_lens, free_pages, free_head)
    B, max_blocks = _table_of(block_table, block_size)
    if not 0 <= num_tokens < 2 ** 31 - 1024:
        raise ValueError(f"num_tokens must be in [0, 2^31 - 1024), got {num_tokens}")
    context_lens = _int32("context_lens", context_lens, (B,), block_table)
    new_lens = _int32("new_lens", new_lens, (B,), block_table)
    if not isinstance(free_pages, torch.Tensor) or free_pages.ndim != 1:
        raise ValueError("free_pages must be a 1D tensor")
    free_pages = _int32("free_pages", free_pages, tuple(free_pages.shape), block_table)
    free_head = _int32("free_head", free_head, (1,), block_table)
    if traced:
        return PagedSlots(*K._ops().paged_assign_slots(block_table, context_lens, new_lens, free_pages, free_head,
                                                       num_tokens, block_size))
    now = (context_lens, new_lens, free_pages, free_head)
    if key is not None and all(a is b for a, b in zip(now, given)):
        R._keep(_PLANS, key, _assign_plan(block_table, free_pages, num_tokens, block_size))
    return _assign_direct(block_table, *now, num_tokens, block_size)


def _assign_plan(block_table, free_pages, num_tokens, block_size):
    B, max_blocks = block_table.shape
    return (block_table.get_device(), *R._held("sa_paged_assign_slots", 1, _ld(block_table)),
            *R._held("sa_paged_assign_slots", 5, free_pages.shape[0]), [num_tokens, B + 1, B, 1],
            R._held("sa_paged_assign_slots", 12, B, num_tokens, max_blocks, block_size))


def _assign_direct(block_table, context_lens, new_lens, free_pages, free_head, num_tokens, block_size):
    with K._on(block_table.device):
        return _assign_call(_assign_plan(block_table, free_pages, num_tokens, block_size), block_table, context_lens,
                            new_lens, free_pages, free_head)


def _assign_call(plan, block_table, context_lens, new_lens, free_pages, free_head):
    device, ld, num_free, parts, dims = plan
    N, _, B, _ = parts
    slots = block_table.new_empty(N, dtype=torch.int64)
    i32 = block_table.new_empty(N + 2 * B + 2)
    p = i32.data_ptr()
    st = _lib.load().sa_paged_assign_slots(
        block_table.data_ptr(), ld, context_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(), num_free,
        free_head.data_ptr(), slots.data_ptr(), p, p + 4 * N, p + 4 * (N + B + 1), p + 4 * (N + 2 * B + 1), *dims,
        torch._C._cuda_getCurrentRawStream(device))
    _lib.check(st, "sa_paged_assign_slots")
    return PagedSlots(slots, *torch.unsafe_split_with_sizes(i32, parts))


def paged_release_pages(block_table, context_lens, done, free_pages, free_head, *, block_size=16):
    """Gives the pages of ended requests back to the pool, on the device.

    The ceil(context_lens[b] / block_size) pages of every request with done[b] go, in request and
    page order, to the entries of free_pages (int32 [P], in place) in front of free_head, so they are
    the next to be taken.  Returns (context_lens with 0 for those requests, the new free_head); the
    arguments themselves are not changed.  block_table keeps its entries.  Giving back more pages than
    were taken (a request released twice from stale lengths) leaves those out that have no entry and
    is reported by ``sa_device_status``, as is a page below 0 that goes to the list.  A page belongs
    to one request: pages that requests share would be given back once for each.  done: bool [B].
    """
    block_size = int(block_size)
    traced = R._traced(block_table)
    key = None
    if not traced:
        key, plan = _plan("release", block_size, (block_table, context_lens, done, free_pages, free_head))
        if plan is not None and plan[0] == torch._C._cuda_getDevice():
            return _release_call(plan, block_table, context_lens, done, free_pages, free_head)
    given = (context_lens, done, free_head)
    B, _ = _table_of(block_table, block_size)
    context_lens = _int32("context_lens", context_lens, (B,), block_table)
    if not isinstance(done, torch.Tensor):
        raise TypeError("done must be a torch.Tensor")
    if done.dtype is not torch.bool or tuple(done.shape) != (B,):
        raise ValueError(f"done must be bool [{B}], got {done.dtype} {tuple(done.shape)}")
    if not isinstance(free_pages, torch.Tensor) or free_pages.ndim != 1:
        raise ValueError("free_pages must be a 1D tensor")
    _same_device(block_table, done=done)
    free_pages = _int32("free_pages", free_pages, tuple(free_pages.shape), block_table, exact=True)
    free_head = _int32("free_head", free_head, (1,), block_table)
    done = done.contiguous()
    if traced:
        return K._ops().paged_release_pages(block_table, context_lens, done, free_pages, free_head, block_size)
    if key is not None and all(a is b for a, b in zip((context_lens, done, free_head), given)):
        R._keep(_PLANS, key, _release_plan(block_table, free_pages, block_size))
    return _release_direct(block_table, context_lens, done, free_pages, free_head, block_size)


def _release_plan(block_table, free_pages, block_size):
    return (block_table.get_device(), *R._held("sa_paged_release_pages", 1, _ld(block_table)),
            *R._held("sa_paged_release_pages", 5, free_pages.shape[0]),
            R._held("sa_paged_release_pages", 9, *block_table.shape, block_size))


def _release_direct(block_table, context_lens, done, free_pages, free_head, block_size):
    with K._on(block_table.device):
        return _release_call(_release_plan(block_table, free_pages, block_size), block_table, context_lens, done,
                             free_pages, free_head)


def _release_call(plan, block_table, context_lens, done, free_pages, free_head):
    device, ld, num_free, dims = plan
    ctx, head = torch.empty_like(context_lens), torch.empty_like(free_head)
    st = _lib.load().sa_paged_release_pages(
        block_table.data_ptr(), ld, context_lens.data_ptr(), done.data_ptr(), free_pages.data_ptr(), num_free,
        free_head.data_ptr(), ctx.data_ptr(), head.data_ptr(), *dims, torch._C._cuda_getCurrentRawStream(device))
    _lib.check(st, "sa_paged_release_pages")
    return ctx, head


# ------------------------------------------------------------------ append


def _check_caches(k_cache, v_cache):
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        K._validate_cuda_tensor(t, name=name)
        if t.ndim != 4:
            raise ValueError(f"{name} must be [num_blocks, H_kv, block_size, D], got {tuple(t.shape)}")
        if not t.is_contiguous():  # (updated or read in place; the C ABI checks the base's alignment)
            raise ValueError(f"{name} must be contiguous")
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype or k_cache.device != v_cache.device:
        raise ValueError("k_cache and v_cache must have one shape, dtype and device")


def qk_norm_rope_paged_append(q, k, v, k_cache, v_cache, slot_mapping, cos=None, sin=None, *, positions=None,
                              q_weight=None, k_weight=None, eps=1e-6):
    """``qk_norm_rope`` of N new tokens whose keys and values go straight into a paged cache; returns q.

    q: [N, H_q, D], k, v: [N, H_kv, D] (fp16 or bf16, any token and head strides: views of a fused
    projection are read in place); k_cache, v_cache: [num_blocks, H_kv, block_size, D], updated in
    place; slot_mapping: int64 [N], page * block_size + offset of each token, no slot twice in a call.
    q and k are normalised and rotated as ``qk_norm_rope`` does (cos, sin, q_weight, k_weight, eps as
    there; positions: int32 or int64 [N], needed with tables), v is copied.  A token with a negative
    slot is padding: its q row is zeros and the caches are left as they are.  A slot past the cache is
    treated the same and reported by ``sa_device_status``, as is a position outside the tables.
    Returns the queries, contiguous [N, H_q, D]: ``q[:, :, None]`` is what ``sp2norm_paged_attention``
    takes for one token of each of N sequences.  Forward only.
    """
    eps = None if eps is None else float(eps)
    traced = R._traced(q)
    key = plan = None
    if not traced:
        key, plan = _plan("append", eps, (q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight))
    if plan is None:
        _check_append(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight, eps)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
            or R._has_tangent(q, k, v, q_weight, k_weight, cos, sin)):
        raise ValueError("the append has no backward (nor a forward derivative): call it under torch.no_grad() or on "
                         "detached tensors")
    if traced:
        return K._ops().qk_norm_rope_paged_append(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions,
                                                  q_weight, k_weight, eps)
    if plan is None and key is not None and q.shape[0] > 0 and slot_mapping.is_contiguous() and all(
            R._stride_ok(t) for t in (q, k, v)) and R._plain(cos, sin, q_weight, k_weight, positions):
        plan = R._keep(_PLANS, key, _AppendPlan(q, k, v, k_cache, cos, q_weight, k_weight, positions, eps))
    if plan is not None and plan.device == torch._C._cuda_getDevice():
        out = plan.run(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight)
        if out is not None:
            return out
    return _append_direct(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight, eps)


def _check_append(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight, eps):
    assert q.ndim == 3 and k.ndim == 3 and v.ndim == 3
    N, H_q, D = q.shape
    H_kv = k.shape[1]
    assert H_kv > 0 and k.shape == (N, H_kv, D) and v.shape == (N, H_kv, D)
    for name, t in (("q", q), ("k", k), ("v", v)):
        K._validate_cuda_tensor(t, name=name)
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"append needs bf16 or fp16 q/k/v of one dtype, got {q.dtype}/{k.dtype}/{v.dtype}")
    _check_caches(k_cache, v_cache)
    if k_cache.dtype != q.dtype or k_cache.shape[1] != H_kv or k_cache.shape[3] != D:
        raise ValueError(f"caches {tuple(k_cache.shape)} {k_cache.dtype} do not match k {tuple(k.shape)} {k.dtype}")
    if D % 16 or not 16 <= D <= R.QK_MAX_HEAD_DIM:
        raise ValueError(f"head dim {D} not supported (a multiple of 16, 16 to {R.QK_MAX_HEAD_DIM})")
    if not isinstance(slot_mapping, torch.Tensor):
        raise TypeError("slot_mapping must be a torch.Tensor")
    if slot_mapping.dtype is not torch.int64 or tuple(slot_mapping.shape) != (N,):
        raise ValueError(f"slot_mapping must be int64 [{N}], got {slot_mapping.dtype} {tuple(slot_mapping.shape)}")
    _same_device(q, k=k, v=v, k_cache=k_cache, slot_mapping=slot_mapping)
    R._check_norm(eps, q_weight, k_weight)
    R._check_weight(q_weight, "q_weight", D, q)
    R._check_weight(k_weight, "k_weight", D, q)
    rotary, _ = R._check_tables(cos, sin, D, q)
    R._check_positions(positions, ((N,),), q)
    if rotary and positions is None:
        raise ValueError("positions are needed with cos / sin tables")


class _AppendPlan:
    """qk_norm_rope_paged_append of one signature whose arguments need no copy."""

    def __init__(self, q, k, v, k_cache, cos, q_weight, k_weight, positions, eps):
        N, H_q, D = q.shape
        num_blocks, H_kv, block_size, _ = k_cache.shape
        w, cs, pos_bytes, _, rows = R._row_args(cos, cos, q_weight, k_weight, positions, N)
        (self.w,) = R._held("sa_qk_norm_rope_paged_append", 9, w)
        (self.cs,) = R._held("sa_qk_norm_rope_paged_append", 12, cs)
        self.rest = R._held(
            "sa_qk_norm_rope_paged_append", 14, pos_bytes, rows, N, H_q, H_kv, D, 0 if cos is None else 2 * cos.shape[1],
            num_blocks, block_size, R._strides(q), R._strides(k), R._strides(v), 0.0 if eps is None else float(eps),
            int(eps is not None), K._DTYPE_CODE[q.dtype])
        self.device = q.get_device()

    def run(self, q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight):
        """The queries, or None where a base is off a 16-byte boundary."""
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        st = _lib.load().sa_qk_norm_rope_paged_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            slot_mapping.data_ptr(), None if q_weight is None else q_weight.data_ptr(),
            None if k_weight is None else k_weight.data_ptr(), self.w, None if cos is None else cos.data_ptr(),
            None if sin is None else sin.data_ptr(), self.cs, None if positions is None else positions.data_ptr(),
            *self.rest, torch._C._cuda_getCurrentRawStream(self.device))
        if st != _lib.SA_OK:
            if st == _lib.SA_ERR_ALIGN:
                return None
            _lib.check(st, "sa_qk_norm_rope_paged_append")
        return out


def _append_direct(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight, eps):
    N, H_q, D = q.shape
    num_blocks, H_kv, block_size, _ = k_cache.shape
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if N == 0:
        return out
    q, k, v = R._rows(q), R._rows(k), R._rows(v)
    wq, wk, w_code = R._weights(q_weight, k_weight)
    cos, sin, cs_code = R._tables(cos, sin)
    pos, pos_bytes, _ = R._positions(positions if cos is not None else None, N)
    slot_mapping = slot_mapping.contiguous()
    with K._on(q.device):
        st = _lib.load().sa_qk_norm_rope_paged_append(
            K._ptr(q), k.data_ptr(), v.data_ptr(), K._ptr(out), K._ptr(k_cache), K._ptr(v_cache),
            slot_mapping.data_ptr(), K._ptr(wq), K._ptr(wk), w_code, K._ptr(cos), K._ptr(sin), cs_code, K._ptr(pos),
            pos_bytes, 0 if cos is None else cos.shape[0], N, H_q, H_kv, D, 0 if cos is None else 2 * cos.shape[1],
            num_blocks, block_size, R._strides(q), R._strides(k), R._strides(v), 0.0 if eps is None else float(eps),
            int(eps is not None), K._DTYPE_CODE[q.dtype], K._stream(q))
    _lib.check(st, "sa_qk_norm_rope_paged_append")
    return out


# ------------------------------------------------------------------ pages chosen by a cheap score


def _check_pages(like, block_table, context_lens, B):
    if not isinstance(block_table, torch.Tensor) or block_table.ndim != 2:
        raise ValueError("block_table must be a 2D tensor")
    block_table = _int32("block_table", block_table, (B, block_table.shape[1]), like)
    return block_table, _int32("context_lens", context_lens, (B,), like)


def _check_means(key_means, num_blocks, H_kv, D, dtype, like):
    K._validate_cuda_tensor(key_means, name="key_means")
    if tuple(key_means.shape) != (num_blocks, H_kv, D) or key_means.dtype != dtype or key_means.device != like.device:
        raise ValueError(f"key_means must be {dtype} {(num_blocks, H_kv, D)} on {like.device}, got {key_means.dtype} "
                         f"{tuple(key_means.shape)}")
    if not key_means.is_contiguous():
        raise ValueError("key_means must be contiguous")


def paged_key_means(key_means, k_cache, block_table, context_lens, *, start_lens=None):
    """Mean key of every full page, for ``sp2norm_sparse_paged_attention``; key_means is updated in place.

    k_cache: [num_blocks, H_kv, block_size, D] (fp16 or bf16, D in {32, 64, 128, 256});
    key_means: [num_blocks, H_kv, D] of its dtype, the mean in fp32 rounded once.  Of sequence b the
    pages that context_lens[b] tokens fill are set, with start_lens only those that start_lens[b]
    tokens did not fill yet: after a step, pass the lengths before and after it.  Other pages' rows
    are left as they are.  A block_table entry outside the cache is skipped and reported by
    ``sa_device_status``.  At most 65535 sequences times key heads.  Returns key_means.
    """
    traced = R._traced(k_cache)
    key = None
    if not traced:
        key, plan = _plan("means", None, (key_means, k_cache, block_table, context_lens, start_lens))
        if plan is not None and plan[0] == torch._C._cuda_getDevice():
            return _means_call(plan, key_means, k_cache, block_table, context_lens, start_lens)
    given = (block_table, context_lens, start_lens)
    K._validate_cuda_tensor(k_cache, name="k_cache")
    if k_cache.ndim != 4 or not k_cache.is_contiguous():
        raise ValueError("k_cache must be a contiguous [num_blocks, H_kv, block_size, D]")
    num_blocks, H_kv, block_size, D = k_cache.shape
    if k_cache.dtype not in (torch.bfloat16, torch.float16) or D not in K.PAGED_HEAD_DIMS:
        raise ValueError(f"k_cache {k_cache.dtype} with head dim {D} not supported (bf16 or fp16, {K.PAGED_HEAD_DIMS})")
    _check_means(key_means, num_blocks, H_kv, D, k_cache.dtype, k_cache)
    B = block_table.shape[0] if isinstance(block_table, torch.Tensor) and block_table.ndim == 2 else -1
    block_table, context_lens = _check_pages(k_cache, block_table, context_lens, B)
    if start_lens is not None:
        start_lens = _int32("start_lens", start_lens, (B,), k_cache)
    if traced:
        K._ops().paged_key_means(key_means, k_cache, block_table, context_lens, start_lens)
        return key_means
    if key is not None and block_table.numel() and k_cache.numel() and all(
            a is b for a, b in zip((block_table, context_lens, start_lens), given)):
        R._keep(_PLANS, key, _means_plan(k_cache, block_table))
    return _means_direct(key_means, k_cache, block_table, context_lens, start_lens)


def _means_plan(k_cache, block_table):
    num_blocks, H_kv, block_size, D = k_cache.shape
    B, max_blocks = block_table.shape
    return k_cache.get_device(), R._held("sa_paged_key_means", 5, B, H_kv, num_blocks, block_size, max_blocks, D,
                                         K._DTYPE_CODE[k_cache.dtype])


def _means_direct(key_means, k_cache, block_table, context_lens, start_lens):
    if block_table.numel() == 0 or k_cache.numel() == 0:
        return key_means
    with K._on(k_cache.device):
        return _means_call(_means_plan(k_cache, block_table), key_means, k_cache, block_table, context_lens, start_lens)


def _means_call(plan, key_means, k_cache, block_table, context_lens, start_lens):
    device, dims = plan
    st = _lib.load().sa_paged_key_means(
        k_cache.data_ptr(), key_means.data_ptr(), block_table.data_ptr(), context_lens.data_ptr(),
        None if start_lens is None else start_lens.data_ptr(), *dims, torch._C._cuda_getCurrentRawStream(device))
    _lib.check(st, "sa_paged_key_means")
    return key_means


def _check_query(q, key_means, block_table, context_lens, num_pages, block_size):
    assert q.ndim == 4 and q.shape[2] == 1, "Decode: q must be [B, H, 1, D]"
    B, H_q, _, D = q.shape
    K._validate_cuda_tensor(q, name="q")
    K._validate_cuda_tensor(key_means, name="key_means")
    if key_means.ndim != 3:
        raise ValueError(f"key_means must be [num_blocks, H_kv, D], got {tuple(key_means.shape)}")
    num_blocks, H_kv, _ = key_means.shape
    assert H_kv > 0 and H_q % H_kv == 0
    if q.dtype not in (torch.bfloat16, torch.float16) or D not in K.PAGED_HEAD_DIMS:
        raise ValueError(f"q {q.dtype} with head dim {D} not supported (bf16 or fp16, {K.PAGED_HEAD_DIMS})")
    _check_means(key_means, num_blocks, H_kv, D, q.dtype, q)
    block_table, context_lens = _check_pages(q, block_table, context_lens, B)
    if num_pages < 1:
        raise ValueError(f"num_pages must be at least 1, got {num_pages}")
    if block_size < 1:
        raise ValueError(f"block_size must be at least 1, got {block_size}")
    return block_table, context_lens, min(num_pages, block_table.shape[1])


def sp2norm_paged_select(q, key_means, block_table, context_lens, num_pages, *, scale=None, block_size=16):
    """The pages that ``sp2norm_sparse_paged_attention`` reads: (pages, lens).

    q: [B, H_q, 1, D]; key_means: [num_blocks, H_kv, D] from ``paged_key_means``.  Of a sequence's
    n = ceil(context_len / block_size) pages, every key head keeps the last one and the num_pages - 1
    others with the highest::

        score(page) = sum over the group's query heads of squareplus(2 scale q . key_mean - 1)^2

    (the weight the attention would give the page's mean token, before it is normalised: of a group's
    heads one with large queries has more say; in 64 bits; ties go to the lowest page, NaN counts as
    the highest).  pages: int32 [B, H_kv, min(num_pages, max_blocks)], indices
    into the sequence's row of block_table, ascending, then -1; lens: int32 [B, H_kv], the tokens in
    them.  Lengths outside [0, max_blocks * block_size] are clamped; block_table entries outside the
    cache are read as page 0 and reported by ``sa_device_status``.  At most 65535 sequences times key
    heads.
    """
    num_pages, block_size = int(num_pages), int(block_size)
    block_table, context_lens, n = _check_query(q, key_means, block_table, context_lens, num_pages, block_size)
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    if R._traced(q):
        return K._ops().paged_select(q, key_means, block_table, context_lens, n, scale, block_size)
    return _select_direct(q, key_means, block_table, context_lens, n, scale, block_size)


def _select_direct(q, key_means, block_table, context_lens, n, scale, block_size):
    B, H_q, _, D = q.shape
    num_blocks, H_kv, _ = key_means.shape
    max_blocks = block_table.shape[1]
    pages = torch.empty(B, H_kv, n, device=q.device, dtype=torch.int32)
    lens = torch.empty(B, H_kv, device=q.device, dtype=torch.int32)
    if B == 0:
        return pages, lens
    if max_blocks == 0 or num_blocks == 0:
        return pages.fill_(-1), lens.zero_()
    q = R._dense(q)
    lib = _lib.load()
    with K._on(q.device):
        nbytes = int(lib.sa_paged_select_workspace_size(B, H_kv, max_blocks))
        if nbytes < 0:
            _lib.check(nbytes, "sa_paged_select_workspace_size")
        ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
        st = lib.sa_paged_select(q.data_ptr(), key_means.data_ptr(), block_table.data_ptr(), context_lens.data_ptr(),
                                 pages.data_ptr(), lens.data_ptr(), ws.data_ptr(), nbytes, B, H_q, H_kv, num_blocks,
                                 block_size, max_blocks, n, D, scale, K._DTYPE_CODE[q.dtype], K._stream(q))
    _lib.check(st, "sa_paged_select")
    return pages, lens


def sp2norm_sparse_paged_attention(q, k_cache, v_cache, key_means, block_table, context_lens, num_pages, *,
                                   scale=None, block_size=16, return_pages=False):
    """``sp2norm_paged_attention`` over the num_pages pages of each sequence and key head that a cheap score chooses.

    q, k_cache, v_cache, block_table, context_lens, scale, block_size as ``sp2norm_paged_attention``
    (caches contiguous); key_means and the choice as ``sp2norm_paged_select``.  The normaliser runs
    over the tokens of the chosen pages alone; with num_pages >= ceil(context_len / block_size) that
    is every token.  Returns the bf16 [B, H_q, D] output, with return_pages also the chosen pages
    (int32 [B, H_kv, min(num_pages, max_blocks)], as ``sp2norm_paged_select``).
    """
    num_pages, block_size, scale = int(num_pages), int(block_size), None if scale is None else float(scale)
    traced = R._traced(q)
    key = None
    if not traced:
        # (the decode kernel, and so the workspace, is chosen by this variable too)
        key, plan = _plan("sparse", (num_pages, block_size, scale, os.environ.get("SA_PAGED_DECODE_KERNEL")),
                          (q, k_cache, v_cache, key_means, block_table, context_lens))
        if plan is not None and plan[0] == torch._C._cuda_getDevice():
            out, pages = _sparse_call(plan, q, k_cache, v_cache, key_means, block_table, context_lens, return_pages)
            return (out, pages) if return_pages else out
    given = (block_table, context_lens)
    block_table, context_lens, n = _check_query(q, key_means, block_table, context_lens, num_pages, block_size)
    _check_caches(k_cache, v_cache)
    num_blocks, H_kv, D = key_means.shape
    if tuple(k_cache.shape) != (num_blocks, H_kv, block_size, D) or k_cache.dtype != q.dtype:
        raise ValueError(f"caches {tuple(k_cache.shape)} {k_cache.dtype} do not match key_means "
                         f"{tuple(key_means.shape)} {key_means.dtype} and block_size {block_size}")
    _same_device(q, k_cache=k_cache)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if traced:
        out, pages = K._ops().sparse_paged_decode(q, k_cache, v_cache, key_means, block_table, context_lens, n, scale,
                                                  block_size)
    else:
        if key is not None and q.numel() and block_table.numel() and num_blocks and q.is_contiguous() and all(
                a is b for a, b in zip((block_table, context_lens), given)):
            R._keep(_PLANS, key, _sparse_plan(q, key_means, block_table, n, scale, block_size))
        out, pages = _sparse_direct(q, k_cache, v_cache, key_means, block_table, context_lens, n, scale, block_size,
                                    return_pages)
    return (out, pages) if return_pages else out


def _sparse_plan(q, key_means, block_table, n, scale, block_size):
    B, H_q, _, D = q.shape
    num_blocks, H_kv, _ = key_means.shape
    max_blocks = block_table.shape[1]
    code = K._DTYPE_CODE[q.dtype]
    with K._on(q.device):
        nbytes = int(_lib.load().sa_sparse_paged_decode_workspace_size(B, H_q, H_kv, max_blocks, n, block_size, D,
                                                                       code))
    if nbytes < 0:
        _lib.check(nbytes, "sa_sparse_paged_decode_workspace_size")
    return (q.get_device(), nbytes, (B, H_q, D), (B, H_kv, n),
            R._held("sa_sparse_paged_decode", 9, nbytes, B, H_q, H_kv, num_blocks, block_size, max_blocks, n, D, scale,
                    code))


def _sparse_call(plan, q, k_cache, v_cache, key_means, block_table, context_lens, with_pages):
    device, nbytes, out_shape, pages_shape, dims = plan
    if q.data_ptr() % 16:
        q = R._copied(q)
    out = q.new_empty(out_shape, dtype=torch.bfloat16)
    pages = block_table.new_empty(pages_shape) if with_pages else None
    ws = block_table.new_empty(nbytes, dtype=torch.uint8)
    st = _lib.load().sa_sparse_paged_decode(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), key_means.data_ptr(), out.data_ptr(),
        block_table.data_ptr(), context_lens.data_ptr(), pages.data_ptr() if with_pages else None, ws.data_ptr(),
        *dims, torch._C._cuda_getCurrentRawStream(device))
    _lib.check(st, "sa_sparse_paged_decode")
    return out, pages


def _sparse_direct(q, k_cache, v_cache, key_means, block_table, context_lens, n, scale, block_size, with_pages=True):
    B, H_q, _, D = q.shape
    num_blocks, H_kv, _ = key_means.shape
    if q.numel() == 0 or block_table.numel() == 0 or num_blocks == 0:
        return (torch.zeros(B, H_q, D, device=q.device, dtype=torch.bfloat16),
                torch.full((B, H_kv, n), -1, device=q.device, dtype=torch.int32) if with_pages else None)
    with K._on(q.device):
        q = q.contiguous()
        return _sparse_call(_sparse_plan(q, key_means, block_table, n, scale, block_size), q, k_cache, v_cache,
                            key_means, block_table, context_lens, with_pages)
