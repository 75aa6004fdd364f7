"""``torch.library`` custom ops over the C ABI, so that ``torch.compile``
(and any other tracer: ``make_fx``, ``torch.export``) records each fused
kernel as one opaque node instead of breaking the graph at a ctypes call.

The reference's Triton kernels are traced by ``torch.compile`` as user
kernels; a ctypes launch is not traceable, so the public functions in
``kernels.py`` route through these ops whenever they run under a tracer
(``_tracing``) and call the C ABI directly otherwise (a custom-op dispatch
costs tens of microseconds, which would dominate the small decode calls).

Each op's real implementation is the direct launcher; its fake
implementation allocates outputs of the same shapes, dtypes and strides.
Outputs never alias inputs; the paged cache's ops update the arguments marked
* in place.  Ops (namespace ``smooth_attn_b200``):

* ``norm_fwd(x, alpha, theta, power, causal, with_rowsum) -> (out, rowsum)``
* ``norm_causal_bwd(x, g, rowsum, alpha, theta, power) -> dx``
* ``flash_fwd(q, k, v, scale, window_size, use_fast_sqrt, with_residual) -> (o, row_sums, o_lo)``
* ``flash_bwd(q, k, v, o, o_lo, do, row_sums, scale, window_size, use_fast_sqrt, deterministic) -> (dq, dk, dv)``
* ``flash_fwd_chunk(q, k, v, q_offset, scale, window_size, exact_math, with_residual) -> (o, row_sums, o_lo)``
* ``flash_bwd_chunk(q, k, v, o, o_lo, do, row_sums, q_offset, scale, window_size, exact_math, deterministic)
  -> (dq, dk, dv)``

``o_lo`` is the residual of o's 16-bit rounding (empty when not requested);
the backward ops take an empty ``o_lo`` for "none".
* ``rope_flash_fwd(q, k, v, cos, sin, scale, window_size) -> o``
* ``out_proj(a, w) -> a @ w`` (the RoPE projection GEMM)
* ``fp8_flash_fwd(q, k, v, scale, window_size) -> o``
* ``qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps) -> (q, k)``
* ``qk_norm_rope_bwd(q, k, dq_out, dk_out, q_weight, k_weight, cos, sin, positions, eps, need_dw)
  -> (dq, dk, dq_weight, dk_weight)`` (an empty gradient for a weight that is None or not needed)
* ``paged_assign_slots(*block_table, context_lens, new_lens, free_pages, free_head, num_tokens, block_size)
  -> (slot_mapping, positions, cu_seqlens, context_lens, free_head)``
* ``paged_release_pages(block_table, context_lens, done, *free_pages, free_head, block_size)
  -> (context_lens, free_head)``
* ``qk_norm_rope_paged_append(q, k, v, *k_cache, *v_cache, slot_mapping, cos, sin, positions, q_weight,
  k_weight, eps) -> q``
* ``paged_key_means(*key_means, k_cache, block_table, context_lens, start_lens)``
* ``paged_select(q, key_means, block_table, context_lens, num_pages, scale, block_size) -> (pages, lens)``
* ``sparse_paged_decode(q, k_cache, v_cache, key_means, block_table, context_lens, num_pages, scale,
  block_size) -> (out, pages)``
* ``paged_decode(q, k_cache, v_cache, block_table, context_lens, scale, block_size) -> out``
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import kernels as K
from . import paged_cache as P
from . import qk_rope as R

NS = "smooth_attn_b200"


def _rows(x: Tensor) -> int:
    L = x.shape[-1]
    return x.numel() // L if L else 0


# ------------------------------------------------------------------ norm


@torch.library.custom_op(f"{NS}::norm_fwd", mutates_args=(), device_types="cuda")
def norm_fwd(x: Tensor, alpha: float, theta: float, power: int, causal: bool,
             with_rowsum: bool) -> tuple[Tensor, Tensor]:
    x = x.contiguous()
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    rowsum = torch.empty(_rows(x) if with_rowsum else 0, device=x.device, dtype=torch.float32)
    if x.numel():
        L = x.shape[-1]
        fam = K.FamilyConfig(alpha=alpha, theta=theta, power=power)
        K._norm_fwd_direct(x.view(-1, L), out.view(-1, L), fam, causal, rowsum if with_rowsum else None)
    return out, rowsum


@norm_fwd.register_fake
def _(x, alpha, theta, power, causal, with_rowsum):
    return (torch.empty(x.shape, device=x.device, dtype=x.dtype),
            torch.empty(_rows(x) if with_rowsum else 0, device=x.device, dtype=torch.float32))


@torch.library.custom_op(f"{NS}::norm_causal_bwd", mutates_args=(), device_types="cuda")
def norm_causal_bwd(x: Tensor, g: Tensor, rowsum: Tensor, alpha: float, theta: float, power: int) -> Tensor:
    x, g, rowsum = x.contiguous(), g.contiguous(), rowsum.contiguous()
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if x.numel():
        L = x.shape[-1]
        fam = K.FamilyConfig(alpha=alpha, theta=theta, power=power)
        K._norm_bwd_direct(x.view(-1, L), g.view(-1, L), rowsum, dx.view(-1, L), fam, True)
    return dx


@norm_causal_bwd.register_fake
def _(x, g, rowsum, alpha, theta, power):
    return torch.empty(x.shape, device=x.device, dtype=x.dtype)


# ------------------------------------------------------------------ flash attention


@torch.library.custom_op(f"{NS}::flash_fwd", mutates_args=(), device_types="cuda")
def flash_fwd(q: Tensor, k: Tensor, v: Tensor, scale: float, window_size: int,
              use_fast_sqrt: bool, with_residual: bool) -> tuple[Tensor, Tensor, Tensor]:
    q, k, v = K._flash_ready(q), K._flash_ready(k), K._flash_ready(v)
    o = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    res = K._flash_fwd_direct(q, k, v, scale, window_size, use_fast_sqrt, o=o, with_residual=with_residual)
    return res if with_residual else (res[0], res[1], q.new_empty(0))


@flash_fwd.register_fake
def _(q, k, v, scale, window_size, use_fast_sqrt, with_residual):
    B, H, T, _ = q.shape
    return (torch.empty(q.shape, device=q.device, dtype=q.dtype),
            torch.empty(B, H, T, device=q.device, dtype=torch.float32),
            torch.empty(q.shape if with_residual else (0,), device=q.device, dtype=q.dtype))


@torch.library.custom_op(f"{NS}::flash_bwd", mutates_args=(), device_types="cuda")
def flash_bwd(q: Tensor, k: Tensor, v: Tensor, o: Tensor, o_lo: Tensor, do: Tensor, row_sums: Tensor, scale: float,
              window_size: int, use_fast_sqrt: bool, deterministic: bool) -> tuple[Tensor, Tensor, Tensor]:
    q, k, v, o = (K._flash_ready(t) for t in (q, k, v, o))
    return K._flash_bwd_direct(q, k, v, o, do, row_sums.contiguous(), scale, window_size, use_fast_sqrt,
                               o_lo=o_lo if o_lo.numel() else None, deterministic=deterministic)


@flash_bwd.register_fake
def _(q, k, v, o, o_lo, do, row_sums, scale, window_size, use_fast_sqrt, deterministic):
    return tuple(torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))


@torch.library.custom_op(f"{NS}::flash_fwd_chunk", mutates_args=(), device_types="cuda")
def flash_fwd_chunk(q: Tensor, k: Tensor, v: Tensor, q_offset: int, scale: float, window_size: int,
                    exact_math: bool, with_residual: bool) -> tuple[Tensor, Tensor, Tensor]:
    res = K._flash_fwd_chunk_direct(q, k, v, q_offset, scale, window_size, exact_math, with_residual)
    return res if with_residual else (res[0], res[1], q.new_empty(0))


@flash_fwd_chunk.register_fake
def _(q, k, v, q_offset, scale, window_size, exact_math, with_residual):
    B, H, T, _ = q.shape
    return (torch.empty(q.shape, device=q.device, dtype=q.dtype),
            torch.empty(B, H, T, device=q.device, dtype=torch.float32),
            torch.empty(q.shape if with_residual else (0,), device=q.device, dtype=q.dtype))


@torch.library.custom_op(f"{NS}::flash_bwd_chunk", mutates_args=(), device_types="cuda")
def flash_bwd_chunk(q: Tensor, k: Tensor, v: Tensor, o: Tensor, o_lo: Tensor, do: Tensor, row_sums: Tensor,
                    q_offset: int, scale: float, window_size: int, exact_math: bool,
                    deterministic: bool) -> tuple[Tensor, Tensor, Tensor]:
    return K._flash_bwd_chunk_direct(q, k, v, o, do, row_sums.contiguous(), q_offset, scale, window_size,
                                     exact_math, o_lo if o_lo.numel() else None, deterministic)


@flash_bwd_chunk.register_fake
def _(q, k, v, o, o_lo, do, row_sums, q_offset, scale, window_size, exact_math, deterministic):
    return tuple(torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))


@torch.library.custom_op(f"{NS}::rope_flash_fwd", mutates_args=(), device_types="cuda")
def rope_flash_fwd(q: Tensor, k: Tensor, v: Tensor, cos: Tensor, sin: Tensor, scale: float,
                   window_size: int) -> Tensor:
    return K._rope_flash_fwd_direct(q, k, v, cos, sin, scale, window_size)[0]


@rope_flash_fwd.register_fake
def _(q, k, v, cos, sin, scale, window_size):
    return torch.empty(q.shape, device=q.device, dtype=q.dtype)


@torch.library.custom_op(f"{NS}::out_proj", mutates_args=(), device_types="cuda")
def out_proj(a: Tensor, w: Tensor) -> Tensor:
    return K._out_proj_direct(a, w)


@out_proj.register_fake
def _(a, w):
    return torch.empty(a.shape[0], w.shape[1], device=a.device, dtype=a.dtype)


@torch.library.custom_op(f"{NS}::fp8_flash_fwd", mutates_args=(), device_types="cuda")
def fp8_flash_fwd(q: Tensor, k: Tensor, v: Tensor, scale: float, window_size: int) -> Tensor:
    return K._fp8_flash_fwd_direct(q, k, v, scale, window_size)


@fp8_flash_fwd.register_fake
def _(q, k, v, scale, window_size):
    return torch.empty(q.shape, device=q.device, dtype=torch.bfloat16)


@torch.library.custom_op(f"{NS}::paged_decode", mutates_args=(), device_types="cuda")
def paged_decode(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, context_lens: Tensor,
                 scale: float, block_size: int) -> Tensor:
    # (the graphs of mode="reduce-overhead" allow no allocation that outlives the call: no kept workspace)
    return K._paged_decode_direct(q, k_cache, v_cache, block_table, context_lens, scale, block_size, False)


@paged_decode.register_fake
def _(q, k_cache, v_cache, block_table, context_lens, scale, block_size):
    B, H, _, D = q.shape
    return torch.empty(B, H, D, device=q.device, dtype=torch.bfloat16)


# ------------------------------------------------------------------ head norm and rotation


@torch.library.custom_op(f"{NS}::qk_norm_rope", mutates_args=(), device_types="cuda")
def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Tensor | None, k_weight: Tensor | None, cos: Tensor | None,
                 sin: Tensor | None, positions: Tensor | None, eps: float | None) -> tuple[Tensor, Tensor]:
    return R._fwd_direct(q, k, q_weight, k_weight, cos, sin, positions, eps)


@qk_norm_rope.register_fake
def _(q, k, q_weight, k_weight, cos, sin, positions, eps):
    return tuple(R._like(t) for t in (q, k))


@torch.library.custom_op(f"{NS}::qk_norm_rope_bwd", mutates_args=(), device_types="cuda")
def qk_norm_rope_bwd(q: Tensor, k: Tensor, dq_out: Tensor, dk_out: Tensor, q_weight: Tensor | None,
                     k_weight: Tensor | None, cos: Tensor | None, sin: Tensor | None, positions: Tensor | None,
                     eps: float | None, need_dw: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dq, dk, dwq, dwk = R._bwd_direct(q, k, dq_out, dk_out, q_weight, k_weight, cos, sin, positions, eps, need_dw)
    return (dq, dk, dwq if dwq is not None else q.new_empty(0), dwk if dwk is not None else q.new_empty(0))


@qk_norm_rope_bwd.register_fake
def _(q, k, dq_out, dk_out, q_weight, k_weight, cos, sin, positions, eps, need_dw):
    dw = tuple(torch.empty(w.shape, device=q.device, dtype=w.dtype) if need_dw and w is not None else q.new_empty(0)
               for w in (q_weight, k_weight))
    return tuple(R._like(t) for t in (q, k)) + dw


# ------------------------------------------------------------------ paged cache


@torch.library.custom_op(f"{NS}::paged_assign_slots", mutates_args=("block_table",), device_types="cuda")
def paged_assign_slots(block_table: Tensor, context_lens: Tensor, new_lens: Tensor, free_pages: Tensor,
                       free_head: Tensor, num_tokens: int,
                       block_size: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    # (outputs of a custom op may not share storage: the direct call's int32 ones do)
    s = P._assign_direct(block_table, context_lens, new_lens, free_pages, free_head, num_tokens, block_size)
    return (s.slot_mapping, s.positions.clone(), s.cu_seqlens.clone(), s.context_lens.clone(), s.free_head.clone())


@paged_assign_slots.register_fake
def _(block_table, context_lens, new_lens, free_pages, free_head, num_tokens, block_size):
    B, dev = block_table.shape[0], block_table.device
    return (torch.empty(num_tokens, device=dev, dtype=torch.int64),
            *(torch.empty(n, device=dev, dtype=torch.int32) for n in (num_tokens, B + 1, B, 1)))


@torch.library.custom_op(f"{NS}::paged_release_pages", mutates_args=("free_pages",), device_types="cuda")
def paged_release_pages(block_table: Tensor, context_lens: Tensor, done: Tensor, free_pages: Tensor,
                        free_head: Tensor, block_size: int) -> tuple[Tensor, Tensor]:
    return P._release_direct(block_table, context_lens, done, free_pages, free_head, block_size)


@paged_release_pages.register_fake
def _(block_table, context_lens, done, free_pages, free_head, block_size):
    return torch.empty_like(context_lens), torch.empty_like(free_head)


@torch.library.custom_op(f"{NS}::qk_norm_rope_paged_append", mutates_args=("k_cache", "v_cache"), device_types="cuda")
def qk_norm_rope_paged_append(q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, slot_mapping: Tensor,
                              cos: Tensor | None, sin: Tensor | None, positions: Tensor | None,
                              q_weight: Tensor | None, k_weight: Tensor | None, eps: float | None) -> Tensor:
    return P._append_direct(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight, eps)


@qk_norm_rope_paged_append.register_fake
def _(q, k, v, k_cache, v_cache, slot_mapping, cos, sin, positions, q_weight, k_weight, eps):
    return torch.empty(q.shape, device=q.device, dtype=q.dtype)


@torch.library.custom_op(f"{NS}::paged_key_means", mutates_args=("key_means",), device_types="cuda")
def paged_key_means(key_means: Tensor, k_cache: Tensor, block_table: Tensor, context_lens: Tensor,
                    start_lens: Tensor | None) -> None:
    P._means_direct(key_means, k_cache, block_table, context_lens, start_lens)


@paged_key_means.register_fake
def _(key_means, k_cache, block_table, context_lens, start_lens):
    return None


@torch.library.custom_op(f"{NS}::paged_select", mutates_args=(), device_types="cuda")
def paged_select(q: Tensor, key_means: Tensor, block_table: Tensor, context_lens: Tensor, num_pages: int, scale: float,
                 block_size: int) -> tuple[Tensor, Tensor]:
    return P._select_direct(q, key_means, block_table, context_lens, num_pages, scale, block_size)


@paged_select.register_fake
def _(q, key_means, block_table, context_lens, num_pages, scale, block_size):
    B, Hkv = q.shape[0], key_means.shape[1]
    return (torch.empty(B, Hkv, num_pages, device=q.device, dtype=torch.int32),
            torch.empty(B, Hkv, device=q.device, dtype=torch.int32))


@torch.library.custom_op(f"{NS}::sparse_paged_decode", mutates_args=(), device_types="cuda")
def sparse_paged_decode(q: Tensor, k_cache: Tensor, v_cache: Tensor, key_means: Tensor, block_table: Tensor,
                        context_lens: Tensor, num_pages: int, scale: float,
                        block_size: int) -> tuple[Tensor, Tensor]:
    return P._sparse_direct(q, k_cache, v_cache, key_means, block_table, context_lens, num_pages, scale, block_size)


@sparse_paged_decode.register_fake
def _(q, k_cache, v_cache, key_means, block_table, context_lens, num_pages, scale, block_size):
    B, H, _, D = q.shape
    return (torch.empty(B, H, D, device=q.device, dtype=torch.bfloat16),
            torch.empty(B, key_means.shape[1], num_pages, device=q.device, dtype=torch.int32))
