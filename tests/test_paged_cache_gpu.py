"""The paged cache's operators against plain statements of them: slots and
release against Python loops (whole numbers, equal), the append and the mean
keys against the formula in 64 bits, the choice of pages against a 64-bit sort
(equal), the decode over them against the formula over the chosen pages, and a
serving run of all of them together.

Tolerances count roundings as in test_qk_norm_rope_gpu.py (whose 64-bit row
formula is used here); the decode's are derived at ``_attend``."""

import ctypes
import gc
import math
import threading

import pytest
import torch

import smooth_attn as sa
from smooth_attn import _lib
from tests._util import randn
from tests.test_qk_norm_rope_gpu import U, _angles, _check, _half_step, _ref64

pytestmark = pytest.mark.gpu
CUDA = "cuda"
I32 = torch.int32


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA required")


def _i32(v):
    return torch.tensor(v, dtype=I32, device=CUDA)


def _status():
    return _lib.load().sa_device_status(1)


# ------------------------------------------------------------------ slots


def slots_by_loop(table, ctx, new, pool, head, N, bs):
    """paged_assign_slots on lists; table is changed."""
    cap = len(table[0]) * bs if table else 0
    slots, pos, cu, out = [-1] * N, [0] * N, [0], []
    at = 0  # flat tokens seen
    for b, row in enumerate(table):
        c = min(max(ctx[b], 0), cap)
        want = min(max(new[b], 0), N - min(at, N), cap - c)
        need = -(-(c + want) // bs) - -(-c // bs)
        have = max(0, min(need, len(pool) - head))
        fits = min(want, (-(-c // bs) + have) * bs - c)
        for j in range(have):
            row[-(-c // bs) + j] = pool[head + j]
        for j in range(fits):
            p = c + j
            slots[min(at, N) + j] = row[p // bs] * bs + p % bs
            pos[min(at, N) + j] = p
        head = min(head + need, len(pool))
        at += max(new[b], 0)
        cu.append(min(at, N))
        out.append(c + fits)
    return slots, pos, cu, out, head


def _requests(seed, B, mb, bs, spare, most_new):
    g = torch.Generator().manual_seed(seed)
    ctx = torch.randint(0, mb * bs // 2 + 1, (B,), generator=g).tolist()
    new = torch.randint(0, most_new + 1, (B,), generator=g).tolist()
    held = [-(-c // bs) for c in ctx]
    pool = torch.randperm(sum(held) + spare, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(pool[at:at + h] + [-7] * (mb - h))
        at += h
    return table, ctx, new, pool, sum(held)


SLOT_CASES = [  # B, max_blocks, bs, spare pages, most new tokens, tokens in the buffer (None: their sum)
    (1, 1, 1, 1, 1, None), (1, 4, 16, 8, 40, None), (3, 8, 16, 30, 1, None), (64, 20, 16, 400, 1, 64),
    (7, 9, 5, 100, 30, None), (33, 40, 8, 1000, 90, 2000), (33, 40, 8, 1000, 90, 700),  # padding; a buffer too small
    (20, 30, 16, 11, 200, None),  # the pool runs out
    (20, 6, 16, 300, 300, None),  # rows run out
    (517, 12, 32, 2000, 64, None), (1500, 6, 64, 9000, 100, None), (6, 4, 128, 0, 60, None),
]


@pytest.mark.parametrize("case", SLOT_CASES, ids=str)
def test_slots_match_the_loop(case):
    B, mb, bs, spare, most_new, N = case
    table, ctx, new, pool, head = _requests(B + mb, B, mb, bs, spare, most_new)
    N = sum(new) if N is None else N
    wide = torch.full((B, mb + 3), -9, dtype=I32, device=CUDA)  # rows apart in memory
    t = wide[:, :mb]
    t.copy_(_i32(table))
    args = (_i32(ctx), _i32(new), _i32(pool), _i32([head]))
    keep = [a.clone() for a in args]
    s = sa.paged_assign_slots(t, *args, N, block_size=bs)
    want = slots_by_loop(table, ctx, new, pool, head, N, bs)
    assert t.tolist() == table and (wide[:, mb:] == -9).all()
    assert [s.slot_mapping.tolist(), s.positions.tolist(), s.cu_seqlens.tolist(), s.context_lens.tolist(),
            s.free_head.item()] == list(want)
    assert all(torch.equal(a, b) for a, b in zip(args, keep))
    assert s.slot_mapping.dtype == torch.int64 and s.positions.dtype == s.cu_seqlens.dtype == I32
    # again on the same state: the same
    r = sa.paged_assign_slots(t, *args, N, block_size=bs)
    assert all(torch.equal(a, b) for a, b in zip(s, r)) and t.tolist() == table


def test_slots_of_odd_lengths_and_types():
    table = [[3, -1], [4, 5], [-1, -1], [6, 7]]
    ctx, new = [-5, 99, 0, 17], [3, 2, -4, 1]  # out of range: counted as 0, a full row, 0
    t = _i32(table)
    s = sa.paged_assign_slots(t, torch.tensor(ctx, device=CUDA), torch.tensor(new, device=CUDA),
                              torch.tensor([9, 8], device=CUDA), torch.tensor([0], device=CUDA), 8)
    want = slots_by_loop(table, ctx, new, [9, 8], 0, 8, 16)
    assert [x.tolist() for x in s[:4]] == [list(x) for x in want[:4]] and s.free_head.item() == want[4]
    assert t.tolist() == table


def test_slots_of_nothing():
    e = torch.empty(0, dtype=I32, device=CUDA)
    s = sa.paged_assign_slots(torch.empty(0, 4, dtype=I32, device=CUDA), e, e, _i32([1, 2]), _i32([1]), 3)
    assert s.slot_mapping.tolist() == [-1] * 3 and s.cu_seqlens.tolist() == [0] and s.free_head.item() == 1
    t = _i32([[5, -1]])
    s = sa.paged_assign_slots(t, _i32([16]), _i32([4]), e, _i32([0]), 0)
    assert s.slot_mapping.numel() == 0 and s.context_lens.tolist() == [16] and t.tolist() == [[5, -1]]


def test_slots_of_the_largest_batch_and_buffer():
    B, bs = 16384, 16
    t = torch.full((B, 2), -1, dtype=I32, device=CUDA)
    ctx = torch.arange(B, device=CUDA, dtype=I32) % 2 * 16
    t[:, 0] = torch.where(ctx > 0, torch.arange(B, device=CUDA, dtype=I32), -1)
    pool = torch.arange(B, 2 * B, device=CUDA, dtype=I32).flip(0).contiguous()
    s = sa.paged_assign_slots(t, ctx, torch.ones_like(ctx), pool, _i32([0]), B, block_size=bs)
    col = (ctx > 0).long()[:, None]
    assert torch.equal(t.gather(1, col)[:, 0], pool) and s.free_head.item() == B
    assert torch.equal(s.slot_mapping, pool.long() * bs) and torch.equal(s.positions, ctx)
    # one request with over two million tokens
    n = 2_100_001
    t = torch.full((1, n // 16 + 1), -1, dtype=I32, device=CUDA)
    pool = torch.randperm(n // 16 + 1, device=CUDA).to(I32)
    s = sa.paged_assign_slots(t, _i32([0]), _i32([n]), pool, _i32([0]), n + 5)
    i = torch.arange(n, device=CUDA)
    assert torch.equal(s.slot_mapping[:n], pool.long()[i // 16] * 16 + i % 16) and torch.equal(t[0], pool)
    assert s.slot_mapping[n:].tolist() == [-1] * 5


def test_release_matches_the_loop():
    for B, mb, bs in ((1, 3, 16), (70, 9, 16), (1100, 5, 8)):
        table, ctx, _, pool, head = _requests(B, B, mb, bs, 13, 1)
        done = torch.rand(B, generator=torch.Generator().manual_seed(B)) < 0.5
        t, free, c = _i32(table), _i32(pool), _i32(ctx)
        keep = c.clone()
        out, h = sa.paged_release_pages(t, c, done.to(CUDA), free, _i32([head]), block_size=bs)
        back = [p for b in range(B) if done[b] for p in table[b][:-(-ctx[b] // bs)]]
        pool[head - len(back):head] = back
        assert free.tolist() == pool and h.item() == head - len(back) and torch.equal(c, keep)
        assert out.tolist() == [0 if done[b] else ctx[b] for b in range(B)] and t.tolist() == table
    _status()
    free = _i32([0, 1, 2])
    out, h = sa.paged_release_pages(_i32([[7, 8]]), _i32([32]), torch.tensor([True], device=CUDA), free, _i32([1]))
    assert h.item() == 0 and free.tolist() == [8, 1, 2]  # one page too many: left out
    assert _status() == _lib.SA_ERR_ARG and _status() == _lib.SA_OK


# ------------------------------------------------------------------ append


def _append_inputs(N, Hq, Hkv, D, dt, seed):
    qkv = randn((N, (Hq + 2 * Hkv) * D), seed, dt, CUDA)
    return (qkv[:, :Hq * D].view(N, Hq, D), qkv[:, Hq * D:(Hq + Hkv) * D].view(N, Hkv, D),
            qkv[:, (Hq + Hkv) * D:].view(N, Hkv, D))


@pytest.mark.parametrize("N,pad,Hq,Hkv,D,R,bs,dt,norm", [
    (1, 0, 1, 1, 32, 32, 1, torch.float16, True), (64, 0, 32, 8, 128, 128, 16, torch.bfloat16, True),
    (37, 5, 12, 12, 64, 32, 16, torch.bfloat16, True), (129, 1, 9, 3, 80, 80, 5, torch.float16, True),
    (50, 0, 4, 4, 256, 0, 32, torch.bfloat16, True), (77, 3, 8, 2, 128, 64, 64, torch.bfloat16, False),
    (513, 0, 16, 1, 16, 16, 8, torch.float16, False), (3, 3, 2, 2, 64, 64, 16, torch.bfloat16, True),
    (9001, 700, 32, 8, 64, 64, 16, torch.bfloat16, True),  # whole units of heads: slots and angles read ahead
    (9001, 7, 24, 8, 128, 64, 16, torch.float16, True),
])
@pytest.mark.parametrize("layout", ["fused", "heads first", "off"])
def test_append_matches_the_formula(N, pad, Hq, Hkv, D, R, bs, dt, norm, layout):
    g = torch.Generator().manual_seed(N + D)
    q, k, v = _append_inputs(N, Hq, Hkv, D, dt, N)
    if layout == "heads first":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    elif layout == "off":  # rows off a 16-byte boundary
        q, k, v = (torch.nn.functional.pad(t, (1, 0))[..., 1:] for t in (q, k, v))
    P = -(-N // bs) + 3
    slots = torch.randperm(P * bs, generator=g)[:N]
    slots[torch.randperm(N, generator=g)[:pad]] = -1 - torch.arange(pad)
    slots = slots.to(CUDA)
    pos = torch.randint(0, 900, (N,), generator=g).to(CUDA)
    cos, sin = (None, None) if R == 0 else _angles(900, R)
    wq, wk = (1 + randn((D,), 5 + i, torch.float32, CUDA, 0.3) for i in range(2)) if norm else (None, None)
    kc, vc = (randn((P, Hkv, bs, D), 90 + i, dt, CUDA) for i in range(2))
    kc0, vc0 = kc.clone(), vc.clone()
    eps = 1e-5 if norm else None
    out = sa.qk_norm_rope_paged_append(q, k, v, kc, vc, slots, cos, sin, positions=None if R == 0 else pos, q_weight=wq,
                                       k_weight=wk, eps=eps)
    real = slots >= 0
    yq, tq = _ref64(q.transpose(0, 1)[None], wq, cos, sin, pos[None], eps)
    yk, tk = _ref64(k.transpose(0, 1)[None], wk, cos, sin, pos[None], eps)
    yq, tq, yk, tk = (t[0].transpose(0, 1) for t in (yq, tq, yk, tk))
    assert out.is_contiguous() and (out[~real] == 0).all()
    _check(out[real], yq[real], tq[real])
    s = slots[real]
    _check(kc[s // bs, :, s % bs], yk[real], tk[real])
    assert torch.equal(vc[s // bs, :, s % bs], v[real])
    kc[s // bs, :, s % bs] = kc0[s // bs, :, s % bs]
    vc[s // bs, :, s % bs] = vc0[s // bs, :, s % bs]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)  # no other row was touched


def test_append_far_into_a_long_cache():
    """Element offsets past 2^31: 18 million rows of 128."""
    P, Hkv, bs, D = 140_001, 8, 16, 128
    kc, vc = (torch.zeros(P, Hkv, bs, D, device=CUDA, dtype=torch.bfloat16) for _ in range(2))
    q, k, v = _append_inputs(3, 8, Hkv, D, torch.bfloat16, 1)
    slots = torch.tensor([P * bs - 1, 5, 131_073 * bs + 7], device=CUDA)
    sa.qk_norm_rope_paged_append(q, k, v, kc, vc, slots, eps=None)
    assert torch.equal(vc[slots // bs, :, slots % bs], v) and torch.equal(kc[slots // bs, :, slots % bs], k)
    assert kc.count_nonzero() == k.count_nonzero() and vc.count_nonzero() == v.count_nonzero()
    # and read from there: the last page of one sequence, its mean, and a decode over it
    means = torch.zeros(P, Hkv, D, device=CUDA, dtype=torch.bfloat16)
    bt = _i32([[131_073, P - 1]])
    sa.paged_key_means(means, kc, bt, _i32([32]))
    _check(means[bt[0].long()], kc[bt[0].long()].double().mean(2),
           16 * U * kc[bt[0].long()].double().abs().mean(2))
    qd = q[:1, :, None]
    o = sa.sp2norm_sparse_paged_attention(qd, kc, vc, means, bt, _i32([32]), 2)
    _attend(o, qd, kc, vc, bt, [32], [[list(range(2))] * Hkv])


def test_append_reports_slots_past_the_cache():
    _status()
    kc, vc = (torch.zeros(2, 1, 4, 64, device=CUDA, dtype=torch.bfloat16) for _ in range(2))
    q, k, v = _append_inputs(3, 2, 1, 64, torch.bfloat16, 2)
    out = sa.qk_norm_rope_paged_append(q, k, v, kc, vc, torch.tensor([8, 2, 1 << 40], device=CUDA))
    assert _status() == _lib.SA_ERR_ARG
    assert (out[0] == 0).all() and (out[2] == 0).all() and (out[1] != 0).any()
    assert torch.equal(vc[0, 0, 2], v[1, 0]) and vc.count_nonzero() == v[1].count_nonzero()
    cos, sin = _angles(5, 64)
    sa.qk_norm_rope_paged_append(q, k, v, kc, vc, torch.tensor([0, 1, 2], device=CUDA), cos, sin,
                                 positions=torch.tensor([0, 5, -2], device=CUDA))
    assert _status() == _lib.SA_ERR_ARG and _status() == _lib.SA_OK
    assert sa.qk_norm_rope_paged_append(q[:0], k[:0], v[:0], kc, vc, torch.empty(0, dtype=torch.int64, device=CUDA)
                                        ).shape == (0, 2, 64)


# ------------------------------------------------------------------ mean keys


@pytest.mark.parametrize("Hkv,D,bs,dt", [(1, 32, 16, torch.float16), (8, 128, 16, torch.bfloat16),
                                         (3, 64, 8, torch.bfloat16), (2, 256, 64, torch.float16),
                                         (2, 128, 5, torch.bfloat16), (1, 64, 1, torch.bfloat16)])
def test_key_means(Hkv, D, bs, dt):
    B, mb = 5, 9
    g = torch.Generator().manual_seed(bs)
    ctx, start = [0, bs - 1, mb * bs, 4 * bs + bs // 2, 7 * bs], [0, 0, 2 * bs + 1, 4 * bs, 7 * bs - 1]
    kc = randn((B * mb, Hkv, bs, D), 1, dt, CUDA) + 1
    bt = torch.randperm(B * mb, generator=g).to(I32).view(B, mb).to(CUDA)
    for st in (None, start):
        means = randn((B * mb, Hkv, D), 2, dt, CUDA)
        before = means.clone()
        r = sa.paged_key_means(means, kc, bt, _i32(ctx), start_lens=None if st is None else _i32(st))
        assert r is means
        full = [bt[b, j].item() for b in range(B) for j in range((st[b] if st else 0) // bs, ctx[b] // bs)]
        ids = torch.tensor(full, dtype=torch.long, device=CUDA)
        # the sum of bs rows in fp32, the division
        _check(means[ids], kc[ids].double().mean(2), (bs + 1) * U * kc[ids].double().abs().mean(2))
        means[ids] = before[ids]
        assert torch.equal(means, before)


def test_key_means_reports_bad_pages():
    _status()
    kc = randn((4, 2, 16, 64), 1, torch.bfloat16, CUDA)
    means = torch.zeros(4, 2, 64, device=CUDA, dtype=torch.bfloat16)
    sa.paged_key_means(means, kc, _i32([[4, 1], [-1, 2]]), _i32([32, 16]))
    assert _status() == _lib.SA_ERR_ARG and _status() == _lib.SA_OK
    assert (means[[0, 2, 3]] == 0).all() and (means[1] != 0).any()


# ------------------------------------------------------------------ choice and decode


def _act64(a):
    root = torch.sqrt(a * a + 4)
    return torch.where(a < 0, 2 / (root - a), (a + root) / 2)


def choose64(q, means, bt, ctx, K, scale, bs):
    """[B][Hkv] lists of chosen pages."""
    B, Hq, _, D = q.shape
    Hkv = means.shape[1]
    q = q.double().view(B, Hkv, Hq // Hkv, D)
    res = []
    for b, c in enumerate(ctx):
        n = -(-c // bs)
        rows = []
        for h in range(Hkv):
            m = means[bt[b, :max(n - 1, 0)].long(), h].double()
            s = _act64(2 * scale * (q[b, h] @ m.T) - 1).square().sum(0)
            # NaN above infinity above the rest (a sort of raw NaN goes by their sign bits)
            s = s.nan_to_num(nan=1.7e308, posinf=1.6e308)
            top = torch.sort(s, descending=True, stable=True).indices[:K - 1].tolist()
            rows.append(sorted(top) + [n - 1] if n else [])
        res.append(rows)
    return res


def _attend(out, q, kc, vc, bt, ctx, chosen, scale=None):
    """out against the formula over the chosen pages.  With a = 2 s - 1 off by da (D + 8 roundings of
    the dot's terms) squareplus moves by at most da plus 2^-20 (|a| + 2) (its own root and sum), its
    square by twice that times its size, plus 2^-15 of it (the tensor-core kernel carries it as two
    16-bit halves); the sums over T tokens add (T + 64) roundings of their terms; then half a step."""
    B, Hq, _, D = q.shape
    Hkv, bs = kc.shape[1], kc.shape[2]
    G, scale = Hq // Hkv, D ** -0.5 if scale is None else scale
    for b in range(B):
        for h in range(Hkv):
            ids = chosen[b][h]
            o = out[b, h * G:(h + 1) * G].double()
            if not ids:
                assert (o == 0).all()
                continue
            T = (len(ids) - 1) * bs + ctx[b] - ids[-1] * bs
            k, v = (t[bt[b, ids].long(), h].reshape(-1, D)[:T].double() for t in (kc, vc))
            qh = q[b, h * G:(h + 1) * G, 0].double()
            a = 2 * scale * (qh @ k.T) - 1
            da = 2 * scale * (D + 8) * U * (qh.abs() @ k.abs().T) + U * (a.abs() + 1) + 2.0 ** -20 * (a.abs() + 2)
            sp = _act64(a)
            y = sp * sp
            dy = 2 * sp * da + da * da + 2.0 ** -15 * y
            R = y.sum(1, keepdim=True) + 1e-12
            ref = (y @ v) / R
            tol = (dy @ v.abs() + ref.abs() * dy.sum(1, keepdim=True) + (T + 64) * U * (y @ v.abs())) / R
            _check(out[b, h * G:(h + 1) * G], ref, tol * (1 + 2.0 ** -6))


def _cache(B, Hq, Hkv, D, mb, bs, dt, seed, spread=0.6):
    g = torch.Generator().manual_seed(seed)
    P = B * mb + 2
    kc = (randn((P, Hkv, bs, D), seed, torch.float32, CUDA)
          + spread * randn((P, Hkv, 1, D), seed + 1, torch.float32, CUDA)).to(dt)
    vc = randn((P, Hkv, bs, D), seed + 2, dt, CUDA)
    bt = torch.randperm(P, generator=g)[:B * mb].to(I32).view(B, mb).to(CUDA)
    q = randn((B, Hq, 1, D), seed + 3, dt, CUDA, 1.5)
    means = kc.float().mean(2).to(dt)
    return q, kc, vc, means, bt


CHOICES = [  # B, Hq, Hkv, D, max_blocks, bs, dtype, contexts, K
    (1, 1, 1, 32, 1, 16, torch.float16, [1], 1), (2, 8, 2, 128, 40, 16, torch.bfloat16, [640, 333], 7),
    (3, 8, 2, 128, 40, 16, torch.bfloat16, [0, 17, 601], 12), (2, 4, 4, 64, 33, 16, torch.float16, [500, 528], 4),
    (1, 6, 2, 128, 50, 8, torch.bfloat16, [395], 3), (2, 16, 2, 64, 20, 32, torch.bfloat16, [640, 100], 5),
    (1, 8, 1, 256, 150, 16, torch.bfloat16, [2391], 33), (2, 32, 8, 128, 300, 16, torch.bfloat16, [4800, 2], 64),
    (1, 5, 1, 128, 70, 16, torch.float16, [1111], 1), (2, 8, 2, 128, 9, 5, torch.bfloat16, [45, 41], 3),
    (1, 32, 2, 128, 40, 128, torch.bfloat16, [5000], 6), (2, 8, 2, 128, 10, 16, torch.bfloat16, [160, 150], 99),
]


@pytest.mark.parametrize("case", CHOICES, ids=str)
def test_choice_and_decode(case):
    B, Hq, Hkv, D, mb, bs, dt, ctx, K = case
    q, kc, vc, means, bt = _cache(B, Hq, Hkv, D, mb, bs, dt, B + mb)
    chosen = choose64(q, means, bt, ctx, min(K, mb), D ** -0.5, bs)
    pages, lens = sa.sp2norm_paged_select(q, means, bt, _i32(ctx), K, block_size=bs)
    n = min(K, mb)
    assert pages.shape == (B, Hkv, n)
    assert pages.tolist() == [[r + [-1] * (n - len(r)) for r in row] for row in chosen]
    assert lens.tolist() == [[(len(r) - 1) * bs + ctx[b] - r[-1] * bs if r else 0 for r in row]
                             for b, row in enumerate(chosen)]
    out, p2 = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), K, block_size=bs, return_pages=True)
    assert torch.equal(p2, pages) and out.dtype == torch.bfloat16 and out.shape == (B, Hq, D)
    _attend(out, q, kc, vc, bt, ctx, chosen)
    alone = sa.sp2norm_sparse_paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, means, bt.long(),
                                              torch.tensor(ctx, device=CUDA), K, block_size=bs)
    assert torch.equal(alone, out)
    if K >= mb:  # every page: what the dense decode gives
        dense = sa.sp2norm_paged_attention(q, kc, vc, bt, _i32(ctx), block_size=bs)
        _attend(dense, q, kc, vc, bt, ctx, chosen)


def test_choice_of_ties_and_odd_values():
    B, Hq, Hkv, D, mb, bs = 1, 4, 1, 64, 600, 16
    q, kc, vc, means, bt = _cache(B, Hq, Hkv, D, mb, bs, torch.bfloat16, 3)
    ctx = [mb * bs]
    same = means.clone()
    same[:] = means[:1]  # every page alike: the lowest are taken
    pages, _ = sa.sp2norm_paged_select(q, same, bt, _i32(ctx), 50)
    assert pages[0, 0].tolist() == list(range(49)) + [mb - 1]
    two = same.clone()  # two values: the higher ones first, then the lowest pages
    hot = [590, 77, 401]
    two[bt[0, hot].long()] = 3 * q[0, :, 0].float().mean(0).to(torch.bfloat16)
    pages, _ = sa.sp2norm_paged_select(q, two, bt, _i32(ctx), 10)
    assert pages[0, 0].tolist() == sorted(hot + list(range(6))) + [mb - 1]
    odd = means.clone()
    odd[bt[0, 500].long(), 0, 3] = math.nan
    odd[bt[0, 300].long(), 0, :] = q[0, 0, 0] * math.inf  # +inf where q is positive: the dot is +inf
    want = choose64(q, odd, bt, ctx, 20, D ** -0.5, bs)
    pages, _ = sa.sp2norm_paged_select(q, odd, bt, _i32(ctx), 20)
    assert pages[0].tolist() == want[0] and 500 in want[0][0]
    scale = 0.37
    want = choose64(q, means, bt, ctx, 20, scale, bs)
    out, pages = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), 20, scale=scale, return_pages=True)
    assert pages[0].tolist() == want[0]
    _attend(out, q, kc, vc, bt, ctx, want, scale)


@pytest.mark.parametrize("mb,K", [(500, 40), (3000, 200)])  # scores kept in registers, and read again
def test_choice_among_pages_that_32_bits_cannot_tell_apart(mb, K):
    """Mean keys that differ in single last bits of single channels: many real scores inside one fp32 rounding."""
    q, kc, vc, means, bt = _cache(1, 8, 2, 128, mb, 16, torch.bfloat16, 21)
    g = torch.Generator().manual_seed(3)
    for share in (0.05, 0.3, 1.0):  # of the pages: a handful at the border, then all of them
        near = means.clone()
        alike = torch.randperm(mb - 1, generator=g)[:max(2, int(share * (mb - 1)))].to(CUDA)
        score = choose64(q, means, bt, [mb * 16], K, 128 ** -0.5, 16)[0][0][K // 2]  # a page in the middle of the chosen
        near[bt[0, alike].long()] = means[bt[0, score].long()]
        for p in alike.tolist()[::2]:
            c = int(torch.randint(0, 128, (1,), generator=g))
            bits = near[bt[0, p].long(), :, c].view(torch.int16)
            near[bt[0, p].long(), :, c] = (bits ^ 1).view(torch.bfloat16)
        want = choose64(q, near, bt, [mb * 16], K, 128 ** -0.5, 16)
        pages, _ = sa.sp2norm_paged_select(q, near, bt, _i32([mb * 16]), K)
        assert pages[0].tolist() == want[0]


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1.0, 1e4, 1e20, 1e30, -0.3])
def test_choice_at_odd_scales(scale):
    """Scores that are all alike, far negative, or past fp32: the choice is the 64-bit one."""
    for dt in (torch.bfloat16, torch.float16):
        q, kc, vc, means, bt = _cache(2, 6, 2, 64, 700, 16, dt, 22)
        ctx = [700 * 16 - 5, 3000]
        want = choose64(q, means, bt, ctx, 33, scale, 16)
        pages, _ = sa.sp2norm_paged_select(q, means, bt, _i32(ctx), 33, scale=scale)
        assert pages.tolist() == [[r + [-1] * (33 - len(r)) for r in row] for row in want]


def test_choice_of_a_long_context():
    """65536 pages, more than one staging of everything; far negative scores too."""
    q, kc, vc, means, bt = _cache(1, 4, 1, 128, 65536, 16, torch.bfloat16, 5, spread=3.0)
    q *= 4
    ctx = [65536 * 16 - 3]
    want = choose64(q, means, bt, ctx, 1000, 128 ** -0.5, 16)
    out, pages = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), 1000, return_pages=True)
    assert pages[0].tolist() == want[0]
    _attend(out, q, kc, vc, bt, ctx, want)


@pytest.mark.parametrize("K", [9000, 8999, 8300])
def test_choice_of_nearly_all_of_a_long_table(K):
    """Every page taken, or all but a few, among more than a block keeps in registers."""
    q, kc, vc, means, bt = _cache(2, 2, 1, 32, 9000, 1, torch.float16, 15)
    ctx = [9000, 8301]
    want = choose64(q, means, bt, ctx, K, 32 ** -0.5, 1)
    out, pages = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), K, block_size=1, return_pages=True)
    assert pages.tolist() == [[r + [-1] * (K - len(r)) for r in row] for row in want]
    _attend(out, q, kc, vc, bt, ctx, want)


def test_rows_past_the_context_do_not_matter():
    """NaN in the cache behind the last token and in unused pages, -1 in the table behind it."""
    q, kc, vc, means, bt = _cache(2, 8, 2, 128, 12, 16, torch.bfloat16, 8)
    ctx = [100, 23]
    a = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), 4)
    used = torch.zeros(kc.shape[0], 16, dtype=torch.bool, device=CUDA)
    for b, c in enumerate(ctx):
        for t in range(c):
            used[bt[b, t // 16].long(), t % 16] = True
    kc.masked_fill_(~used[:, None, :, None], math.nan)
    vc.masked_fill_(~used[:, None, :, None], math.nan)
    means.masked_fill_(~used.all(1)[:, None, None], math.nan)
    for b, c in enumerate(ctx):
        bt[b, -(-c // 16):] = -1
    _status()
    assert torch.equal(a, sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), 4))
    assert _status() == _lib.SA_OK


def test_lengths_outside_the_table_are_clamped():
    q, kc, vc, means, bt = _cache(3, 4, 2, 128, 6, 16, torch.bfloat16, 12)
    far, cut = _i32([1000, -5, 2 ** 31 - 1]), _i32([96, 0, 96])
    a, b = (sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, c, 3, return_pages=True) for c in (far, cut))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and (a[0][1] == 0).all() and (a[1][1] == -1).all()
    m0, m1 = torch.zeros_like(means), torch.zeros_like(means)
    sa.paged_key_means(m0, kc, bt, far, start_lens=_i32([-9, -9, 2 ** 31 - 1]))
    sa.paged_key_means(m1, kc, bt, _i32([96, 0, 0]))
    assert torch.equal(m0, m1)


def test_bad_pages_are_read_as_page_zero_and_reported():
    q, kc, vc, means, bt = _cache(1, 4, 2, 128, 8, 16, torch.bfloat16, 9)
    good = bt.clone()
    good[0, 2] = 0
    bt[0, 2] = kc.shape[0]
    _status()
    o, p = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32([128]), 4, return_pages=True)
    assert _status() == _lib.SA_ERR_ARG
    og, pg = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, good, _i32([128]), 4, return_pages=True)
    assert torch.equal(p, pg) and torch.equal(o, og)
    assert _status() == _lib.SA_OK


def test_empty_batches():
    q, kc, vc, means, bt = _cache(2, 4, 2, 64, 4, 16, torch.bfloat16, 9)
    cl = _i32([5, 9])
    assert sa.sp2norm_sparse_paged_attention(q[:0], kc, vc, means, bt[:0], cl[:0], 2).shape == (0, 4, 64)
    assert sa.sp2norm_paged_select(q[:0], means, bt[:0], cl[:0], 2)[0].shape == (0, 2, 2)
    o, p = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt[:, :0], cl, 2, return_pages=True)
    assert (o == 0).all() and p.shape == (2, 2, 0)
    o, p = sa.sp2norm_sparse_paged_attention(q, kc[:0], vc[:0], means[:0], bt, cl, 2, return_pages=True)
    assert (o == 0).all() and (p == -1).all()
    before = means.clone()
    assert torch.equal(sa.paged_key_means(means, kc, bt[:0], cl[:0]), before)


# ------------------------------------------------------------------ together


def _graph(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    gc.collect()
    gc.disable()
    try:
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            out = fn()
    finally:
        gc.enable()
    return g, out


def test_two_graphs_at_once_on_two_streams():
    """Each captured call has a workspace of its own: replays may overlap."""
    sets = [_cache(2, 8, 2, 128, 300, 16, torch.bfloat16, s) for s in (1, 2)]
    cl = _i32([4700, 3100])
    calls = [lambda s=s: sa.sp2norm_sparse_paged_attention(s[0], s[1], s[2], s[3], s[4], cl, 40) for s in sets]
    want = [c() for c in calls]
    graphs = [_graph(c) for c in calls]
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)


def test_a_serving_run():
    """Requests come, grow and go; every step is slots -> append -> mean keys -> decode, the decode
    checked against the formula on the sequence's own raw keys and values."""
    Hq, Hkv, D, bs, mb, B, P = 8, 2, 128, 16, 16, 5, 60
    dt, K = torch.bfloat16, 4
    kc, vc = (torch.full((P, Hkv, bs, D), math.nan, device=CUDA, dtype=dt) for _ in range(2))
    means = torch.full((P, Hkv, D), math.nan, device=CUDA, dtype=dt)
    table = torch.full((B, mb), -1, dtype=I32, device=CUDA)
    ctx, head = torch.zeros(B, dtype=I32, device=CUDA), _i32([0])
    pool = torch.randperm(P, generator=torch.Generator().manual_seed(1)).to(I32).to(CUDA)
    cos, sin = _angles(mb * bs, D)
    wq, wk = (1 + randn((D,), i, torch.float32, CUDA, 0.3) for i in (1, 2))
    seqs = [[] for _ in range(B)]  # per request: (k rows as cached, v rows)
    g = torch.Generator().manual_seed(2)
    _status()
    for step in range(12):
        if step in (5, 9):  # two requests end; others take their places
            done = torch.zeros(B, dtype=torch.bool)
            done[[1, 3]] = True
            ctx, head = sa.paged_release_pages(table, ctx, done.to(CUDA), pool, head, block_size=bs)
            for b in (1, 3):
                seqs[b] = []
        new = [int(torch.randint(1, 60, (1,), generator=g)) if not seqs[b] else 1 for b in range(B)]
        N = sum(new) + 3  # a padded batch
        q, k, v = _append_inputs(N, Hq, Hkv, D, dt, 100 + step)
        s = sa.paged_assign_slots(table, ctx, _i32(new), pool, head, N, block_size=bs)
        assert (s.slot_mapping >= 0).sum() == sum(new) and (s.slot_mapping[sum(new):] == -1).all()
        qo = sa.qk_norm_rope_paged_append(q, k, v, kc, vc, s.slot_mapping, cos, sin, positions=s.positions,
                                          q_weight=wq, k_weight=wk)
        assert (qo[sum(new):] == 0).all()
        sa.paged_key_means(means, kc, table, s.context_lens, start_lens=ctx)
        last = s.cu_seqlens[1:].long() - 1  # each request's newest token asks
        qd = qo[last][:, :, None]
        out, pages = sa.sp2norm_sparse_paged_attention(qd, kc, vc, means, table, s.context_lens, K, block_size=bs,
                                                       return_pages=True)
        cu = s.cu_seqlens.tolist()
        yk, tk = _ref64(k.transpose(0, 1)[None], wk, cos, sin, s.positions[None].long(), 1e-6)
        for b in range(B):
            seqs[b] += [(yk[0, :, i], tk[0, :, i], v[i]) for i in range(cu[b], cu[b + 1])]
        lens = [len(x) for x in seqs]
        assert s.context_lens.tolist() == lens
        owned = [p for b in range(B) for p in table[b, :-(-lens[b] // bs)].tolist()]
        assert len(set(owned)) == len(owned) and not set(owned) & set(pool[s.free_head.item():].tolist())
        for b in range(B):  # the cache holds the sequence's own rows, in order
            t = torch.arange(lens[b], device=CUDA)
            at = table[b, t // bs].long()
            _check(kc[at, :, t % bs], torch.stack([x[0] for x in seqs[b]]), torch.stack([x[1] for x in seqs[b]]))
            assert torch.equal(vc[at, :, t % bs], torch.stack([x[2] for x in seqs[b]]))
            full = table[b, :lens[b] // bs].long()
            _check(means[full], kc[full].double().mean(2), 17 * U * kc[full].double().abs().mean(2))
        chosen = choose64(qd, means, table, lens, K, D ** -0.5, bs)
        assert pages.tolist() == [[r + [-1] * (K - len(r)) for r in row] for row in chosen]
        _attend(out, qd, kc, vc, table, lens, chosen)
        ctx, head = s.context_lens, s.free_head
    assert _status() == _lib.SA_OK


def test_a_captured_decode_step():
    """The four calls of a decode step in one graph, replayed over page borders; the lengths live in
    buffers that the graph itself advances."""
    Hq, Hkv, D, bs, mb, B, P = 8, 2, 128, 16, 12, 4, 48
    dt = torch.bfloat16
    cos, sin = _angles(mb * bs, D)
    q, k, v = _append_inputs(B, Hq, Hkv, D, dt, 1)
    ones = torch.ones(B, dtype=I32, device=CUDA)

    def fresh():
        table = torch.full((B, mb), -1, dtype=I32, device=CUDA)
        pool = torch.arange(P, dtype=I32, device=CUDA)
        ctx = _i32([15, 40, 31, 1])
        s = sa.paged_assign_slots(table, torch.zeros_like(ctx), ctx, pool, _i32([0]), 87, block_size=bs)
        kc, vc = (randn((P, Hkv, bs, D), i, dt, CUDA) for i in (3, 4))
        means = torch.zeros(P, Hkv, D, device=CUDA, dtype=dt)
        sa.paged_key_means(means, kc, table, ctx)
        return [table, pool, ctx, s.free_head.clone(), kc, vc, means]

    def step(st):
        table, pool, ctx, head, kc, vc, means = st
        s = sa.paged_assign_slots(table, ctx, ones, pool, head, B, block_size=bs)
        qo = sa.qk_norm_rope_paged_append(q, k, v, kc, vc, s.slot_mapping, cos, sin, positions=s.positions)
        sa.paged_key_means(means, kc, table, s.context_lens, start_lens=ctx)
        o = sa.sp2norm_sparse_paged_attention(qo[:, :, None], kc, vc, means, table, s.context_lens, 2, block_size=bs)
        ctx.copy_(s.context_lens)
        head.copy_(s.free_head)
        return o

    eager, st = fresh(), fresh()
    gr, out = _graph(lambda: step(st))  # warm-up advances st by one step; capturing runs nothing
    step(eager)
    for _ in range(20):
        gr.replay()
        want = step(eager)
        assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(st, eager))


@pytest.mark.parametrize("Hq,Hkv,D,sizes", [(2, 2, 32, (16, 8, 16)), (4, 1, 32, (16, 8, 1, 16)),
                                            (2, 2, 128, (16, 20, 16)), (3, 1, 256, (16, 5, 16)), (8, 1, 64, (64, 8, 64))])
def test_decode_of_several_page_sizes_in_one_process(Hq, Hkv, D, sizes):
    """A cache of smaller pages in between does not take the larger ones' shared memory away."""
    for dt in (torch.float16, torch.bfloat16):
        for bs in sizes:
            mb = 320 // bs
            q, kc, vc, means, bt = _cache(2, Hq, Hkv, D, mb, bs, dt, 40 + bs)
            ctx = [mb * bs, mb * bs - bs // 2 - 1]
            every = [[list(range(-(-c // bs)))] * Hkv for c in ctx]
            _attend(sa.sp2norm_paged_attention(q, kc, vc, bt, _i32(ctx), block_size=bs), q, kc, vc, bt, ctx, every)
            out = sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), mb, block_size=bs)
            _attend(out, q, kc, vc, bt, ctx, every)


# ------------------------------------------------------------------ odd calls


def test_append_copies_infinities_without_touching_their_neighbours():
    """An infinity in channel R + n of token n's query and key, without a norm: copied, and nothing else changes."""
    R, D, bs = 16, 64, 8
    N = D - R
    cos, sin = _angles(N, R)
    n = torch.arange(N, device=CUDA)
    for dt in (torch.bfloat16, torch.float16):
        q, k, v = (t.contiguous() for t in _append_inputs(N, 4, 2, D, dt, 31))
        for value in (math.inf, math.nan):
            res = []
            for bad in (False, True):
                kc, vc = (torch.zeros(N // bs, 2, bs, D, device=CUDA, dtype=dt) for _ in range(2))
                if bad:
                    q[n, :, R + n] = value
                    k[n, :, R + n] = value
                res.append((sa.qk_norm_rope_paged_append(q, k, v, kc, vc, n, cos, sin, positions=n, eps=None),
                            kc.transpose(1, 2).reshape(N, 2, D), vc))
            for x, got, clean in ((q, res[1][0], res[0][0]), (k, res[1][1], res[0][1])):
                assert torch.equal(got[..., R:].nan_to_num(7.0), x[..., R:].nan_to_num(7.0))
                assert torch.equal(got[..., :R], clean[..., :R])
            assert torch.equal(res[0][2], res[1][2])
            q, k, v = (t.contiguous() for t in _append_inputs(N, 4, 2, D, dt, 31))


def test_large_batches_from_two_threads():
    """Two host threads whose batches need different shared memory: no launch is refused."""
    lib, bs, bad, start = _lib.load(), 16, [], threading.Barrier(2)
    p = lambda t: t.data_ptr()  # noqa: E731

    def work(B):
        table = torch.arange(B, device=CUDA, dtype=I32)[:, None].contiguous()
        own, full, ones = (torch.full((B, 1), n, device=CUDA, dtype=I32) for n in (-1, 16, 1))
        pool, done = torch.zeros(B, device=CUDA, dtype=I32), torch.ones(B, device=CUDA, dtype=torch.bool)
        head, zero, none = _i32([B]), _i32([0]), torch.zeros(B, device=CUDA, dtype=I32)
        slots = torch.zeros(B, device=CUDA, dtype=torch.int64)
        pos, cu, ctx, ctx2 = (torch.zeros(B + 4, device=CUDA, dtype=I32) for _ in range(4))
        h1, h2 = _i32([0]), _i32([0])
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        assign = (p(own), 1, p(none), p(ones), p(table), B, p(zero), p(slots), p(pos), p(cu), p(ctx), p(h1), B, B, 1, bs,
                  st.cuda_stream)
        release = (p(table), 1, p(full), p(done), p(pool), B, p(head), p(ctx2), p(h2), B, 1, bs, st.cuda_stream)
        start.wait()
        for _ in range(3000):
            bad.extend(r for r in (lib.sa_paged_assign_slots(*assign), lib.sa_paged_release_pages(*release)) if r != 0)
        st.synchronize()
        if not (torch.equal(pool, table[:, 0]) and h2.item() == 0 and h1.item() == B
                and torch.equal(slots, torch.arange(B, device=CUDA) * bs)):
            bad.append("outputs")

    threads = [threading.Thread(target=work, args=(B,)) for B in (16384, 7000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, (len(bad), bad[:3])


def test_append_without_queries_reports_slots_past_the_cache():
    _status()
    kc, vc = (torch.zeros(2, 1, 4, 64, device=CUDA, dtype=torch.bfloat16) for _ in range(2))
    q, k, v = _append_inputs(3, 0, 1, 64, torch.bfloat16, 2)
    call = lambda s: sa.qk_norm_rope_paged_append(q, k, v, kc, vc, torch.tensor(s, device=CUDA))  # noqa: E731
    assert call([8, 2, 1 << 40]).shape == (3, 0, 64)
    assert _status() == _lib.SA_ERR_ARG
    assert torch.equal(vc[0, 0, 2], v[1, 0]) and vc.count_nonzero() == v[1].count_nonzero()
    call([-1, 2, -1 << 40])  # padding is no error
    assert _status() == _lib.SA_OK


def test_64_bit_integers_are_not_cut_to_32():
    """Lengths and pages outside 32 bits are as far out as they say, not their last 32 bits."""
    q, kc, vc, means, bt = _cache(2, 4, 2, 128, 6, 16, torch.bfloat16, 12)
    far, cut = torch.tensor([2 ** 32 + 5, -2 ** 32 + 40], device=CUDA), _i32([96, 0])
    a, b = (sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, c, 3, return_pages=True) for c in (far, cut))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    m = [torch.zeros_like(means) for _ in range(2)]
    for n, (ctx, start) in enumerate(((far, torch.tensor([-2 ** 33 + 48, 0], device=CUDA)), (cut, _i32([0, 0])))):
        sa.paged_key_means(m[n], kc, bt, ctx, start_lens=start)
    assert torch.equal(*m) and m[0].count_nonzero() > 0
    _status()
    wide = bt.long()
    wide[0, 2] += 2 ** 32
    sa.sp2norm_sparse_paged_attention(q, kc, vc, means, wide, cut, 3)
    assert _status() == _lib.SA_ERR_ARG and _status() == _lib.SA_OK
    # slots: a request longer than its row, more new tokens than fit, a list's head past its end
    t = [_i32([[3, -1], [-1, -1]]) for _ in range(2)]
    big = 2 ** 32
    args = [(torch.tensor([big + 3, 0], device=CUDA), torch.tensor([1, big + 20], device=CUDA)),
            (_i32([32, 0]), _i32([1, 2 ** 31 - 1]))]
    s = [sa.paged_assign_slots(x, *y, _i32([7, 8]), _i32([0]), 50) for x, y in zip(t, args)]
    assert all(torch.equal(x, y) for x, y in zip(*s)) and torch.equal(*t) and s[0].context_lens.tolist() == [32, 32]
    s = sa.paged_assign_slots(t[0], _i32([3, 0]), _i32([20, 0]), _i32([7, 8]), torch.tensor([big], device=CUDA), 20)
    assert s.free_head.item() == 2 and s.context_lens.tolist() == [16, 0]


def test_pages_that_are_none_are_reported():
    """A negative page, in a row's held part or in the list: its tokens have no slot, and it is said."""
    _status()
    t = _i32([[3, -1], [-5, -1]])
    s = sa.paged_assign_slots(t, _i32([16, 3]), _i32([2, 2]), _i32([6]), _i32([0]), 4)
    assert s.slot_mapping.tolist() == [96, 97, -1, -1]
    assert _status() == _lib.SA_ERR_ARG
    s = sa.paged_assign_slots(_i32([[-1]]), _i32([0]), _i32([1]), _i32([-2]), _i32([0]), 1)
    assert s.slot_mapping.tolist() == [-1] and _status() == _lib.SA_ERR_ARG
    free = _i32([0, 1, 2])
    sa.paged_release_pages(_i32([[7, -1]]), _i32([20]), torch.tensor([True], device=CUDA), free, _i32([3]))
    assert _status() == _lib.SA_ERR_ARG
    # rows and lists whose unused entries are negative are ordinary
    t = _i32([[3, -1], [-1, -1]])
    sa.paged_assign_slots(t, _i32([15, 0]), _i32([1, 1]), _i32([-9, 6, -9]), _i32([1]), 5)
    sa.paged_release_pages(t, _i32([16, 0]), torch.tensor([True, True], device=CUDA), free, _i32([3]))
    assert _status() == _lib.SA_OK


def test_c_abi_append_without_a_norm_leaves_the_weights_out():
    """normalize = 0 is n = x, whatever weights come with it."""
    lib, N, Hq, Hkv, D, bs = _lib.load(), 5, 2, 1, 64, 8
    q, k, v = (t.contiguous() for t in _append_inputs(N, Hq, Hkv, D, torch.bfloat16, 3))
    kc, vc = (torch.zeros(1, Hkv, bs, D, device=CUDA, dtype=torch.bfloat16) for _ in range(2))
    w, out, slots = torch.full((D,), 3.0, device=CUDA), torch.zeros_like(q), torch.arange(N, device=CUDA)
    s = [(ctypes.c_int64 * 3)(H * D, D, 1) for H in (Hq, Hkv, Hkv)]
    p = lambda t: t.data_ptr()  # noqa: E731
    assert lib.sa_qk_norm_rope_paged_append(p(q), p(k), p(v), p(out), p(kc), p(vc), p(slots), p(w), p(w), _lib.SA_F32, None,
                                            None, 0, None, 0, 0, N, Hq, Hkv, D, 0, 1, bs, *s, 1e-6, 0, _lib.SA_BF16,
                                            None) == _lib.SA_OK
    torch.cuda.synchronize()
    assert torch.equal(out, q) and torch.equal(kc[0, :, :N].transpose(0, 1), k)


def test_sparse_decode_repeats_bitwise():
    """The same call on other memory, over workspaces of other contents, on another stream."""
    ctx = [8192, 5003, 7777, 17, 0, 6001, 8191, 5120]
    first = None
    for run in range(6):
        filler = torch.full((64 << 20,), (0x7F, 0xFF, 0x00)[run % 3], device=CUDA, dtype=torch.uint8)
        del filler  # (what the next tensors and workspaces are made of)
        q, kc, vc, means, bt = _cache(8, 32, 8, 128, 512, 16, torch.bfloat16, 77)
        with torch.cuda.stream(torch.cuda.Stream() if run % 2 else torch.cuda.current_stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            got = [sa.sp2norm_sparse_paged_attention(q, kc, vc, means, bt, _i32(ctx), 64, return_pages=True)
                   for _ in range(20)]
        torch.cuda.synchronize()
        first = got[0] if first is None else first
        for out, pages in got:
            assert torch.equal(out, first[0]) and torch.equal(pages, first[1])


def test_key_means_of_a_mixed_batch():
    """One new prompt among sequences of one token: only its full pages, and theirs that the token fills."""
    Hkv, D, bs, mb, B = 8, 128, 16, 512, 64
    P = 1300
    kc = randn((P, Hkv, bs, D), 1, torch.bfloat16, CUDA)
    bt = torch.full((B, mb), -1, dtype=I32, device=CUDA)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(3)).to(I32).to(CUDA)
    ctx, start, at = [], [], 0
    for b in range(B):
        n = 8191 if b == 17 else 5 * b + 1  # those of 16, 96, .. tokens end on a page
        ctx.append(n)
        start.append(0 if b == 17 else n - 1)
        p = -(-n // bs)
        bt[b, :p] = order[at:at + p]
        at += p
    assert at <= P
    means = randn((P, Hkv, D), 2, torch.bfloat16, CUDA)
    before = means.clone()
    sa.paged_key_means(means, kc, bt, _i32(ctx), start_lens=_i32(start))
    ids = torch.cat([bt[b, s // bs:c // bs] for b, (s, c) in enumerate(zip(start, ctx))]).long()
    assert ids.numel() > 511
    _check(means[ids], kc[ids].double().mean(2), (bs + 1) * U * kc[ids].double().abs().mean(2))
    means[ids] = before[ids]
    assert torch.equal(means, before)


def test_narrowing_of_64_bit_integers():
    from smooth_attn import paged_cache as P

    edge = [0, 1, -1, -2, 2 ** 31 - 1, 2 ** 31, -2 ** 31, 2 ** 32, 2 ** 32 + 7, -2 ** 32 + 7, 2 ** 63 - 1, -2 ** 63, 12345]
    for n in (0, 1, len(edge), 300_001):
        wide = torch.tensor((edge * (n // len(edge) + 1))[:n], dtype=torch.int64, device=CUDA)
        for t in (wide, torch.stack((wide, wide), 1)[:, 1]):  # contiguous, and not
            got = P._int32("t", t, (n,), t)
            assert got.dtype == I32 and torch.equal(got.long(), wide.clamp(-1, 2 ** 31 - 1))
    assert torch.equal(P._int32("t", wide[:6].view(2, 3), (2, 3), wide), wide[:6].view(2, 3).clamp(-1, 2 ** 31 - 1).to(I32))
