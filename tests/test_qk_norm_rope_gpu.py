"""Head norm with rotation (``qk_norm_rope``) and its backward against the
formula in 64 bits, the attention that trains through it, and what it must
leave alone.

Tolerances count roundings.  y is rounded once to its type (at most half a
step, eps / 2 of the value; half the smallest step below the type's normal
range); before that every fp32 operation adds at most 2^-24 of its result.
A row's sum of squares has 16 terms a lane and at most 4 exchange steps, so
r = rsqrt(mean + eps) is within 16 steps of 2^-24 (half the sum's 20, two
for rsqrtf, the rest for the division and eps); two products, one more and a
subtraction for the rotation give 24 * 2^-24 of |n1| + |n2|.  dx and the
weights' gradients are bounded the same way by their terms' magnitudes (see
each check)."""

import ctypes
import gc
import math

import pytest
import torch

import smooth_attn as sa
from smooth_attn import _lib
from oracle import sa_oracle as O
from tests._util import check_bf16_grads, np32, randn

pytestmark = pytest.mark.gpu
CUDA = "cuda"
U = 2.0 ** -24  # one fp32 rounding


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA required")


def _angles(rows, R, dtype=torch.float32):
    cos, sin = sa.precompute_rope_cos_sin(R, rows, device=CUDA)
    return cos.to(dtype), sin.to(dtype)


def _rot(x, cos, sin):
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]), -1)


def _amp(x, R):
    """|x1| + |x2| of each rotated pair, |x| elsewhere."""
    h = R // 2
    p = x[..., :h].abs() + x[..., h:R].abs()
    return torch.cat((p, p, x[..., R:].abs()), -1)


def _half_step(ref, dtype):
    fi = torch.finfo(dtype)
    return torch.clamp(ref.abs() * fi.eps / 2, min=fi.smallest_normal * fi.eps / 2)


def _ref64(x, w, cos, sin, pos, eps, dy=None):
    """(y, tol_y, dx, tol_dx, dw, tol_dw) in 64 bits; tolerances without the final rounding."""
    x = x.double()
    R = 0 if cos is None else 2 * cos.shape[1]
    c, s = (None, None) if cos is None else (t.double()[pos.long()][:, None] for t in (cos, sin))
    w = torch.ones(x.shape[-1], device=x.device, dtype=torch.float64) if w is None else w.double()
    r = torch.ones_like(x[..., :1]) if eps is None else torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r * (1 if eps is None else w)
    y = n if R == 0 else _rot(n, c, s)
    tol = 24 * U * (n.abs() if R == 0 else _amp(n, R))
    if dy is None:
        return y, tol
    dy = dy.double()
    dn = dy if R == 0 else _rot(dy, c, -s)
    g = dy.abs() if R == 0 else _amp(dy, R)
    if eps is None:
        return y, tol, dn, 8 * U * g, None, None
    gw = dn * w
    dx = r * (gw - x * r * r * (gw * x).mean(-1, keepdim=True))
    # r off by 16 U, cubed; the mean's sum by 20 U of its terms' magnitudes
    tol_dx = 80 * U * r * (g * w.abs() + x.abs() * r * r * (g * w.abs() * x.abs()).mean(-1, keepdim=True))
    terms = (g * x * r).abs()
    # a lane adds the rows of its tasks one by one (8 at these sizes), then 5 exchanges, 8 warps, and at
    # most 2 * 148 / 32 + 5 block sums: under 64 additions; 24 for each term
    return y, tol, dx, tol_dx, (dn * x * r).sum((0, 1, 2)), 88 * U * terms.sum((0, 1, 2))


def _check(got, ref, tol):
    assert got.shape == ref.shape
    err = (got.double() - ref).abs() - tol - _half_step(ref, got.dtype)
    assert not got.isnan().any() and (err <= 0).all(), f"worst excess {err.max().item():.3g}"


CASES = [  # B, Hq, Hkv, T, D, R, dtype, weights, norm, positions
    (1, 1, 1, 1, 16, 16, torch.float32, torch.float32, True, "none"),
    (2, 3, 1, 5, 32, 32, torch.float16, torch.float16, True, "none"),
    (1, 4, 2, 67, 64, 32, torch.bfloat16, torch.bfloat16, True, "row32"),
    (2, 32, 8, 33, 128, 128, torch.bfloat16, torch.float32, True, "batch64"),
    (3, 5, 5, 19, 80, 16, torch.float32, None, True, "batch32"),
    (2, 2, 1, 130, 112, 112, torch.float16, torch.bfloat16, True, "row64"),
    (1, 9, 3, 31, 256, 64, torch.bfloat16, torch.float16, True, "one"),
    (1, 9, 3, 31, 240, 240, torch.float32, torch.float32, True, "none"),
    (2, 4, 2, 40, 128, 128, torch.bfloat16, None, False, "batch32"),   # rotation alone
    (2, 4, 2, 40, 128, 0, torch.bfloat16, torch.bfloat16, True, "none"),  # norm alone
    (8, 32, 8, 1, 128, 128, torch.bfloat16, torch.bfloat16, True, "batch32"),  # one new token
]


def _make(case, seed=0, scale=1.0):
    B, Hq, Hkv, T, D, R, dt, wdt, norm, ps = case
    q, k = randn((B, Hq, T, D), seed + 1, dt, CUDA, scale), randn((B, Hkv, T, D), seed + 2, dt, CUDA, scale)
    dq, dk = randn(q.shape, seed + 3, dt, CUDA), randn(k.shape, seed + 4, dt, CUDA)
    wq, wk = (None, None) if wdt is None else ((1 + randn((D,), seed + i, torch.float32, CUDA, 0.3)).to(wdt)
                                               for i in (5, 6))
    cos, sin = (None, None) if R == 0 else _angles(T + 300, R)
    g = torch.Generator().manual_seed(seed + 7)
    n = {"row32": (T,), "row64": (T,), "one": (1, T), "batch32": (B, T), "batch64": (B, T)}.get(ps)
    pos = None if n is None else torch.randint(0, T + 300, n, generator=g).to(
        torch.int64 if ps.endswith("64") else torch.int32).to(CUDA)
    full = torch.arange(T, device=CUDA).expand(B, T) if pos is None else pos.expand(B, T)
    return q, k, dq, dk, wq, wk, cos, sin, pos, full, (1e-6 if norm else None)


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}H{c[1]}_{c[2]}T{c[3]}D{c[4]}R{c[5]}{c[9]}")
@pytest.mark.parametrize("layout", ["bhtd", "bthd", "off"])
def test_matches_the_formula(case, layout):
    q, k, dq, dk, wq, wk, cos, sin, pos, full, eps = _make(case)
    if layout == "bthd":
        q, k, dq, dk = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, dq, dk))
    elif layout == "off":  # rows and base off a 16-byte boundary: taken through a copy
        def off(t):
            b = torch.zeros(t.numel() // t.shape[-1] * (t.shape[-1] + 1) + 1, device=CUDA, dtype=t.dtype)
            v = b[1:].view(*t.shape[:-1], t.shape[-1] + 1)[..., :-1]
            return v.copy_(t)
        q, k, dq, dk = (off(t) for t in (q, k, dq, dk))
    req = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, wq, wk)]
    yq, yk = sa.qk_norm_rope(req[0], req[1], cos, sin, q_weight=req[2], k_weight=req[3], eps=eps, positions=pos)
    assert yq.dtype == q.dtype
    for t in (yq, yk):  # dense, in the inputs' order of dims
        assert (t.transpose(1, 2) if layout == "bthd" else t).is_contiguous()
    ins = [t for t in req if t is not None]
    grads = dict(zip([id(t) for t in ins], torch.autograd.grad((yq, yk), ins, (dq, dk))))
    assert grads[id(req[0])].stride() == yq.stride() and grads[id(req[1])].stride() == yk.stride()
    for x, w, xr, wr, y, dy in ((q, wq, req[0], req[2], yq, dq), (k, wk, req[1], req[3], yk, dk)):
        ref = _ref64(x, w, cos, sin, full, eps, dy)
        _check(y.detach(), ref[0], ref[1])
        _check(grads[id(xr)], ref[2], ref[3])
        if w is not None and eps is not None:
            assert grads[id(wr)].dtype == w.dtype
            _check(grads[id(wr)], ref[4], ref[5])


@pytest.mark.parametrize("cs", [torch.bfloat16, torch.float16, torch.float64])
def test_table_types(cs):
    q, k, *_ = _make(CASES[3])
    cos, sin = _angles(40, 128, cs)
    y, _ = sa.qk_norm_rope(q, k, cos, sin)
    ref = _ref64(q, None, cos.float(), sin.float(), torch.arange(33, device=CUDA).expand(2, 33), 1e-6)
    _check(y, *ref)


@pytest.mark.parametrize("B,Hq,Hkv,T,D,R,dt,ps", [
    (2, 16, 4, 2100, 128, 128, torch.bfloat16, "batch32"),
    (3, 32, 8, 3001, 128, 128, torch.bfloat16, "batch64"),  # many whole rows in full units: fewer, deeper warps
    (2, 64, 16, 3801, 64, 32, torch.float16, "row32"),
    (2, 24, 8, 5003, 64, 32, torch.float16, "none"),
    (2, 20, 9, 4099, 80, 80, torch.bfloat16, "row32"),  # heads that units do not divide
    (1, 8, 16, 5001, 128, 64, torch.float32, "row64"),
])
def test_gradient_of_a_larger_problem_repeats_bitwise(B, Hq, Hkv, T, D, R, dt, ps):
    """Many blocks, both sides; the weights' sums join in a fixed order."""
    q, k, dq, dk, wq, wk, cos, sin, pos, full, eps = _make((B, Hq, Hkv, T, D, R, dt, torch.float32, True, ps))
    res = []
    for _ in range(2):
        ins = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        y = sa.qk_norm_rope(ins[0], ins[1], cos, sin, q_weight=ins[2], k_weight=ins[3], positions=pos)
        res.append(torch.autograd.grad(y, ins, (dq, dk)))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    for x, w, dx, dw, dy in ((q, wq, res[0][0], res[0][2], dq), (k, wk, res[0][1], res[0][3], dk)):
        ref = _ref64(x, w, cos, sin, full, eps, dy)
        _check(dx, ref[2], ref[3])
        # a lane's chain: all rows over the warps of its side (a ninth of 1700 at least) and the tokens of a
        # warp (2 at least), doubled for uneven shares
        chain = 64 + 2 * (x.numel() // D) // (190 * 2)
        _check(dw, ref[4], ref[5] * (24 + chain) / 88)
    y = sa.qk_norm_rope(q, k, cos, sin, q_weight=wq, k_weight=wk, positions=pos)
    for x, w, o in ((q, wq, y[0]), (k, wk, y[1])):
        _check(o, *_ref64(x, w, cos, sin, full, eps))


def test_offsets_past_32_bits():
    """2.4 billion elements of q: rows at both ends against the formula."""
    T, D = 590_001, 128
    q = torch.zeros(1, T, 32, D, device=CUDA, dtype=torch.bfloat16).transpose(1, 2)
    k = torch.zeros(1, 1, T, D, device=CUDA, dtype=torch.bfloat16)
    ends = torch.tensor([0, 1, T // 2, T - 2, T - 1], device=CUDA)
    q[:, :, ends] = randn((1, 32, 5, D), 1, torch.bfloat16, CUDA)
    k[:, :, ends] = randn((1, 1, 5, D), 2, torch.bfloat16, CUDA)
    cos, sin = _angles(T, D, torch.bfloat16)
    q.requires_grad_(True)
    yq, yk = sa.qk_norm_rope(q, k, cos, sin)
    qe, ke = q.detach()[:, :, ends], k[:, :, ends]
    _check(yq.detach()[:, :, ends], *_ref64(qe, None, cos.float(), sin.float(), ends[None], 1e-6))
    _check(yk[:, :, ends], *_ref64(ke, None, cos.float(), sin.float(), ends[None], 1e-6))
    assert yq.count_nonzero() == yq[:, :, ends].count_nonzero()
    (dq,) = torch.autograd.grad(yq, q, torch.ones_like(yq))
    ref = _ref64(qe, None, cos.float(), sin.float(), ends[None], 1e-6, torch.ones_like(qe))
    _check(dq[:, :, ends], ref[2], ref[3])


def test_bases_off_a_boundary_and_mixed_weight_types():
    """Contiguous views that start off 16 bytes; weights of two types, each with its own gradient type."""
    def off(t):
        b = torch.empty(t.numel() + 1, device=CUDA, dtype=t.dtype)
        return b[1:].view(t.shape).copy_(t)

    q, k, dq, dk, wq, wk, cos, sin, pos, full, eps = _make((2, 4, 2, 9, 64, 64, torch.bfloat16, torch.bfloat16, True,
                                                            "batch64"))
    want = [t.clone() for t in (q, k, wq, wk)]
    for base, mixed in ((True, False), (False, True), (True, True)):
        ins = [off(t) if base else t.clone() for t in want]
        if mixed:
            ins[2] = off(want[2].float())
        ins = [t.detach().requires_grad_(True) for t in ins]
        c, s = (off(cos), off(sin)) if base else (cos, sin)
        y = sa.qk_norm_rope(ins[0], ins[1], c, s, q_weight=ins[2], k_weight=ins[3], positions=off(pos) if base else pos)
        g = torch.autograd.grad(y, ins, (off(dq), off(dk)) if base else (dq, dk))
        assert g[2].dtype == ins[2].dtype and g[3].dtype == torch.bfloat16
        for x, w, o, dx, dw, dy in ((q, wq, y[0], g[0], g[2], dq), (k, wk, y[1], g[1], g[3], dk)):
            ref = _ref64(x, w, cos, sin, full, eps, dy)
            _check(o.detach(), ref[0], ref[1])
            _check(dx, ref[2], ref[3])
            # (bf16 weights beside fp32 ones are taken as fp32: one more rounding to their gradient's type)
            _check(dw, ref[4], ref[5] + 4 * U * ref[4].abs())


def test_hooks_on_saved_tensors():
    """Saved tensors that come back in another layout (an offload) give the same gradients."""
    q, k, dq, dk, wq, wk, cos, sin, pos, full, eps = _make((2, 8, 2, 33, 64, 64, torch.bfloat16, torch.float32, True,
                                                            "batch32"))
    q = q.transpose(1, 2).contiguous().transpose(1, 2)

    def grads(hooked):
        ins = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
        pack = torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().cpu(), lambda t: t.to(CUDA))
        if hooked:
            with pack:
                y = sa.qk_norm_rope(ins[0], ins[1], cos, sin, q_weight=ins[2], k_weight=ins[3], positions=pos)
        else:
            y = sa.qk_norm_rope(ins[0], ins[1], cos, sin, q_weight=ins[2], k_weight=ins[3], positions=pos)
        return torch.autograd.grad(y, ins, (dq, dk))

    assert all(torch.equal(a, b) for a, b in zip(grads(False), grads(True)))


def test_a_changed_input_is_noticed():
    """The backward reads the forward's inputs: changing one in between is an error, as for torch's own operators."""
    q, k, *_ = _make(CASES[1])
    x = q.clone().requires_grad_(True)
    held = x * 1
    y, _ = sa.qk_norm_rope(held, k)
    held.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_gradient_against_differences():
    """fp32: the gradient along a direction against a central difference of the kernel's own forward."""
    case = (1, 2, 1, 9, 64, 32, torch.float32, torch.float32, True, "none")
    q, k, dq, dk, wq, wk, cos, sin, pos, full, eps = _make(case)
    ins = [t.detach().requires_grad_(True) for t in (q, wq)]
    y, _ = sa.qk_norm_rope(ins[0], k, cos, sin, q_weight=ins[1], k_weight=wk)
    gq, gw = torch.autograd.grad(y, ins, dq)
    vq, vw, h = randn(q.shape, 50, torch.float32, CUDA), randn(wq.shape, 51, torch.float32, CUDA), 2.0 ** -6

    def f(sign, fn):
        return (fn(q + sign * h * vq, wq + sign * h * vw).double() * dq.double()).sum()

    kern = lambda a, w: sa.qk_norm_rope(a, k, cos, sin, q_weight=w, k_weight=wk)[0]  # noqa: E731
    exact = lambda a, w: _ref64(a, w, cos, sin, full, eps)[0]  # noqa: E731
    diff = (f(1, kern) - f(-1, kern)) / (2 * h)
    along = (gq.double() * vq.double()).sum() + (gw.double() * vw.double()).sum()
    # the difference's own truncation, from the formula in 64 bits, and both sides' roundings
    ref = _ref64(q, wq, cos, sin, full, eps, dq)
    truncation = ((f(1, exact) - f(-1, exact)) / (2 * h)
                  - (ref[2] * vq.double()).sum() - (ref[4] * vw.double()).sum()).abs()
    hi = _ref64(q.abs() + h * vq.abs(), wq.abs() + h * vw.abs(), cos, sin, full, eps)
    roundings = ((hi[1] + _half_step(hi[0], torch.float32)) * dq.abs()).sum() / h
    roundings += ((ref[3] + _half_step(ref[2], torch.float32)) * vq.abs()).sum()
    roundings += ((ref[5] + _half_step(ref[4], torch.float32)) * vw.abs()).sum()
    assert (diff - along).abs() <= truncation * 1.001 + roundings
    assert truncation + roundings < 1e-2 * ((ref[2] * vq).abs().sum() + (ref[4] * vw).abs().sum())  # it says something


def test_rows_of_zeros_infinities_and_nan():
    q, k, *_ = _make((1, 4, 1, 6, 64, 64, torch.bfloat16, None, True, "none"))
    cos, sin = _angles(6, 64)
    clean = sa.qk_norm_rope(q, k, cos, sin)[0]
    q[0, 0, 1] = 0
    q[0, 1, 2, 5] = math.inf
    q[0, 2, 3, 7] = math.nan
    q[0, 3, 4] = 1e30  # its square passes fp32: the formula in 32 bits says 0
    x = q.clone().requires_grad_(True)
    y = sa.qk_norm_rope(x, k, cos, sin)[0]
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert (y[0, 0, 1] == 0).all() and torch.isfinite(dx[0, 0, 1]).all()
    assert y[0, 1, 2].isnan().any() and y[0, 2, 3].isnan().any()
    same = torch.ones(4, 6, dtype=torch.bool, device=CUDA)
    same[0, 1] = same[1, 2] = same[2, 3] = same[3, 4] = False
    assert torch.equal(y[0][same], clean[0][same])  # no row touches another
    assert torch.isfinite(dx[0][same]).all()


def test_expanded_and_partial_gradients():
    """A query shared over heads (stride 0), a gradient that is an expanded scalar, gradients of some inputs only."""
    one = randn((2, 1, 7, 64), 1, torch.float32, CUDA).requires_grad_(True)
    k = randn((2, 2, 7, 64), 2, torch.float32, CUDA)
    w = (1 + randn((64,), 3, torch.float32, CUDA, 0.3)).requires_grad_(True)
    cos, sin = _angles(7, 64)
    yq, yk = sa.qk_norm_rope(one.expand(2, 3, 7, 64), k, cos, sin, q_weight=w)
    g1, gw = torch.autograd.grad(yq.sum() + 0 * yk.sum(), (one, w), retain_graph=False)
    ref = _ref64(one.detach(), w.detach(), cos, sin, torch.arange(7, device=CUDA).expand(2, 7), 1e-6,
                 torch.ones_like(one))
    _check(g1, 3 * ref[2], 3 * ref[3] + 4 * U * 3 * ref[2].abs())
    _check(gw, 3 * ref[4], 3 * ref[5])
    only_k = k.clone().requires_grad_(True)
    yq, yk = sa.qk_norm_rope(one.detach().expand(2, 3, 7, 64), only_k, cos, sin, q_weight=w.detach())
    (gk,) = torch.autograd.grad(yk, only_k, torch.ones_like(yk))
    ref = _ref64(k, None, cos, sin, torch.arange(7, device=CUDA).expand(2, 7), 1e-6, torch.ones_like(k))
    _check(gk, ref[2], ref[3])


def test_empty():
    cos, sin = _angles(4, 64)
    for shape_q, shape_k in (((2, 4, 0, 64), (2, 2, 0, 64)), ((0, 4, 3, 64), (0, 2, 3, 64)),
                             ((2, 4, 3, 64), (2, 0, 3, 64)), ((2, 0, 3, 64), (2, 1, 3, 64))):
        q = torch.ones(shape_q, device=CUDA, requires_grad=True)
        k = torch.ones(shape_k, device=CUDA, requires_grad=True)
        w = torch.ones(64, device=CUDA, requires_grad=True)
        yq, yk = sa.qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w)
        assert yq.shape == shape_q and yk.shape == shape_k
        grads = torch.autograd.grad((yq, yk), (q, k, w), (torch.ones_like(yq), torch.ones_like(yk)))
        assert torch.isfinite(grads[2]).all()
        if q.numel() + k.numel() == 0:
            assert (grads[2] == 0).all()


def test_far_positions_are_read_as_row_zero_and_reported():
    lib = _lib.load()
    lib.sa_device_status(1)
    q, k, *_ = _make((1, 2, 1, 4, 64, 64, torch.bfloat16, None, True, "none"))
    cos, sin = _angles(10, 64)
    at = lambda p: sa.qk_norm_rope(q, k, cos, sin, positions=torch.tensor(p, device=CUDA))  # noqa: E731
    y = at([3, 10, -1, 9])
    assert lib.sa_device_status(1) == _lib.SA_ERR_ARG
    assert torch.equal(y[0], at([3, 0, 0, 9])[0])
    assert lib.sa_device_status(1) == _lib.SA_OK
    # the same where a warp's positions are read ahead of their use
    q, k = randn((1, 32, 9000, 64), 1, torch.bfloat16, CUDA), randn((1, 8, 9000, 64), 2, torch.bfloat16, CUDA)
    pos = torch.arange(9000, device=CUDA, dtype=torch.int32) % 10
    good = sa.qk_norm_rope(q, k, cos, sin, positions=pos)
    assert lib.sa_device_status(1) == _lib.SA_OK
    pos[::10] = torch.where(torch.arange(900, device=CUDA) % 2 == 0, -7, 2 ** 31 - 1).to(torch.int32)  # row 0 as before
    assert all(torch.equal(a, b) for a, b in zip(good, sa.qk_norm_rope(q, k, cos, sin, positions=pos)))
    assert lib.sa_device_status(1) == _lib.SA_ERR_ARG


def test_replayed_from_a_graph_and_on_another_stream():
    q, k, dq, dk, wq, wk, cos, sin, pos, full, eps = _make(CASES[3])
    f = lambda: sa.qk_norm_rope(q, k, cos, sin, q_weight=wq, k_weight=wk, positions=pos)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = f()
    torch.cuda.current_stream().wait_stream(side)
    gc.collect()
    gc.disable()
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            out = f()
    finally:
        gc.enable()
    assert all(torch.equal(a, b) for a, b in zip(on_side, f()))
    q.copy_(randn(q.shape, 90, q.dtype, CUDA))
    pos.add_(1).remainder_(300)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, f()))


def test_graphed_training_step():
    q, k, dq, dk, wq, wk, cos, sin, pos, full, eps = _make(CASES[3])
    sample = [t.detach().clone().requires_grad_(True) for t in (q, k, wq, wk)]
    gc.collect()
    fn = torch.cuda.make_graphed_callables(
        lambda a, b, c, d: sa.qk_norm_rope(a, b, cos, sin, q_weight=c, k_weight=d, positions=pos), tuple(sample))
    for step in range(2):
        ins = [randn(t.shape, 30 + step + i, torch.float32, CUDA).to(t.dtype).requires_grad_(True)
               for i, t in enumerate(sample)]
        ref = [t.detach().clone().requires_grad_(True) for t in ins]
        ga = torch.autograd.grad(fn(*ins), ins, (dq, dk))
        gr = torch.autograd.grad(sa.qk_norm_rope(ref[0], ref[1], cos, sin, q_weight=ref[2], k_weight=ref[3],
                                                 positions=pos), ref, (dq, dk))
        assert all(torch.equal(a, b) for a, b in zip(ga, gr))


def test_second_derivative_is_refused():
    q, k, *_ = _make(CASES[1])
    q = q.float().requires_grad_(True)
    y, _ = sa.qk_norm_rope(q, k.float())
    (g,) = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("compiled", [False, True])
def test_attention_trains_through_it(compiled):
    """sp2norm_qk_norm_rope_flash_attention: the output and every gradient against the oracle's
    attention on queries and keys normalised and rotated in 64 bits."""
    B, Hq, Hkv, T, D = 1, 4, 2, 200, 64
    q, k, do, _, wq, wk, cos, sin, pos, full, eps = _make((B, Hq, Hkv, T, D, D, torch.bfloat16, torch.bfloat16, True,
                                                           "batch32"))
    v = randn(k.shape, 9, torch.bfloat16, CUDA)
    ins = [t.detach().requires_grad_(True) for t in (q, k, v, wq, wk)]

    def f(q, k, v, wq, wk):
        return sa.sp2norm_qk_norm_rope_flash_attention(q, k, v, cos, sin, q_weight=wq, k_weight=wk, positions=pos)

    o = (torch.compile(f, fullgraph=True, backend="aot_eager") if compiled else f)(*ins)
    grads = torch.autograd.grad(o, ins, do)
    yq, yk = (_ref64(x, w, cos, sin, full, eps)[0].to(torch.bfloat16) for x, w in ((q, wq), (k, wk)))
    args = (np32(yq), np32(yk), np32(v))
    import numpy as np

    ref = O.sp2norm_flash_attention(*args)
    np.testing.assert_allclose(np32(o), ref, rtol=2e-2, atol=1e-2)
    d64 = O.sp2norm_flash_attention_bwd(*args, np32(do), acc=np.float64)
    emu = O.sp2norm_flash_attention_bwd(*args, np32(do), emulate=True)
    # through the norm's own 64-bit backward: dq and dk as the attention hands them over (bf16)
    yg = torch.autograd.grad(sa.sp2norm_flash_attention(*(a := [yq.clone().requires_grad_(True),
                                                                yk.clone().requires_grad_(True),
                                                                v.clone().requires_grad_(True)])), a, do)
    check_bf16_grads(np32(grads[2]), d64[2], emu[2])
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        check_bf16_grads(np32(yg[i]), d64[i], emu[i])
        r = _ref64(x, w, cos, sin, full, eps, yg[i])
        # yq / yk may round to the other neighbour and dQ sums in another order: 2^-7 of the gradients' size
        rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
        assert rel(grads[i], r[2]) < 2.0 ** -7 and rel(grads[3 + i], r[4]) < 2.0 ** -7


@pytest.mark.parametrize("eps", [0.0, 1e-50])  # (the second is 0 in fp32)
@pytest.mark.parametrize("B,Hq,Hkv,T,D,R,dt", [
    (1, 1, 1, 1, 128, 128, torch.bfloat16), (1, 3, 1, 7, 16, 16, torch.float32), (3, 5, 2, 5, 80, 32, torch.float16),
    (1, 4, 4, 33, 64, 64, torch.float16), (2, 4, 2, 27, 128, 64, torch.float32), (1, 2, 1, 5, 256, 256, torch.bfloat16),
])
def test_gradients_without_eps(B, Hq, Hkv, T, D, R, dt, eps):
    """Rows that are not zero need no eps; what lies behind the last token adds nothing to the weights' gradients."""
    q, k, dq, dk, wq, wk, cos, sin, pos, full, _ = _make((B, Hq, Hkv, T, D, R, dt, torch.float32, True, "batch32"))
    ins = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    y = sa.qk_norm_rope(ins[0], ins[1], cos, sin, q_weight=ins[2], k_weight=ins[3], eps=eps, positions=pos)
    g = torch.autograd.grad(y, ins, (dq, dk))
    for x, w, o, dx, dw, dy in ((q, wq, y[0], g[0], g[2], dq), (k, wk, y[1], g[1], g[3], dk)):
        ref = _ref64(x, w, cos, sin, full, eps, dy)
        _check(o.detach(), ref[0], ref[1])
        _check(dx, ref[2], ref[3])
        _check(dw, ref[4], ref[5])


@pytest.mark.parametrize("R", [0, 16, 32, 48])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_channels_that_are_not_rotated_keep_to_themselves(dt, R):
    """An infinity or NaN in channel R + t of token t: no other channel that is not rotated may see it."""
    D = 64
    T = D - R
    cos, sin = (None, None) if R == 0 else _angles(T, R)
    t = torch.arange(T, device=CUDA)
    for value in (math.inf, -math.inf, math.nan):
        q, k = randn((1, 3, T, D), 1, dt, CUDA), randn((1, 1, T, D), 2, dt, CUDA)
        clean = sa.qk_norm_rope(q, k, cos, sin, eps=None)
        x = [v.clone() for v in (q, k)]
        for v in x:
            v[:, :, t, R + t] = value
        x = [v.requires_grad_(True) for v in x]
        y = sa.qk_norm_rope(x[0], x[1], cos, sin, eps=None)
        for a, b, c in zip(x, y, clean):  # without a norm they are copied
            assert torch.equal(a[..., R:].nan_to_num(7.0), b[..., R:].nan_to_num(7.0))
            assert torch.equal(b[..., :R], c[..., :R])
        g = [randn(v.shape, 3, dt, CUDA) for v in y]
        clean_g = torch.autograd.grad(y, x, g, retain_graph=True)
        for v in g:
            v[:, :, t, R + t] = value
        for a, b, c in zip(g, torch.autograd.grad(y, x, g), clean_g):
            assert torch.equal(a[..., R:].nan_to_num(7.0), b[..., R:].nan_to_num(7.0))
            assert torch.equal(b[..., :R], c[..., :R])
    # with a norm a row that holds an infinity is x / inf * w: NaN there, 0 elsewhere
    x = randn((1, 2, T, D), 4, dt, CUDA)
    x[:, :, t, R + t] = math.inf
    w = 1 + randn((D,), 5, torch.float32, CUDA, 0.3)
    y = sa.qk_norm_rope(x, x, cos, sin, q_weight=w)
    for v in y:
        at = torch.zeros(T, D, dtype=torch.bool, device=CUDA)
        at[t, R + t] = True
        assert v[:, :, at].isnan().all() and (v[:, :, ~at] == 0).all()
    # an infinite weight reaches its own channel alone
    q, w2 = randn((1, 2, T, D), 6, dt, CUDA), w.clone()
    w2[R + 1] = math.inf
    rest = torch.arange(D, device=CUDA) != R + 1
    a, b = (sa.qk_norm_rope(q, q, cos, sin, q_weight=v)[0] for v in (w, w2))
    assert torch.equal(a[..., rest], b[..., rest]) and b[..., R + 1].isinf().all()


def test_forward_mode_derivatives_are_refused():
    """As by sp2norm_flash_attention: never an output that has silently lost its tangent."""
    q, k, dq, _, wq, wk, cos, sin, *_ = _make(CASES[3])
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        plain = sa.qk_norm_rope(q, k, cos, sin, q_weight=wq, k_weight=wk)  # nothing here has one
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args, w in (((dual(q), k, cos, sin), wq), ((q, dual(k), cos, sin), wq), ((q, k, cos, sin), dual(wq)),
                        ((q, k, dual(cos), sin), wq)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                    sa.qk_norm_rope(*args, q_weight=w, k_weight=wk)
    assert all(torch.equal(a, b) for a, b in zip(plain, sa.qk_norm_rope(q, k, cos, sin, q_weight=wq, k_weight=wk)))


def test_c_abi_without_a_norm_leaves_the_weights_out():
    """normalize = 0 is n = x, in both directions, whatever weights come with it."""
    lib, T, D = _lib.load(), 5, 64
    x, dy = randn((1, 2, T, D), 1, torch.float32, CUDA), randn((1, 2, T, D), 2, torch.float32, CUDA)
    w = 1 + randn((D,), 3, torch.float32, CUDA, 0.5)
    cos, sin = _angles(T, 32)
    s = (ctypes.c_int64 * 4)(2 * T * D, T * D, D, 1)
    y, dx = torch.full_like(x, 9.0), torch.full_like(x, 9.0)
    p = lambda t: t.data_ptr()  # noqa: E731
    tables = (p(cos), p(sin), _lib.SA_F32, None, 0, 0, T)
    for weight in (None, p(w)):
        assert lib.sa_qk_norm_rope(p(x), None, p(y), None, weight, weight, _lib.SA_F32, *tables, 1, 2, 0, T, D, 32, s, s, s,
                                   s, 1e-6, 0, _lib.SA_F32, None) == _lib.SA_OK
        assert lib.sa_qk_norm_rope_bwd(p(x), None, p(dy), None, p(dx), None, weight, weight, _lib.SA_F32, None, None,
                                       *tables, None, 0, 1, 2, 0, T, D, 32, s, s, s, s, s, s, 1e-6, 0, _lib.SA_F32,
                                       None) == _lib.SA_OK
        torch.cuda.synchronize()
        ref = _ref64(x, None, cos, sin, torch.arange(T, device=CUDA)[None], None, dy)
        _check(y, ref[0], ref[1])
        _check(dx, ref[2], ref[3])


@pytest.mark.parametrize("dynamic", [False, True])
def test_one_tensor_for_queries_and_keys(dynamic):
    """The same tensor as q and k, and one weight for both: the gradients of both uses add up, compiled too."""
    x, _, dq, dk, w, *_ = _make((2, 3, 3, 17, 64, 64, torch.float32, torch.float32, True, "none"))
    cos, sin = _angles(17, 64)
    full = torch.arange(17, device=CUDA).expand(2, 17)
    ref = [_ref64(x, w, cos, sin, full, 1e-6, dy) for dy in (dq, dk)]
    f = lambda q, k, a, b: sa.qk_norm_rope(q, k, cos, sin, q_weight=a, k_weight=b)  # noqa: E731
    for call in (f, torch.compile(f, fullgraph=True, backend="aot_eager", dynamic=dynamic)):
        ins = [t.clone().requires_grad_(True) for t in (x, w)]
        gx, gw = torch.autograd.grad(call(ins[0], ins[0], ins[1], ins[1]), ins, (dq, dk))
        # the two are added once more
        _check(gx, ref[0][2] + ref[1][2], ref[0][3] + ref[1][3] + 4 * U * (ref[0][2].abs() + ref[1][2].abs()))
        _check(gw, ref[0][4] + ref[1][4], ref[0][5] + ref[1][5] + 4 * U * (ref[0][4].abs() + ref[1][4].abs()))
