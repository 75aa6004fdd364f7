"""What is measured of the operators around the attention kernels: the head
norms with the position rotation, the bookkeeping of a paged key-value cache,
the append into it, and the decode over pages chosen by a cheap score.

``run`` computes an operator in its plain form (elementary torch operations in
32 bits, 64 where an order of values hangs on them) or, where ``own`` is true,
through ``smooth_attn``'s entry points.  ``exact`` states each operator once
more in 64 bits.  Sizes are those of this repository's decode and rotation
benchmarks (32 query heads over 8 key heads of 128 channels, pages of 16
tokens, contexts of 8192 and 32768), and odd ones around them.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # A decode step's queries and keys, eight sequences at positions of their own: latency.
        dict(name="norm rope, 8 new tokens", op="norm_rope", B=8, T=1, Hq=32, Hkv=8, D=128, R=128, dtype="bf16",
             layout="bthd", train=False, table=8192),
        # A small model's training step: odd length, fp16, half of each head's channels rotated.
        dict(name="norm rope training, 509 tokens", op="norm_rope", B=4, T=509, Hq=12, Hkv=12, D=64, R=32,
             dtype="fp16", layout="bhtd", train=True, table=509),
        # A training step at the attention benchmark's length, projections laid out token by token.
        dict(name="norm rope training, 4x4096", op="norm_rope", B=4, T=4096, Hq=32, Hkv=8, D=128, R=128,
             dtype="bf16", layout="bthd", train=True, table=4096),
        # A scheduler's decode step: one more token for each of 64 requests.
        dict(name="slots, 64 requests, one token", op="slots", B=64, max_blocks=512, bs=16, ctx=8191, new=1,
             tokens=64, spare=64),
        # A scheduler's prefill step: 512 requests with chunks of very different lengths, about a million tokens.
        dict(name="slots, 512 ragged prompts", op="slots", B=512, max_blocks=512, bs=16, ctx=2047, new=4096,
             tokens=1000003, spare=90000),
        # Half of 512 requests ended: their pages go back to the pool.
        dict(name="release, 512 requests", op="release", B=512, max_blocks=512, bs=16, ctx=8191),
        # The decode step's append: one token for each of 64 sequences, into pages of their own.
        dict(name="append, 64 sequences", op="append", N=64, pad=0, Hq=32, Hkv=8, D=128, R=128, bs=16, pages=4096,
             dtype="bf16", per_request=1, norm=True),
        # A prefill step's append: ragged prompts, a padded batch, queries, keys and values of one fused projection.
        dict(name="append, prompts of 8191 tokens", op="append", N=8191, pad=65, Hq=32, Hkv=8, D=128, R=128, bs=16,
             pages=4096, dtype="bf16", per_request=1000, norm=True),
        # After a decode step: the few pages that it filled get their mean key.
        dict(name="key means, 64 sequences, one token", op="means", B=64, max_blocks=128, ctx=2048, new=1, Hkv=8,
             D=128, bs=16, dtype="bf16"),
        # After a prefill: the mean keys of whole prompts.
        dict(name="key means, 8 prompts of 8191", op="means", B=8, max_blocks=512, ctx=8191, new=8191, Hkv=8, D=128,
             bs=16, dtype="bf16"),
        # One long sequence, a sixteenth of its pages read: latency of the choice.
        dict(name="page choice, 1x32768, 128 pages", op="sparse", B=1, Hq=32, Hkv=8, D=128, bs=16, max_blocks=2048,
             ctx=32761, least=32761, num_pages=128, dtype="bf16"),
        # A batch of ragged contexts, an eighth of the longest one's pages read.
        dict(name="page choice, 32x8192, 64 pages", op="sparse", B=32, Hq=32, Hkv=8, D=128, bs=16, max_blocks=512,
             ctx=8192, least=5000, num_pages=64, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("norm_rope", "norm_rope", "slots", "release", "append", "means", "sparse", "sparse"))
    Hkv = rng.choice((1, 2, 4, 8))
    G = rng.choice((1, 2, 4, 8))
    if op == "norm_rope":
        D = rng.choice((32, 64, 80, 128, 256))
        R = rng.choice((D, D, 16, 32))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        most = 4 * 4096 * 40 * 128 // (2 if dtype == "fp32" else 1) // (Hkv * (G + 1) * D)  # tokens
        T = _spread(rng, 1, min(8192, most))
        B = rng.randint(1, max(1, min(16, most // T)))
        return dict(op=op, B=B, T=T, Hq=Hkv * G, Hkv=Hkv, D=D, R=R, dtype=dtype,
                    layout=rng.choice(("bthd", "bhtd")), train=rng.random() < 0.6, table=T + rng.randint(0, 700))
    if op == "slots":
        B, bs, new = _spread(rng, 1, 1024), rng.choice((8, 16, 32, 64, 128)), _spread(rng, 1, 4096)
        cap, want = 8192, B * (new + 1) // 2
        return dict(op=op, B=B, max_blocks=cap // bs, bs=bs, ctx=rng.randint(0, cap - 1), new=new,
                    tokens=max(1, min(1000003, want + rng.randint(-want // 8, want // 8 + 3))),
                    spare=max(1, want // bs + rng.randint(-8, B)))
    if op == "release":
        bs = rng.choice((8, 16, 32, 64))
        return dict(op=op, B=_spread(rng, 1, 1024), max_blocks=4096 // bs, bs=bs, ctx=rng.randint(0, 4096))
    if op == "append":
        D = rng.choice((32, 64, 128, 256))
        N, bs = _spread(rng, 1, 8191), rng.choice((8, 16, 32, 64))
        return dict(op=op, N=N, pad=rng.choice((0, 0, 1, 33)), Hq=Hkv * G, Hkv=Hkv, D=D, R=rng.choice((D, D, 32)),
                    bs=bs, pages=max(8, 2 * N // bs + N // 7 + 1), dtype=rng.choice(("bf16", "fp16")),
                    per_request=_spread(rng, 1, 1000), norm=rng.random() < 0.8)
    if op == "means":
        bs, B = rng.choice((8, 16, 32, 64)), _spread(rng, 1, 64)
        cap = max(bs, min(8192, 8 * 8191 // B))
        ctx = _spread(rng, 1, cap)
        return dict(op=op, B=B, max_blocks=-(-cap // bs), ctx=ctx, new=rng.choice((1, _spread(rng, 1, ctx), ctx)),
                    Hkv=Hkv, D=rng.choice((32, 64, 128, 256)), bs=bs, dtype=rng.choice(("bf16", "fp16")))
    bs, B = rng.choice((16, 16, 32, 64)), _spread(rng, 1, 32)
    D = rng.choice((64, 128, 128))
    cap = min(32768, 16 * 8192 // B)
    ctx = _spread(rng, bs, cap)
    n = -(-ctx // bs)
    return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, D=D, bs=bs, max_blocks=n + rng.randint(0, 3), ctx=ctx,
                least=rng.randint(0, ctx), num_pages=_spread(rng, 1, min(n, 128)), dtype=rng.choice(("bf16", "fp16")))


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(scale).to(dtype)


def _tables(rows, R):
    """cos and sin of position times 10000^(-2i/R), angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _ints(g, lo, hi, n):
    """n whole numbers in lo..hi."""
    return torch.randint(lo, hi + 1, (n,), device="cuda", generator=g)


def _page_table(g, ctx, max_blocks, bs, pool):
    """A block table whose requests hold the first pages of a shuffled pool:
    (table with -1 where nothing is held, the pool, how many of it are held)."""
    pages = (ctx + bs - 1) // bs
    off = torch.cumsum(pages, 0) - pages
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    j = torch.arange(max_blocks, device="cuda")
    held = j[None, :] < pages[:, None]
    table = torch.where(held, order[(off[:, None] + j).clamp(max=pool - 1)], torch.full_like(order[:1], -1))
    return table, order, pages.sum().to(torch.int32).reshape(1)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] == "norm_rope":
        dt = DTYPES[c["dtype"]]
        B, T, D = c["B"], c["T"], c["D"]
        for n, H in (("q", c["Hq"]), ("k", c["Hkv"])):
            per_head = 0.25 + 1.5 * torch.rand((H, 1), device="cuda", generator=g)
            x = (torch.randn((B, T, H, D), device="cuda", generator=g) * per_head).to(dt)
            dy = _randn(g, (B, T, H, D), dt)
            if c["layout"] == "bhtd":
                x, dy = x.transpose(1, 2).contiguous(), dy.transpose(1, 2).contiguous()
            else:  # the projections' own order, seen as [B, H, T, D]
                x, dy = x.transpose(1, 2), dy.transpose(1, 2)
            s[n], s["d" + n] = x, dy
            s["w" + n] = (1 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dt)
            if c["train"]:
                s[n].requires_grad_(True)
                s["w" + n].requires_grad_(True)
        s["cos"], s["sin"] = _tables(c["table"], c["R"])
        s["positions"] = _ints(g, 0, c["table"] - 1, B * T).reshape(B, T).to(torch.int32)
    elif c["op"] in ("slots", "release"):
        B, bs, cap = c["B"], c["bs"], c["max_blocks"] * c["bs"]
        ctx = _ints(g, 0, c["ctx"], B)
        if c["op"] == "slots":
            s["new"] = (_ints(g, 0, c["new"], B) if c["new"] > 1 else torch.ones(B, device="cuda")).to(torch.int32)
        else:
            s["done"] = torch.rand(B, device="cuda", generator=g) < 0.5
        pool = B * -(-min(c["ctx"], cap) // bs) + c.get("spare", 16)
        s["table"], s["free"], s["head"] = _page_table(g, ctx, c["max_blocks"], bs, pool)
        if c["op"] == "slots":  # a short pool: what the requests hold, and `spare` pages
            held = int(s["head"])
            s["free"] = s["free"][: held + c["spare"]].clone()
        s["ctx"] = ctx.to(torch.int32)
    elif c["op"] == "append":
        dt = DTYPES[c["dtype"]]
        N, Hq, Hkv, D, bs = c["N"] + c["pad"], c["Hq"], c["Hkv"], c["D"], c["bs"]
        qkv = _randn(g, (N, (Hq + 2 * Hkv) * D), dt)
        s["q"] = qkv[:, : Hq * D].view(N, Hq, D)
        s["k"] = qkv[:, Hq * D: (Hq + Hkv) * D].view(N, Hkv, D)
        s["v"] = qkv[:, (Hq + Hkv) * D:].view(N, Hkv, D)
        s["wq"], s["wk"] = (1 + _randn(g, (D,), torch.float32, 0.2) for _ in range(2))
        s["cos"], s["sin"] = _tables(c["per_request"] + 4096, c["R"])
        i = torch.arange(N, device="cuda")
        req, at = i // c["per_request"], i % c["per_request"]
        first = _ints(g, 0, 4095, int(N // c["per_request"]) + 1)
        pos = first[req] + at
        # pages of a request: as many as its longest span can touch, from a shuffled pool
        span = -(-c["per_request"] // bs) + 1
        pool = max(c["pages"], int(N // c["per_request"] + 1) * span)
        order = torch.randperm(pool, device="cuda", generator=g)
        slot = order[req * span + pos // bs - first[req] // bs] * bs + pos % bs
        s["positions"] = torch.where(i < c["N"], pos, 0).to(torch.int32)
        s["slots"] = torch.where(i < c["N"], slot, -1)
        s["kc"], s["vc"] = (torch.zeros((pool, Hkv, bs, D), device="cuda", dtype=dt) for _ in range(2))
    elif c["op"] == "means":
        dt = DTYPES[c["dtype"]]
        B, bs = c["B"], c["bs"]
        ctx = torch.clamp(c["ctx"] - _ints(g, 0, min(2 * bs, c["ctx"]), B), min=0)
        s["table"], order, _ = _page_table(g, ctx, c["max_blocks"], bs, B * c["max_blocks"])
        s["kc"] = _randn(g, (B * c["max_blocks"], c["Hkv"], bs, c["D"]), dt)
        s["means"] = _randn(g, (B * c["max_blocks"], c["Hkv"], c["D"]), dt)  # of earlier steps: kept where not renewed
        s["ctx"] = ctx.to(torch.int32)
        s["start"] = torch.clamp(ctx - c["new"], min=0).to(torch.int32)
    else:
        dt = DTYPES[c["dtype"]]
        B, bs, Hkv, D = c["B"], c["bs"], c["Hkv"], c["D"]
        ctx = _ints(g, c["least"], c["ctx"], B)
        s["table"], order, _ = _page_table(g, ctx, c["max_blocks"], bs, B * c["max_blocks"])
        P = B * c["max_blocks"]
        centre = torch.randn((P, Hkv, 1, D), device="cuda", generator=g)  # pages differ, as topics do
        s["kc"] = torch.randn((P, Hkv, bs, D), device="cuda", generator=g).mul_(0.8).add_(centre, alpha=0.6).to(dt)
        s["vc"] = _randn(g, (P, Hkv, bs, D), dt)
        s["means"] = s["kc"].float().mean(2).to(dt)
        s["q"] = _randn(g, (B, c["Hq"], 1, D), dt, 1.5)
        s["ctx"] = ctx.to(torch.int32)
    return s


# ------------------------------------------------------------------ the framework's calls


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "smooth-attn_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import smooth_attn

    return smooth_attn


def _run_own(s):
    sa, c = _package(), s["case"]
    if c["op"] == "norm_rope":
        q, k = sa.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], q_weight=s["wq"], k_weight=s["wk"],
                               positions=s["positions"])
        if not c["train"]:
            return {"q": q, "k": k}
        g = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": g[0], "dk": g[1], "dwq": g[2], "dwk": g[3]}
    if c["op"] == "slots":
        r = sa.paged_assign_slots(s["table"], s["ctx"], s["new"], s["free"], s["head"], c["tokens"],
                                  block_size=c["bs"])
        return {"table": s["table"], "slots": r.slot_mapping, "positions": r.positions, "cu": r.cu_seqlens,
                "ctx": r.context_lens, "head": r.free_head}
    if c["op"] == "release":
        ctx, head = sa.paged_release_pages(s["table"], s["ctx"], s["done"], s["free"], s["head"], block_size=c["bs"])
        return {"free": s["free"], "ctx": ctx, "head": head}
    if c["op"] == "append":
        w = dict(q_weight=s["wq"], k_weight=s["wk"]) if c["norm"] else dict(eps=None)
        q = sa.qk_norm_rope_paged_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["cos"], s["sin"],
                                         positions=s["positions"], **w)
        return {"q": q, "kc": s["kc"], "vc": s["vc"]}
    if c["op"] == "means":
        return sa.paged_key_means(s["means"], s["kc"], s["table"], s["ctx"], start_lens=s["start"])
    out, pages = sa.sp2norm_sparse_paged_attention(s["q"], s["kc"], s["vc"], s["means"], s["table"], s["ctx"],
                                                   c["num_pages"], block_size=c["bs"], return_pages=True)
    return {"out": out, "pages": pages}


# ------------------------------------------------------------------ the plain forms

EPS = 1e-6


def _rotate(x, cos, sin):
    """Rotate-half form on the first 2 * cos.shape[-1] channels."""
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h: 2 * h]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]), -1)


def _norm_rope_plain(x, w, cos, sin, dy):
    """(y, dx, dw) of y = rotate(x / rms(x) * w); no gradients where dy is None."""
    xf, wf = x.detach().float(), w.detach().float()
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    y = _rotate(xf * r * wf, cos, sin).to(x.dtype)
    if dy is None:
        return y, None, None
    dn = _rotate(dy.float(), cos, -sin)  # the rotation's transpose
    hat = xf * r
    gw = dn * wf
    dx = r * (gw - hat * (gw * hat).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), (dn * hat).sum((0, 1, 2)).to(w.dtype)


def _slots_plain(s):
    c = s["case"]
    N, bs, B, mb = c["tokens"], c["bs"], c["B"], c["max_blocks"]
    cap, nfree = mb * bs, s["free"].numel()
    ctx = s["ctx"].long().clamp(0, cap)
    new = s["new"].long().clamp(min=0)
    cu = torch.cat((new.new_zeros(1), torch.cumsum(new, 0))).clamp(max=N)
    want = torch.minimum(cu[1:] - cu[:-1], cap - ctx)
    held = (ctx + bs - 1) // bs
    need = (ctx + want + bs - 1) // bs - held
    at = s["head"].long() + torch.cumsum(need, 0) - need
    have = torch.minimum((nfree - at).clamp(min=0), need)
    fits = torch.minimum(want, (held + have) * bs - ctx)
    i = torch.arange(N, device="cuda")
    b = torch.searchsorted(cu[1:], i, right=True)
    real, b = b < B, b.clamp(max=B - 1)
    pos = ctx[b] + i - cu[b]
    real &= i - cu[b] < fits[b]
    pos = torch.where(real, pos, 0)
    pi = pos // bs
    fresh = s["free"].long()[(at[b] + pi - held[b]).clamp(0, nfree - 1)]
    page = torch.where(pi < held[b], s["table"].long()[b, pi], fresh)
    slots = torch.where(real, page * bs + pos % bs, -1)
    j = torch.arange(mb, device="cuda")[None, :] - held[:, None]
    mine = (j >= 0) & (j < have[:, None])
    took = s["free"][(at[:, None] + j).clamp(0, nfree - 1)]
    s["table"].copy_(torch.where(mine, took, s["table"]))
    return {"table": s["table"], "slots": slots, "positions": pos.to(torch.int32), "cu": cu.to(torch.int32),
            "ctx": (ctx + fits).to(torch.int32), "head": (s["head"].long() + have.sum()).to(torch.int32)}


def _release_plain(s):
    c = s["case"]
    pages = torch.where(s["done"], (s["ctx"].long() + c["bs"] - 1) // c["bs"], 0)
    head = s["head"].long() - pages.sum()
    off = head + torch.cumsum(pages, 0) - pages
    j = torch.arange(c["max_blocks"], device="cuda")[None, :].expand(c["B"], -1)
    mine = j < pages[:, None]
    s["free"][(off[:, None] + j)[mine]] = s["table"][mine]
    return {"free": s["free"], "ctx": torch.where(s["done"], 0, s["ctx"]), "head": head.to(torch.int32)}


def _append_plain(s):
    c = s["case"]
    bs, real = c["bs"], s["slots"] >= 0
    cos, sin = (t[s["positions"].long()][:, None, :] for t in (s["cos"], s["sin"]))
    q, k = s["q"].float(), s["k"].float()
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["wq"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["wk"]
    q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    slot = s["slots"][real]
    s["kc"][slot // bs, :, slot % bs] = k[real].to(s["kc"].dtype)
    s["vc"][slot // bs, :, slot % bs] = s["v"][real]
    return {"q": torch.where(real[:, None, None], q, 0).to(s["q"].dtype), "kc": s["kc"], "vc": s["vc"]}


def _means_plain(s):
    c = s["case"]
    bs = c["bs"]
    j = torch.arange(c["max_blocks"], device="cuda")[None, :]
    done = (j >= s["start"][:, None] // bs) & (j < s["ctx"][:, None] // bs)
    pages = s["table"][done].long()
    s["means"][pages] = s["kc"][pages].float().mean(2).to(s["means"].dtype)
    return s["means"]


def _squareplus(a):
    """(a + sqrt(a^2 + 4)) / 2 without the cancellation of negative a."""
    root = torch.sqrt(a * a + 4)
    return torch.where(a < 0, 2 / (root - a), (a + root) / 2)


def _sparse_plain(s):
    c = s["case"]
    B, Hq, Hkv, D, bs = c["B"], c["Hq"], c["Hkv"], c["D"], c["bs"]
    K, G, scale = min(c["num_pages"], c["max_blocks"]), Hq // Hkv, 1.0 / math.sqrt(D)
    ctx = s["ctx"].long()
    n = (ctx + bs - 1) // bs
    j = torch.arange(c["max_blocks"], device="cuda")
    table = s["table"].long().clamp(min=0)
    # the order of the pages hangs on the scores: 64 bits
    q64 = s["q"].double().view(B, Hkv, G, D)
    m64 = s["means"][table].double().permute(0, 2, 3, 1)  # [B, Hkv, D, pages]
    y = _squareplus(2 * scale * torch.matmul(q64, m64) - 1)
    score = (y * y).sum(2)
    score = torch.where(j < (n - 1)[:, None, None], score, -1.0)  # behind the last page: never
    score = torch.where(j == (n - 1)[:, None, None], math.inf, score)  # the last page: always
    top = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :K]
    picked = torch.arange(K, device="cuda") < n.clamp(max=K)[:, None, None]
    last = torch.full_like(top, c["max_blocks"])
    pages = torch.sort(torch.where(picked, top, last), -1).values
    picked = pages < c["max_blocks"]
    phys = torch.gather(table[:, None].expand(B, Hkv, -1), 2, torch.where(picked, pages, 0))
    h = torch.arange(Hkv, device="cuda")[None, :, None]
    k = s["kc"][phys, h].float().reshape(B, Hkv, K * bs, D)
    v = s["vc"][phys, h].float().reshape(B, Hkv, K * bs, D)
    token = (pages[..., None] * bs + torch.arange(bs, device="cuda")).reshape(B, Hkv, K * bs)
    seen = (token < ctx[:, None, None]) & picked.repeat_interleave(bs, -1)
    sc = torch.matmul(s["q"].float().view(B, Hkv, G, D), k.transpose(-1, -2)) * scale
    a = 2 * sc - 1
    y = 0.5 * (a + torch.sqrt(a * a + 4))
    y = torch.where(seen[:, :, None, :], y * y, 0.0)
    out = torch.matmul(y, v) / (y.sum(-1, keepdim=True) + 1e-12)
    return {"out": out.reshape(B, Hq, D).to(torch.bfloat16),
            "pages": torch.where(picked, pages, -1).to(torch.int32)}


def run(state):
    s = state
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "norm_rope":
        cos, sin = (t[s["positions"].long()][:, None] for t in (s["cos"], s["sin"]))
        q, dq, dwq = _norm_rope_plain(s["q"], s["wq"], cos, sin, s["dq"] if c["train"] else None)
        k, dk, dwk = _norm_rope_plain(s["k"], s["wk"], cos, sin, s["dk"] if c["train"] else None)
        return {"q": q, "k": k} if not c["train"] else {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    return {"slots": _slots_plain, "release": _release_plain, "append": _append_plain, "means": _means_plain,
            "sparse": _sparse_plain}[c["op"]](s)


# ------------------------------------------------------------------ in 64 bits


def _rope64(x, w, cos, sin, eps=EPS):
    """x / sqrt(mean x^2 + eps) * w, each pair turned as a complex number; w None: turned only."""
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    h = cos.shape[-1]
    z = torch.complex(x[..., :h].contiguous(), x[..., h: 2 * h].contiguous()) * torch.complex(cos, sin)
    return torch.cat((z.real, z.imag, x[..., 2 * h:]), -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "norm_rope":
        cos, sin = (t.double()[s["positions"].long()].unsqueeze(1) for t in (s["cos"], s["sin"]))
        r = {}
        for n in ("q", "k"):
            x = s[n].detach().double().requires_grad_(c["train"])
            w = s["w" + n].detach().double().requires_grad_(c["train"])
            y = _rope64(x, w, cos, sin)
            r[n] = y.detach()
            if c["train"]:
                r["d" + n], r["dw" + n] = torch.autograd.grad(y, (x, w), s["d" + n].double())
        return r
    if c["op"] in ("slots", "release"):
        return None  # whole numbers only
    if c["op"] == "append":
        bs = c["bs"]
        cos, sin = (t.double()[s["positions"].long()].unsqueeze(1) for t in (s["cos"], s["sin"]))
        q = _rope64(s["q"].double(), s["wq"].double() if c["norm"] else None, cos, sin)
        k = _rope64(s["k"].double(), s["wk"].double() if c["norm"] else None, cos, sin)
        keep = torch.nonzero(s["slots"] >= 0).flatten()
        q64 = torch.zeros_like(q)
        q64[keep] = q[keep]
        flat = [t.double().transpose(1, 2).reshape(-1, c["Hkv"], c["D"]) for t in (s["kc"], s["vc"])]
        flat[0].index_copy_(0, s["slots"][keep], k[keep])
        flat[1].index_copy_(0, s["slots"][keep], s["v"].double()[keep])
        kc, vc = (t.view(-1, bs, c["Hkv"], c["D"]).transpose(1, 2) for t in flat)
        return {"q": q64, "kc": kc, "vc": vc}
    if c["op"] == "means":
        means, bs = s["means"].double(), c["bs"]
        for row, lo, hi in zip(s["table"].tolist(), s["start"].tolist(), s["ctx"].tolist()):
            ids = torch.tensor(row[lo // bs: hi // bs], device="cuda", dtype=torch.long)
            if ids.numel():
                means[ids] = s["kc"][ids].double().sum(2) / bs
        return means
    out = torch.zeros((c["B"], c["Hq"], c["D"]), device="cuda", dtype=torch.float64)
    G, bs, scale = c["Hq"] // c["Hkv"], c["bs"], c["D"] ** -0.5
    act = lambda a: torch.where(a < 0, 2 / (torch.sqrt(a * a + 4) - a), (a + torch.sqrt(a * a + 4)) / 2) ** 2  # noqa: E731
    for b, n in enumerate(s["ctx"].tolist()):
        if not n:
            continue
        ids = s["table"][b, : -(-n // bs)].long()
        for h in range(c["Hkv"]):
            q = s["q"][b, h * G: (h + 1) * G, 0].double()
            full = ids[:-1]
            sc = act(2 * scale * (q @ s["means"][full, h].double().T) - 1).sum(0)
            best = torch.sort(sc, descending=True, stable=True).indices[: c["num_pages"] - 1]
            mine = torch.cat((full[best.sort().values], ids[-1:]))
            rows = slice(0, (mine.numel() - 1) * bs + n - (ids.numel() - 1) * bs)
            k, v = (t[mine, h].double().reshape(-1, c["D"])[rows] for t in (s["kc"], s["vc"]))
            y = act(2 * scale * (q @ k.T) - 1)
            out[b, h * G: (h + 1) * G] = (y @ v) / (y.sum(1, keepdim=True) + 1e-12)
    return {"out": out, "pages": None}


# ------------------------------------------------------------------ work


def work(case):
    """Bytes each read or written once, and operations, of one pass."""
    c = case
    if c["op"] == "norm_rope":
        e, rows = (4 if c["dtype"] == "fp32" else 2), c["B"] * c["T"] * (c["Hq"] + c["Hkv"])
        tables = min(c["table"], c["B"] * c["T"]) * c["R"] * 4 + c["B"] * c["T"] * 4
        # forward: read x, write y; backward: read x and dy, write dx
        return {"bytes": rows * c["D"] * e * (5 if c["train"] else 2) + tables * (2 if c["train"] else 1),
                "flops": rows * c["D"] * (26 if c["train"] else 8)}
    if c["op"] == "slots":
        new = min(c["tokens"], c["B"] * (c["new"] + 1) // 2)
        # a slot and a position for each token, a table entry read and written for each page, the requests' lengths
        return {"bytes": c["tokens"] * 12 + new // c["bs"] * 8 + c["B"] * 16, "flops": c["tokens"]}
    if c["op"] == "release":
        return {"bytes": c["B"] * (c["ctx"] // 4 // c["bs"] * 8 + 9), "flops": c["B"]}
    if c["op"] == "append":
        rows = c["N"] * (c["Hq"] + 2 * c["Hkv"]) * c["D"]
        return {"bytes": rows * 2 * 2 + c["pad"] * c["Hq"] * c["D"] * 2 + (c["N"] + c["pad"]) * 12
                + min(c["N"], c["per_request"] + 4096) * c["R"] * 4, "flops": rows * 8}
    if c["op"] == "means":
        pages = c["B"] * (c["new"] / c["bs"])
        return {"bytes": pages * c["Hkv"] * c["D"] * 2 * (c["bs"] + 1) + c["B"] * 8,
                "flops": pages * c["Hkv"] * c["D"] * c["bs"]}
    ctx = (c["ctx"] + c["least"]) / 2
    n, K = ctx / c["bs"], min(c["num_pages"], ctx / c["bs"])
    rows = c["B"] * c["Hkv"] * c["D"]
    return {"bytes": rows * 2 * (n + 2 * K * c["bs"]) + c["B"] * c["Hq"] * c["D"] * 4 + c["B"] * n * 4,
            "flops": c["B"] * c["Hq"] * c["D"] * (2 * n + 4 * K * c["bs"])}
