"""The head norm and paged cache operators through the debug library (index
checks that count failures instead of trapping): a child process with
``SA_DEBUG_LIB=1`` runs them on ragged shapes, no check may fail, and every
output equals the release library's bit for bit."""

import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from smooth_attn import _lib

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def run_all(out_path):
    import smooth_attn as sa

    dev, res = "cuda", {}

    def rnd(shape, seed, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)

    for B, Hq, Hkv, T, D, R, dt in ((2, 5, 3, 37, 80, 32, torch.float32), (1, 32, 8, 4001, 128, 128, torch.bfloat16),
                                    (3, 4, 1, 1, 256, 256, torch.float16)):
        cos, sin = sa.precompute_rope_cos_sin(R, T + 9, device=dev)
        ins = [rnd(s, i, dt).requires_grad_(True) for i, s in enumerate(((B, Hq, T, D), (B, Hkv, T, D), (D,), (D,)))]
        y = sa.qk_norm_rope(ins[0], ins[1], cos, sin, q_weight=ins[2], k_weight=ins[3])
        g = torch.autograd.grad(y, ins, [rnd(t.shape, 7, dt) for t in y])
        res.update({f"rope{T}_{i}": t.detach() for i, t in enumerate((*y, *g))})
    Hq, Hkv, D, bs, mb, B = 8, 2, 128, 16, 40, 5
    lens = torch.tensor([1, 0, 333, 17, 600], dtype=torch.int32, device=dev)
    table = torch.full((B, mb), -1, dtype=torch.int32, device=dev)
    pool = torch.randperm(B * mb, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    s = sa.paged_assign_slots(table, torch.zeros_like(lens), lens, pool, zero, 960, block_size=bs)
    kc, vc = (torch.zeros(B * mb, Hkv, bs, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    means = torch.zeros(B * mb, Hkv, D, device=dev, dtype=torch.bfloat16)
    cos, sin = sa.precompute_rope_cos_sin(D, mb * bs, device=dev)
    res["append"] = sa.qk_norm_rope_paged_append(rnd((960, Hq, D), 3), rnd((960, Hkv, D), 4), rnd((960, Hkv, D), 5), kc,
                                                 vc, s.slot_mapping, cos, sin, positions=s.positions)
    sa.paged_key_means(means, kc, table, s.context_lens)
    res["out"], res["pages"] = sa.sp2norm_sparse_paged_attention(rnd((B, Hq, 1, D), 6), kc, vc, means, table,
                                                                 s.context_lens, 7, return_pages=True)
    done = torch.tensor([True, False, True, True, False], device=dev)
    ctx, head = sa.paged_release_pages(table, s.context_lens, done, pool, s.free_head, block_size=bs)
    res.update(slots=s.slot_mapping, positions=s.positions, cu=s.cu_seqlens, kc=kc, vc=vc, means=means, table=table,
               pool=pool, ctx=ctx, head=head)
    torch.cuda.synchronize()
    lib = _lib.load()
    status = lib.sa_device_status(1)
    np.savez(out_path, debug=np.int32(lib.sa_debug_checks()), status=np.int32(status),
             **{k: (v.float() if v.is_floating_point() else v).cpu().numpy() for k, v in res.items()})


def test_debug_library_runs_clean_and_matches_release(tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("CUDA required")
    if not _lib.DEBUG_LIB_PATH.exists():
        pytest.fail("debug library missing: run python smooth-attn_b200/build.py --debug")
    out, ref = tmp_path / "debug.npz", tmp_path / "release.npz"
    code = (f"import sys; sys.path[:0] = [{str(ROOT / 'smooth-attn_b200')!r}, {str(ROOT)!r}]; "
            f"from tests.test_operators_debug_gpu import run_all; run_all({str(out)!r})")
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, SA_DEBUG_LIB="1"), capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    dbg = np.load(out)
    assert int(dbg["debug"]) == 1, "the child did not load the debug library"
    assert int(dbg["status"]) == _lib.SA_OK, f"device status {int(dbg['status'])}: an index check failed"
    run_all(ref)
    rel = np.load(ref)
    assert int(rel["debug"]) == 0 and int(rel["status"]) == _lib.SA_OK
    for key in dbg.files:
        if key not in ("debug", "status"):
            np.testing.assert_array_equal(dbg[key], rel[key], err_msg=key)
