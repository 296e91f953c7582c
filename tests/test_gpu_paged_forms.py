"""The attention over pages in every form that its plan can launch, and the
edges of what mllm_rope_kv_paged and mllm_attn_paged document
(include/mllm.h).  Tolerances: test_gpu_paged.ref_attn's and ref_rope's.
"""
import math

import numpy as np
import pytest

from mllm import abi
from test_gpu_paged import Pool, p, ref_attn, ref_rope, run_attn, run_rope

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
FAR = 2 ** 31 - 1


@gpu
@pytest.mark.parametrize("filler", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("rows", [9, 600])
def test_padding_rows_hold_anything(rows, filler):
    """Padding among and behind the live rows, with any queries, keys, positions
    and lengths: live rows are as the formula has them, the others' outputs and
    the cache stay.  9 rows run in parts, 600 a wave to a unit."""
    g = torch.Generator().manual_seed(41)
    rng = np.random.default_rng(41)
    heads, kvh, hd, seqs = 4, 2, 64, 6
    pool = Pool(g, kvh, hd, 16, seqs, 30 if rows < 100 else 8, "f16")
    top = pool.table.shape[1] * 16
    live = [0, 2, 3, 5]  # rows; the last rows are padding
    seq = np.array([-1, seqs, -FAR - 1, FAR] * rows, np.int32)[:rows]
    pos = np.array([0, FAR, -1, -FAR - 1, 17] * rows, np.int32)[:rows]
    ln = np.array([FAR, 0, -7, top, 33] * rows, np.int32)[:rows]
    for i, r in enumerate(live):
        seq[r], pos[r], ln[r] = i, top - 1 - i, top - i
    q = np.full((rows, heads, hd), filler, np.float32)
    q[live] = rng.standard_normal((len(live), heads, hd))
    x = np.full((rows, (heads + 2 * kvh) * hd), filler, np.float32)
    x[live] = rng.standard_normal((len(live), x.shape[1]))
    o = run_attn(pool, q, seq, ln, heads, 0.125, max_len=top)
    ref, tol = ref_attn(q[live], pool, range(len(live)), ln[live], heads, 0.125)
    assert (np.abs(o[live] - ref) <= tol).all()
    assert (np.delete(o, live, 0) == 7.0).all()
    k0, v0 = pool.k.clone(), pool.v.clone()
    freq = np.ones(hd // 2, np.float32)
    got = run_rope(pool, x, seq, pos, freq, hd, 0, None, None, heads).cpu().numpy().reshape(rows, heads, hd)
    rq, _, _, eq, _ = ref_rope(x[live], pos[live], freq, hd, 0, None, None, 1e-6, heads, kvh, hd)
    assert (np.abs(got[live] - rq) <= eq).all() and (np.delete(got, live, 0) == 7.0).all()
    for i, r in enumerate(live):
        page, slot = int(pool.table[i, pos[r] // 16]), pos[r] % 16
        for new, old in ((pool.k, k0), (pool.v, v0)):
            assert not torch.equal(new[page, :, slot], old[page, :, slot])
            new[page, :, slot] = old[page, :, slot]
    assert torch.equal(pool.k, k0) and torch.equal(pool.v, v0)
