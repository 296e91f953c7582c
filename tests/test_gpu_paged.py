"""The rotation into a cache's pages and the attention over them
(include/mllm.h mllm_rope_kv_paged, mllm_attn_paged) against their formulas in
float64, and a small model's decode step put together from the operators
against the engine.

Tolerances count roundings, u = 2^-24 being half a float32 step:
  rotation   the norm's factor is within 14 u, a cosine or sine within 12 u of
             1, each element adds two rounded products: 32 u (|a| + |b|) of its
             pair, and half a step of the cache's type;
  attention  a score is a sum of hd products, each addition off by at most u of
             the largest partial sum A: a random walk, four standard deviations
             are 4 sqrt(hd) A u, which the numerator and the denominator both
             carry; a weight's exponent X (in powers of two) is rounded twice;
             the sums over n positions walk 4 sqrt(n) u; 32 u for the rest.
"""
import ctypes as C
import math

import numpy as np
import pytest

from mllm import abi, pgw

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}


def p(t):
    return None if t is None else t.data_ptr()


class Pool:
    """Pages in one of the layouts, and a heads-first view [pages][kv][slots][hd]."""

    def __init__(self, g, kv_heads, hd, page, seqs, cols, storage="f16", layout="hnd", fill=None):
        self.page, self.hd, self.kv_heads, self.storage = page, hd, kv_heads, storage
        self.n = seqs * cols + 2
        self.table = torch.randperm(self.n, generator=g)[:seqs * cols].reshape(seqs, cols).to(torch.int32).cuda()
        pad = 8 if layout == "padded" else 0
        shape = ((self.n, page, kv_heads, hd) if layout == "nhd" else (self.n, kv_heads, page + (1 if pad else 0), hd + pad))
        mk = lambda: (torch.randn(shape, generator=g) if fill is None else torch.full(shape, fill)).to(TYPES[storage]).cuda()  # noqa: E731
        self.k, self.v = mk(), mk()
        if layout == "nhd":
            self.strides = (page * kv_heads * hd, hd, kv_heads * hd)
            view = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
        elif layout == "padded":
            self.strides = tuple(self.k.stride()[:3])
            view = lambda t: t[:, :, :page, :hd]  # noqa: E731
        else:
            self.strides = (0, 0, 0)
            view = lambda t: t  # noqa: E731
        self.kh, self.vh = view(self.k), view(self.v)

    def desc(self, table=None):
        t = self.table if table is None else table
        self.kept = t
        return abi.MllmKvPages(p(self.k), p(self.v), CODES[self.storage], self.kv_heads, self.hd, self.n, self.page,
                               *self.strides, p(t), *t.shape)

    def rows(self, which, seq, n):
        """Positions 0 .. n - 1 of a sequence, [n][kv][hd] in float64."""
        pages = self.table[seq, :-(-n // self.page)].long()
        t = (self.kh if which == "k" else self.vh)[pages].double().permute(0, 2, 1, 3)
        return t.reshape(-1, self.kv_heads, self.hd)[:n].cpu().numpy()


# ---------------------------------------------------------------- rotation
def ref_rope(x, pos, freq, rot, inter, gq, gk, eps, heads, kv_heads, hd):
    """q, k, v in float64 and the bound's |a| + |b| for q and k."""
    T = len(pos)
    x = x.astype(np.float64).reshape(T, heads + 2 * kv_heads, hd).copy()
    for sl, gain in ((slice(0, heads), gq), (slice(heads, heads + kv_heads), gk)):
        if gain is not None:
            x[:, sl] = x[:, sl] / np.sqrt((x[:, sl] ** 2).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    size = np.abs(x)
    n = heads + kv_heads
    if rot:
        i = np.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        ang = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)
        xa, xb = x[:, :n, a].copy(), x[:, :n, b].copy()
        x[:, :n, a] = xa * np.cos(ang) - xb * np.sin(ang)
        x[:, :n, b] = xb * np.cos(ang) + xa * np.sin(ang)
        both = size[:, :n, a] + size[:, :n, b]
        size[:, :n, a] = size[:, :n, b] = both
    return x[:, :heads], x[:, heads:n], x[:, n:], 32 * U * size[:, :heads], 32 * U * size[:, heads:n]


def run_rope(pool, x, seq, pos, freq, rot, inter, gq, gk, heads, eps=1e-6, q=None, stream=None):
    T = x.shape[0]
    q = torch.full((T, heads * pool.hd), 7.0, device="cuda") if q is None else q
    dev = [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (x, seq, pos, freq, gq, gk)]
    kv = pool.desc()
    abi.call("mllm_rope_kv_paged", kv, T, heads, p(dev[0]), p(dev[1]), p(dev[2]), p(dev[3]), rot, inter, p(dev[4]), p(dev[5]),
             eps, p(q), stream)
    torch.cuda.synchronize()
    return q


ROPE = [  # heads, kv heads, hd, rot, interleaved, norm, storage, page, layout
    (9, 3, 64, 64, 0, False, "f32", 16, "hnd"), (15, 5, 64, 64, 0, True, "f16", 16, "nhd"),
    (12, 12, 64, 32, 1, False, "f16", 1, "hnd"), (4, 1, 128, 128, 1, True, "bf16", 24, "padded"),
    (4, 4, 96, 24, 0, True, "f16", 7, "hnd"), (3, 1, 32, 32, 0, False, "bf16", 16, "nhd"),
    (2, 2, 256, 64, 1, True, "f32", 5, "padded"), (4, 2, 160, 20, 0, True, "f16", 16, "hnd"),
    (4, 2, 64, 2, 0, False, "f32", 16, "hnd"), (4, 2, 64, 0, 0, True, "f16", 16, "hnd"),
    (40, 8, 224, 50, 1, True, "bf16", 32, "nhd"), (1, 1, 192, 192, 0, False, "f32", 64, "hnd")]


@gpu
@pytest.mark.parametrize("heads,kvh,hd,rot,inter,norm,storage,page,layout", ROPE)
@pytest.mark.parametrize("tokens", [1, 3, 37])
def test_rope_vs_formula(heads, kvh, hd, rot, inter, norm, storage, page, layout, tokens):
    rng = np.random.default_rng(heads * 100 + rot + tokens)
    g = torch.Generator().manual_seed(5)
    seqs, cols = 5, 6
    pool = Pool(g, kvh, hd, page, seqs, cols, storage, layout)
    slots = rng.permutation(seqs * cols * page)[:tokens]
    tokens = len(slots)
    seq, pos = (slots // (cols * page)).astype(np.int32), (slots % (cols * page)).astype(np.int32)
    x = rng.standard_normal((tokens, (heads + 2 * kvh) * hd)).astype(np.float32)
    freq = (1e5 ** (-2.0 * np.arange(max(1, rot // 2)) / max(rot, 1))).astype(np.float32)
    gq, gk = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)] if norm else (None, None)
    k0, v0 = pool.k.clone(), pool.v.clone()
    print(f"rope {heads}/{kvh}x{hd} rot={rot} {storage} page={page} {layout} T={tokens}", flush=True)
    q = run_rope(pool, x, seq, pos, freq if rot else None, rot, inter, gq, gk, heads).cpu().numpy()
    rq, rk, rv, eq, ek = ref_rope(x, pos, freq, rot, inter, gq, gk, 1e-6, heads, kvh, hd)
    assert (np.abs(q.reshape(tokens, heads, hd) - rq) <= eq + 1e-30).all()
    page_of = pool.table.cpu()[torch.from_numpy(seq).long(), torch.from_numpy(pos // page).long()].long()
    slot = torch.from_numpy(pos % page).long()
    gotk = pool.kh[page_of, :, slot].double().cpu().numpy()
    gotv = pool.vh[page_of, :, slot].double().cpu().numpy()
    assert (np.abs(gotk - rk) <= ek * (1 + STEP[storage]) + STEP[storage] * np.abs(rk) + TINY[storage]).all()
    assert np.array_equal(gotv, torch.from_numpy(rv.astype(np.float32)).to(TYPES[storage]).double().numpy())
    # every other slot (and what pads the strides) is what it was
    pool.kh[page_of, :, slot] = torch.zeros((), dtype=TYPES[storage], device="cuda")
    pool.vh[page_of, :, slot] = torch.zeros((), dtype=TYPES[storage], device="cuda")
    k1, v1 = pool.k.clone(), pool.v.clone()
    pool.k.copy_(k0), pool.v.copy_(v0)
    pool.kh[page_of, :, slot] = torch.zeros((), dtype=TYPES[storage], device="cuda")
    pool.vh[page_of, :, slot] = torch.zeros((), dtype=TYPES[storage], device="cuda")
    assert torch.equal(pool.k, k1) and torch.equal(pool.v, v1)


@gpu
def test_rope_far_positions():
    """Angles of positions past 2^20 keep float32's precision (in float32 they
    would be off by a sixteenth of a turn)."""
    g = torch.Generator().manual_seed(6)
    rng = np.random.default_rng(6)
    page, cols = 65536, 32
    pool = Pool(g, 1, 32, page, 1, cols, "f16")
    pos = np.array([0, 1, 1048576, 1999999, 2097151], np.int32)
    x = rng.standard_normal((5, 4 * 32)).astype(np.float32)
    freq = (10000.0 ** (-np.arange(16) / 16.0)).astype(np.float32)
    q = run_rope(pool, x, np.zeros(5, np.int32), pos, freq, 32, 0, None, None, 2).cpu().numpy()
    rq, _, _, eq, _ = ref_rope(x, pos, freq, 32, 0, None, None, 1e-6, 2, 1, 32)
    assert (np.abs(q.reshape(5, 2, 32) - rq) <= eq).all()


@gpu
def test_rope_padding_missing_pages_and_rounding():
    g = torch.Generator().manual_seed(7)
    rng = np.random.default_rng(7)
    pool = Pool(g, 2, 64, 16, 3, 2, "f16", fill=3.0)
    table = pool.table.clone()
    table[1, 0], table[1, 1] = -1, pool.n
    pool.table = table
    # sequences: padding below and above, none of page (1), beyond the table (2, position 32), fine (0)
    seq = np.array([-1, 3, 0, 1, 1, 2, 0], np.int32)
    pos = np.array([4, 4, -1, 0, 20, 32, 5], np.int32)
    x = rng.standard_normal((7, 8 * 64)).astype(np.float32)
    x[6, 4 * 64:] = 70000.0  # keys and values past f16: infinity (rotated: any that stays past it)
    x[6, 6 * 64] = np.nan
    x[6, 6 * 64 + 1] = -1e-8  # below half of f16's least
    freq = np.ones(32, np.float32)
    q = run_rope(pool, x, seq, pos, freq, 64, 0, None, None, 4).cpu().numpy()
    rq, _, _, eq, _ = ref_rope(x, pos, freq, 64, 0, None, None, 1e-6, 4, 2, 64)
    assert (q[:3] == 7.0).all()
    assert (np.abs(q[3:].reshape(4, 4, 64) - rq[3:]) <= eq[3:]).all()
    page = int(table[0, 0])
    v = pool.vh[page, :, 5].float().cpu().numpy()
    assert np.isnan(v[0, 0]) and v[0, 1] == 0.0 and np.isposinf(v[0, 2:]).all() and np.isposinf(v[1]).all()
    pool.kh[page, :, 5] = 3.0
    pool.vh[page, :, 5] = 3.0
    assert bool((pool.k == 3.0).all()) and bool((pool.v == 3.0).all())


@gpu
def test_rope_norm_of_zero_and_of_large_rows():
    """A head of zeros stays zero (eps), a head of 1e15 is normed without
    overflow (its squares' sum is 64e30)."""
    g = torch.Generator().manual_seed(8)
    pool = Pool(g, 1, 64, 16, 1, 1, "f32")
    x = np.zeros((1, 3 * 64), np.float32)
    x[0, 64:128] = 1e15
    gain = np.ones(64, np.float32)
    q = run_rope(pool, x, None, np.array([3], np.int32), np.ones(32, np.float32), 0, 0, gain, gain, 1)
    assert bool((q == 0).all())
    k = pool.kh[int(pool.table[0, 0]), 0, 3].cpu().numpy()
    assert np.abs(k - 1.0).max() <= 16 * U


# ---------------------------------------------------------------- attention
def ref_attn(q, pool, seqs, lens, heads, scale):
    """out in float64 and its bound."""
    out = np.zeros((len(lens), heads, pool.hd))
    tol = np.zeros_like(out)
    rep = heads // pool.kv_heads
    for r, (s, n) in enumerate(zip(seqs, lens)):
        if n <= 0:
            continue
        k, v = pool.rows("k", s, n), pool.rows("v", s, n)
        for h in range(heads):
            qh = q[r, h].astype(np.float64)
            kk, vv = k[:, h // rep], v[:, h // rep]
            sc = scale * (kk @ qh)
            e = sc - sc.max()
            w = np.exp(e)
            w /= w.sum()
            out[r, h] = w @ vv
            big = abs(scale) * (np.abs(kk) @ np.abs(qh)).max()
            walk = 4 * math.sqrt(pool.hd) * big + 4 * (w @ np.abs(e)) * 1.45 + 4 * math.sqrt(n) + 32
            tol[r, h] = U * walk * (w @ np.abs(vv))
    return out, tol


def run_attn(pool, q, seqs, lens, heads, scale, max_len=None, out=None, ws=None, stream=None, table=None):
    R = len(lens)
    dq = torch.from_numpy(np.ascontiguousarray(q.reshape(R, -1))).cuda()
    ds = None if seqs is None else torch.tensor(np.asarray(seqs, np.int32)).cuda()
    dl = torch.tensor(np.asarray(lens, np.int32)).cuda()
    kv = pool.desc(table)
    max_len = max(lens) if max_len is None else max_len
    out = torch.full((R, heads * pool.hd), 7.0, device="cuda") if out is None else out
    n = abi.lib().mllm_attn_paged_workspace(kv, R, heads, max_len)
    if ws is None:
        ws = torch.full((max(n, 16384),), 255, dtype=torch.uint8, device="cuda")  # NaN, where a part were read unwritten
        ws[:16384] = 0
    abi.call("mllm_attn_paged", kv, R, heads, p(dq), p(ds), p(dl), max_len, scale, p(out), p(ws), n, stream)
    torch.cuda.synchronize()
    assert not bool(ws[:16384].any())
    return out.cpu().numpy().reshape(R, heads, pool.hd)


ATTN = [  # heads, kv heads, hd, storage, page, layout, lengths
    (9, 3, 64, "f32", 16, "hnd", [1, 2, 15, 16, 17, 63, 64, 65, 300]),
    (15, 5, 64, "f16", 16, "nhd", [1, 700, 33, 129, 512]), (12, 12, 64, "bf16", 7, "padded", [100, 1, 257]),
    (4, 4, 64, "f16", 1, "hnd", [5, 130]), (8, 1, 64, "f32", 24, "nhd", [200, 49]),
    (20, 1, 64, "f16", 16, "hnd", [90, 3]), (33, 1, 32, "f32", 16, "padded", [70]), (16, 1, 128, "bf16", 32, "hnd", [400, 31]),
    (4, 2, 32, "f16", 16, "hnd", [1000, 40]), (6, 2, 96, "f16", 48, "nhd", [333, 16]), (6, 2, 96, "f32", 16, "hnd", [100]),
    (2, 2, 160, "bf16", 16, "hnd", [77, 128]), (2, 1, 160, "f32", 16, "hnd", [77]), (3, 3, 192, "f16", 5, "hnd", [64, 129]),
    (3, 1, 192, "f32", 16, "hnd", [65]), (4, 2, 224, "f16", 16, "nhd", [50, 80]), (4, 1, 224, "f32", 16, "hnd", [81]),
    (16, 1, 256, "f32", 16, "hnd", [150, 17]), (8, 2, 256, "f16", 16, "padded", [150, 256]), (5, 1, 128, "f32", 16, "hnd", [130]),
    (5, 1, 128, "f16", 16, "hnd", [130]), (2, 1, 64, "bf16", 100, "hnd", [3000, 1, 2999])]


@gpu
@pytest.mark.parametrize("heads,kvh,hd,storage,page,layout,lens", ATTN)
def test_attn_vs_formula(heads, kvh, hd, storage, page, layout, lens):
    g = torch.Generator().manual_seed(heads + hd)
    rng = np.random.default_rng(heads + hd)
    cols = -(-max(lens) // page) + 1
    pool = Pool(g, kvh, hd, page, len(lens), cols, storage, layout)
    q = rng.standard_normal((len(lens), heads, hd)).astype(np.float32)
    scale = 1.0 / math.sqrt(hd)
    print(f"attn {heads}/{kvh}x{hd} {storage} page={page} {layout} lens={lens}", flush=True)
    o = run_attn(pool, q, None, lens, heads, scale)
    ref, tol = ref_attn(q, pool, range(len(lens)), lens, heads, scale)
    assert (np.abs(o - ref) <= tol).all(), float((np.abs(o - ref) / tol).max())


@gpu
def test_attn_many_rows_take_one_part():
    """Rows that fill the chip by themselves are not split; the same rows alone are."""
    g = torch.Generator().manual_seed(11)
    rng = np.random.default_rng(11)
    pool = Pool(g, 4, 64, 16, 300, 9, "f16")
    lens = [int(v) for v in rng.integers(0, 129, 300)]  # a part is 128 positions at least
    q = rng.standard_normal((300, 8, 64)).astype(np.float32)
    assert abi.lib().mllm_attn_paged_workspace(pool.desc(), 300, 8, max(lens)) == 0
    o = run_attn(pool, q, None, lens, 8, 0.125)
    ref, tol = ref_attn(q, pool, range(300), lens, 8, 0.125)
    assert (np.abs(o - ref) <= tol).all()
    for r in (0, 7):
        one = run_attn(pool, q[r:r + 1], [r], lens[r:r + 1], 8, 0.125, max_len=140)
        assert (np.abs(one[0] - ref[r]) <= tol[r]).all()


@gpu
@pytest.mark.parametrize("rows,heads,kvh,hd,storage,page,top", [
    (300, 6, 2, 64, "f16", 16, 512), (200, 24, 3, 64, "bf16", 7, 200), (180, 3, 3, 128, "bf16", 16, 256),
    (530, 12, 1, 64, "f32", 24, 90), (300, 4, 2, 32, "f16", 1, 600), (180, 3, 3, 256, "f32", 16, 64)])
def test_attn_many_short_rows(rows, heads, kvh, hd, storage, page, top):
    """More units than workgroups of four waves fit the chip, each short: a wave
    to a unit; with empty rows, padding, a bad page and a length too long."""
    g = torch.Generator().manual_seed(33)
    rng = np.random.default_rng(33)
    seqs = 40
    pool = Pool(g, kvh, hd, page, seqs, -(-top // page), storage)
    seq = [int(v) for v in rng.integers(0, seqs, rows)]
    lens = [int(v) for v in rng.integers(0, top + 1, rows)]
    lens[:6] = [0, 1, top, top - 1, 2, top]
    seq[:6] = range(6)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    kept = [r for r in range(rows) if r not in (7, 9, 11)]
    seq[7], seq[9] = -1, seqs  # padding
    table = pool.table.clone()
    bad = seqs - 1
    for r in range(rows):
        if seq[r] == bad:
            seq[r] = 0
    seq[11], lens[11] = bad, 1
    table[bad, 0] = pool.k.shape[0]
    out = torch.full((rows, heads * hd), 7.0, device="cuda")
    o = run_attn(pool, q, seq, lens, heads, 0.125, max_len=top, out=out, table=table)
    assert (o[[7, 9]] == 7.0).all() and np.isnan(o[11]).all() and (o[0] == 0).all()
    some = kept[:12] + kept[12::17]
    ref, tol = ref_attn(q[some], pool, [seq[r] for r in some], [lens[r] for r in some], heads, 0.125)
    assert (np.abs(o[some] - ref) <= tol).all()


@gpu
@pytest.mark.parametrize("storage", ["f32", "f16", "bf16"])
def test_attn_infinities_in_many_short_rows(storage):
    """What an infinite key or value does to a row, it does to it in a large batch."""
    g = torch.Generator().manual_seed(34)
    rng = np.random.default_rng(34)
    pool = Pool(g, 2, 64, 16, 6, 8, storage)
    t = pool.table.long()
    pool.k[t[1, 0], 0, 3, 5] = float("inf")
    pool.k[t[2, 1], 1, 0, 7] = float("-inf")
    pool.v[t[3, 2], 1, 1, 9] = float("inf")
    pool.k[t[4, 0], 0, 0] = float("nan")
    q = rng.standard_normal((300, 6, 64)).astype(np.float32)
    seq = [r % 6 for r in range(300)]
    lens = [int(v) for v in rng.integers(40, 129, 300)]
    many = run_attn(pool, q, seq, lens, 6, 0.125, max_len=128)
    few = np.concatenate([run_attn(pool, q[r:r + 12], seq[r:r + 12], lens[r:r + 12], 6, 0.125, max_len=128)
                          for r in range(0, 60, 12)])
    assert np.array_equal(np.isnan(many[:60]), np.isnan(few)) and np.isnan(few).any() and np.isinf(few).any()
    with np.errstate(invalid="ignore"):
        # ref_attn's bound for each: a walk of 4 sqrt(64) max|score| (8) + 4 sqrt(128) + 32 and some, below 350
        # roundings of 2^-24, times at most max|v| (4.5); two of them are below 2^-12
        assert (np.isclose(many[:60], few, rtol=0, atol=2.0 ** -12) | np.isnan(few)).all()


@gpu
@pytest.mark.parametrize("scale", [0.125, 3.0, 0.0, -1.0])
def test_attn_peaked_and_flat_scores(scale):
    g = torch.Generator().manual_seed(12)
    rng = np.random.default_rng(12)
    pool = Pool(g, 2, 64, 16, 2, 30, "f16")
    q = (4 * rng.standard_normal((2, 4, 64))).astype(np.float32)
    o = run_attn(pool, q, None, [470, 211], 4, scale)
    ref, tol = ref_attn(q, pool, range(2), [470, 211], 4, scale)
    assert (np.abs(o - ref) <= tol).all()


@gpu
@pytest.mark.parametrize("rows", [1, 300])
def test_attn_empty_padding_and_bad_rows(rows):
    """Empty rows are 0, padding stays, lengths and pages that cannot be give
    NaN -- in one part (300 rows) and in several, in any part of the length."""
    g = torch.Generator().manual_seed(13)
    rng = np.random.default_rng(13)
    pool = Pool(g, 2, 64, 16, 5, 40, "f16")
    table = pool.table.clone()
    table[2, 39], table[3, 0] = -1, pool.n
    cases = [(0, 0), (-1, 50), (5, 50), (0, -3), (0, 641), (2, 624), (2, 640), (3, 1), (1, 640)]
    if rows > 1:
        cases = cases + [(4, 33)] * (rows - len(cases))
        q = rng.standard_normal((len(cases), 4, 64)).astype(np.float32)
        o = run_attn(pool, q, [s for s, _ in cases], [n for _, n in cases], 4, 0.125, max_len=640, table=table)
    else:
        q = rng.standard_normal((len(cases), 4, 64)).astype(np.float32)
        o = np.concatenate([run_attn(pool, q[i:i + 1], [s], [n], 4, 0.125, max_len=640, table=table)
                            for i, (s, n) in enumerate(cases)])
    assert (o[0] == 0).all()
    assert (o[1] == 7.0).all() and (o[2] == 7.0).all()
    for r in (3, 4, 6, 7):
        assert np.isnan(o[r]).all(), r
    for r in [5] + list(range(8, len(cases))):
        ref, tol = ref_attn(q[r:r + 1], pool, [cases[r][0]], [cases[r][1]], 4, 0.125)
        assert (np.abs(o[r] - ref[0]) <= tol[0]).all(), r


@gpu
@pytest.mark.parametrize("storage", ["f32", "f16", "bf16"])
def test_attn_reads_nothing_behind_the_length(storage):
    """Slots behind the length and free pages hold NaN or infinities: they
    change nothing, in the last page of the length or elsewhere."""
    g = torch.Generator().manual_seed(14)
    rng = np.random.default_rng(14)
    for fill in (float("nan"), float("inf"), -float("inf")):
        pool = Pool(g, 2, 64, 16, 3, 20, storage, fill=fill)
        lens = [1, 131, 300]
        for s, n in enumerate(lens):
            for i in range(n):
                page, slot = int(pool.table[s, i // 16]), i % 16
                pool.kh[page, :, slot] = torch.randn(2, 64, generator=g).to(TYPES[storage]).cuda()
                pool.vh[page, :, slot] = torch.randn(2, 64, generator=g).to(TYPES[storage]).cuda()
        q = rng.standard_normal((3, 6, 64)).astype(np.float32)
        o = run_attn(pool, q, None, lens, 6, 0.125, max_len=320)
        ref, tol = ref_attn(q, pool, range(3), lens, 6, 0.125)
        assert (np.abs(o - ref) <= tol).all()


@gpu
@pytest.mark.parametrize("n", [40, 600])
def test_attn_infinities_within_the_length(n):
    """A key that scores -inf weighs nothing, one that scores +inf or NaN makes
    its heads NaN, every key at -inf is 0 / 0, a value of inf stays inf: as the
    formula has them, and other heads are not touched."""
    g = torch.Generator().manual_seed(15)
    rng = np.random.default_rng(15)
    pool = Pool(g, 4, 64, 16, 5, -(-n // 16), "f16")
    q = np.abs(rng.standard_normal((5, 8, 64))).astype(np.float32)

    def slot(s, i):
        return int(pool.table[s, i // 16]), i % 16

    a, b = slot(0, n // 2)
    pool.kh[a, 0, b, 3] = -math.inf  # heads 0, 1 of row 0: this key weighs 0
    a, b = slot(1, n - 1)
    pool.kh[a, 1, b, 5] = math.inf  # heads 2, 3 of row 1: NaN
    for i in range(n):
        a, b = slot(2, i)
        pool.kh[a, 2, b, 0] = -math.inf  # heads 4, 5 of row 2: 0 / 0
    a, b = slot(3, 1)
    pool.vh[a, 3, b, 7] = math.inf  # heads 6, 7 of row 3: element 7 is inf
    q[4, 1, 0] = np.nan  # head 1 of row 4
    lens = [n] * 5
    o = run_attn(pool, q, None, lens, 8, 0.125)
    with np.errstate(all="ignore"):
        ref, tol = ref_attn(q, pool, range(5), lens, 8, 0.125)
    # row 0, heads 0 and 1: the formula over the other keys
    class Others:
        kv_heads, hd = pool.kv_heads, pool.hd

        @staticmethod
        def rows(which, s, m):
            return np.delete(pool.rows(which, s, m), n // 2, 0)

    with np.errstate(all="ignore"):
        r0, t0 = ref_attn(q[:1], Others, [0], [n], 8, 0.125)
    assert (np.abs(o[0, :2] - r0[0, :2]) <= t0[0, :2]).all()
    assert np.isnan(o[1, 2:4]).all() and np.isnan(o[2, 4:6]).all() and np.isnan(o[4, 1]).all()
    assert np.isposinf(o[3, 6:, 7]).all() and np.isfinite(np.delete(o[3, 6:], 7, -1)).all()
    plain = np.ones((5, 8), bool)
    plain[0, :2] = plain[1, 2:4] = plain[2, 4:6] = plain[3, 6:] = False
    plain[4, 1] = False
    assert (np.abs(o - ref) <= tol)[plain].all()


@gpu
def test_attn_shared_pages_and_speculation_rows():
    """Sequences that share a prefix's pages, and several rows of a sequence."""
    g = torch.Generator().manual_seed(16)
    rng = np.random.default_rng(16)
    pool = Pool(g, 3, 64, 16, 3, 40, "f16")
    pool.table[1, :20] = pool.table[0, :20]
    pool.table[2] = pool.table[0]
    seqs, lens = [0, 1, 2, 0, 0, 0, 1], [640, 500, 333, 511, 512, 513, 320]
    q = rng.standard_normal((7, 9, 64)).astype(np.float32)
    o = run_attn(pool, q, seqs, lens, 9, 0.125)
    ref, tol = ref_attn(q, pool, seqs, lens, 9, 0.125)
    assert (np.abs(o - ref) <= tol).all()


@gpu
def test_attn_calls_of_other_shapes_share_a_workspace():
    g = torch.Generator().manual_seed(20)
    rng = np.random.default_rng(20)
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    for heads, kvh, hd, lens in ((8, 2, 64, [900, 300]), (40, 5, 32, [400] * 30), (4, 4, 128, [5000]), (8, 2, 64, [100, 900])):
        pool = Pool(g, kvh, hd, 16, len(lens), -(-max(lens) // 16), "f16")
        q = rng.standard_normal((len(lens), heads, hd)).astype(np.float32)
        o = run_attn(pool, q, None, lens, heads, 0.125, ws=ws)
        ref, tol = ref_attn(q, pool, range(len(lens)), lens, heads, 0.125)
        assert (np.abs(o - ref) <= tol).all()


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 3e4, 1e9])
@pytest.mark.parametrize("storage", ["f16", "bf16"])
def test_attn_queries_of_any_size(storage, size):
    """Queries far from 1, with elements of very different size in a head."""
    g = torch.Generator().manual_seed(21)
    rng = np.random.default_rng(21)
    pool = Pool(g, 2, 64, 16, 1, 20, storage)
    q = (size * rng.standard_normal((1, 6, 64)) * 2.0 ** rng.uniform(-12, 0, (1, 6, 64))).astype(np.float32)
    o = run_attn(pool, q, None, [310], 6, 1.0 / size)
    ref, tol = ref_attn(q, pool, [0], [310], 6, float(np.float32(1.0 / size)))
    assert (np.abs(o - ref) <= tol).all()


@gpu
def test_offsets_past_32_bits():
    """Pages 5 GiB apart: rotation writes them and attention reads them."""
    heads, kvh, hd, page = 4, 2, 64, 16
    stride = 5 << 29  # elements of 2 bytes
    buf = torch.zeros(2 * stride + kvh * page * hd, dtype=torch.float16, device="cuda")
    vbuf = torch.zeros_like(buf)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    kv = abi.MllmKvPages(p(buf), p(vbuf), 1, kvh, hd, 3, page, stride, page * hd, hd, p(table), 1, 3)
    rng = np.random.default_rng(17)
    n = 45
    x = rng.standard_normal((n, (heads + 2 * kvh) * hd)).astype(np.float32)
    dx = torch.from_numpy(x).cuda()
    seq, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    q = torch.empty(n, heads * hd, device="cuda")
    abi.call("mllm_rope_kv_paged", kv, n, heads, p(dx), p(seq), p(pos), None, 0, 0, None, None, 0.0, p(q), None)
    out = torch.empty(1, heads * hd, device="cuda")
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    nb = abi.lib().mllm_attn_paged_workspace(kv, 1, heads, n)
    ws = torch.zeros(max(nb, 16), dtype=torch.uint8, device="cuda")
    abi.call("mllm_attn_paged", kv, 1, heads, p(q[3:4]), None, p(ln), n, 0.125, p(out), p(ws), nb, None)
    torch.cuda.synchronize()
    assert torch.equal(q, dx[:, :heads * hd])

    class Flat:  # the slots in order of position
        pass

    pl = Flat()
    pl.kv_heads, pl.hd = kvh, hd
    pl.rows = lambda w, s, m: x[:m].reshape(m, -1, hd)[:, heads + (0 if w == "k" else kvh):][:, :kvh].astype(np.float16).astype(np.float64)
    ref, tol = ref_attn(x[3:4].reshape(1, -1, hd)[:, :heads], pl, [0], [n], heads, 0.125)
    assert (np.abs(out.cpu().numpy().reshape(1, heads, hd) - ref) <= tol).all()


@gpu
def test_captured_step_replays_with_new_lengths():
    """Rotation, attention (in parts) and the draw captured into one graph and
    replayed as the sequences grow, against eager calls on another stream."""
    g = torch.Generator().manual_seed(18)
    R, heads, kvh, hd, V = 3, 6, 2, 64, 2000
    pools = [Pool(g, kvh, hd, 16, R, 64, "f16", fill=0.0) for _ in range(2)]
    pools[1].table = pools[0].table.clone()
    x = torch.zeros(R, (heads + 2 * kvh) * hd, device="cuda")
    pos, ln = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")
    freq = (1e4 ** (-torch.arange(32) / 32.0)).float().cuda()
    logits, u = torch.zeros(R, V, device="cuda"), torch.zeros(R, device="cuda")

    def buffers(pool):
        kv = pool.desc()
        n = abi.lib().mllm_attn_paged_workspace(kv, R, heads, 1024)
        assert n > 0
        return (kv, torch.zeros(R, heads * hd, device="cuda"), torch.zeros(R, heads * hd, device="cuda"),
                torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda"))

    def step(b, st):
        kv, q, out, ids, ws = b
        abi.call("mllm_rope_kv_paged", kv, R, heads, p(x), None, p(pos), p(freq), 64, 0, None, None, 1e-6, p(q), st)
        abi.call("mllm_attn_paged", kv, R, heads, p(q), None, p(ln), 1024, 0.125, p(out), p(ws), ws.numel(), st)
        abi.call("mllm_sample", R, V, p(logits), None, None, None, None, p(u), p(ids), None, st)

    cap, eager = buffers(pools[0]), buffers(pools[1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cap, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for t in range(6):
        x.copy_(torch.randn(x.shape, generator=g))
        logits.copy_(torch.randn(logits.shape, generator=g))
        u.copy_(torch.rand(R, generator=g))
        pos.copy_(torch.tensor([t, 100 * t, 17 * t]))
        ln.copy_(pos + 1)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            step(eager, side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].v, pools[1].v)
        assert torch.equal(cap[1], eager[1]) and torch.equal(cap[2], eager[2]) and torch.equal(cap[3], eager[3]), t


@gpu
def test_steps_on_two_streams_at_once():
    """Steps of two batches, each on its stream with its own workspace, against
    the same steps one after another."""
    g = torch.Generator().manual_seed(31)
    rng = np.random.default_rng(31)
    heads, kvh, hd, V = 6, 2, 64, 3001
    lens = ([700, 3, 1500, 64], [900, 1200])
    freq = (1e4 ** (-torch.arange(32) / 32.0)).float().cuda()
    dev = lambda a, t: torch.tensor(a, dtype=t, device="cuda")  # noqa: E731
    batch = []
    for ls in lens:
        R = len(ls)
        pool = Pool(g, kvh, hd, 16, R, 100, "f16", fill=0.5)
        nb = abi.lib().mllm_attn_paged_workspace(pool.desc(), R, heads, 1600)
        batch.append(dict(R=R, pool=pool, ln=dev(ls, torch.int32), pos=dev([n - 1 for n in ls], torch.int32),
                          x=torch.from_numpy(rng.standard_normal((R, (heads + 2 * kvh) * hd)).astype(np.float32)).cuda(),
                          z=torch.from_numpy(rng.standard_normal((R, V)).astype(np.float32)).cuda(), u=torch.rand(R).cuda(),
                          ws=torch.zeros(nb, dtype=torch.uint8, device="cuda"),
                          k=dev([40] * R, torch.int32), tp=torch.full((R,), 0.9, device="cuda")))

    def step(b, st):
        R = b["R"]
        q, o = torch.zeros(R, heads * hd, device="cuda"), torch.zeros(R, heads * hd, device="cuda")
        ids = torch.zeros(R, dtype=torch.int32, device="cuda")
        kv = b["pool"].desc()

        def go():
            abi.call("mllm_rope_kv_paged", kv, R, heads, p(b["x"]), None, p(b["pos"]), p(freq), 64, 0, None, None, 0.0, p(q), st)
            abi.call("mllm_attn_paged", kv, R, heads, p(q), None, p(b["ln"]), 1600, 0.125, p(o), p(b["ws"]), b["ws"].numel(), st)
            abi.call("mllm_sample", R, V, p(b["z"]), None, p(b["k"]), p(b["tp"]), None, p(b["u"]), p(ids), None, st)
        return go, (q, o, ids)

    want = []
    for b in batch:
        go, out = step(b, None)
        go()
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = [[step(b, st.cuda_stream) for b, st in zip(batch, streams)] for _ in range(8)]
    torch.cuda.synchronize()
    for run in runs:
        for go, _ in run:
            go()
    torch.cuda.synchronize()
    for run in runs:
        for (_, out), w in zip(run, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
    assert all(int(b["ws"][:16384].sum()) == 0 for b in batch)


@gpu
def test_attn_a_workspace_for_the_largest_call():
    """One workspace, sized for the most rows and positions, for every smaller
    call; the counters at its head stay zero."""
    g = torch.Generator().manual_seed(32)
    rng = np.random.default_rng(32)
    pool = Pool(g, 2, 64, 16, 40, 375, "f16")
    nb = abi.lib().mllm_attn_paged_workspace(pool.desc(), 40, 8, 6000)
    ws = torch.zeros(nb, dtype=torch.uint8, device="cuda")
    for lens in ([6000, 10], [257], [300] * 40, [2000, 0, 5999, 1, 4000, 256]):
        q = rng.standard_normal((len(lens), 8, 64)).astype(np.float32)
        assert abi.lib().mllm_attn_paged_workspace(pool.desc(), len(lens), 8, max(lens)) <= nb
        o = run_attn(pool, q, None, lens, 8, 0.125, ws=ws)
        ref, tol = ref_attn(q, pool, range(len(lens)), lens, 8, 0.125)
        assert (np.abs(o - ref) <= tol).all(), lens
        assert int(ws[:16384].sum()) == 0


# ---------------------------------------------------------------- a model's step
class PagedLlama:
    """A llama bundle's decode step for several sequences, from the operators."""

    def __init__(self, bundle, seqs, page=16, storage="f32"):
        self.c = c = bundle.cfg
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.w = {}
        for name, t in bundle.tensors.items():
            a = dev(np.array(bundle.array(name)))
            self.w[name] = (a, dev(np.array(bundle.scales(name))).reshape(t["shape"][0], -1)) if t["storage"] == "q4" else a
        self.emb = torch.empty(c.vocab_size, c.d_model, device="cuda")
        q, s = self.w["lm_head"]
        abi.call("mllm_dequant_q4", c.vocab_size, c.d_model, p(q), p(s), 32, p(self.emb), None)
        self.hd = c.d_model // c.n_heads
        g = torch.Generator().manual_seed(1)
        cols = -(-c.max_seq_len // page)
        self.pools = [Pool(g, c.n_kv_heads, self.hd, page, seqs, cols, storage, fill=float("nan")) for _ in range(c.n_layers)]
        half = np.arange(self.hd // 2)
        self.freq = dev((1.0 / c.rope_theta ** (2.0 * half / self.hd)).astype(np.float32))

    def gemm(self, name, x):
        q, s = self.w[name]
        m, n = s.shape[0], s.shape[1] * 32
        y = torch.empty(x.shape[0], m, device="cuda")
        abi.call("mllm_gemm_q4", x.shape[0], m, n, p(q), p(s), 32, p(x), p(y), None)
        return y

    def norm(self, name, x):
        y = torch.empty_like(x)
        abi.call("mllm_rms_norm", x.shape[1], p(x), p(self.w[name]), p(y), x.shape[0], 1e-6, None)
        return y

    def logits(self, ids, seqs, pos):
        """The rows' logits; their keys and values enter the pages."""
        c = self.c
        ds, dp = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in (seqs, pos))
        ln, T = dp + 1, len(ids)
        x = self.emb[torch.tensor(ids, device="cuda")].clone()
        for i, pool in enumerate(self.pools):
            b = f"blocks.{i}."
            qkv = self.gemm(b + "attn.qkv", self.norm(b + "norm1", x))
            q, o = torch.empty(T, c.d_model, device="cuda"), torch.empty(T, c.d_model, device="cuda")
            kv = pool.desc()
            abi.call("mllm_rope_kv_paged", kv, T, c.n_heads, p(qkv), p(ds), p(dp), p(self.freq), self.hd, 0, None, None, 0.0,
                     p(q), None)
            n = abi.lib().mllm_attn_paged_workspace(kv, T, c.n_heads, max(pos) + 1)
            ws = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda")
            abi.call("mllm_attn_paged", kv, T, c.n_heads, p(q), p(ds), p(ln), max(pos) + 1, 1.0 / math.sqrt(self.hd), p(o),
                     p(ws), n, None)
            x = x + self.gemm(b + "attn.proj", o)
            h = self.norm(b + "norm2", x)
            a, up = self.gemm(b + "mlp.w1", h), self.gemm(b + "mlp.w3", h)
            abi.call("mllm_silu_mul", a.numel(), p(a), p(up), None)
            x = x + self.gemm(b + "mlp.w2", a)
        return self.gemm("lm_head", self.norm("norm_f", x))


@gpu
def test_batched_decode_from_operators_equals_the_engine():
    """Three sequences of different lengths, decoded greedily in one batch:
    prompts as rows of one call, then a token each. The engine decodes each of
    them alone. Both round activations to 24 bits per group and sum in float32,
    in other orders: logits within 2e-5 of their scale, as the engine's own
    prompt and decode paths agree."""
    import mllm

    cfg = pgw.small_config("llama", n_layers=3, d_model=192, n_heads=3, n_kv_heads=1, d_ff=256, max_seq_len=96)
    bundle = pgw.parse_pgw(pgw.make_llama(cfg, seed=3, std=0.08))
    rng = np.random.default_rng(19)
    prompts = [[int(v) for v in rng.integers(0, cfg.vocab_size, n)] for n in (1, 23, 40)]
    m = PagedLlama(bundle, 3)
    ids = [t for pr in prompts for t in pr]
    seqs = [s for s, pr in enumerate(prompts) for _ in pr]
    pos = [i for pr in prompts for i in range(len(pr))]
    last = np.cumsum([len(pr) for pr in prompts]) - 1
    lg = m.logits(ids, seqs, pos)[torch.tensor(last, device="cuda")].contiguous()
    steps, toks = [lg], []
    greedy, u = torch.zeros(3, device="cuda"), torch.full((3,), 0.5, device="cuda")
    for t in range(12):
        nxt = torch.empty(3, dtype=torch.int32, device="cuda")
        abi.call("mllm_sample", 3, cfg.vocab_size, p(steps[-1]), p(greedy), None, None, None, p(u), p(nxt), None, None)
        toks.append(nxt.tolist())
        steps.append(m.logits(toks[-1], [0, 1, 2], [len(pr) + t for pr in prompts]))
    torch.cuda.synchronize()
    for s, pr in enumerate(prompts):
        e = mllm.PetitGPT(bundle)
        want = e.forwardPrompt(pr).copy()
        for t in range(13):
            got = steps[t][s].cpu().numpy()
            assert np.abs(got - want).max() <= 2e-5 * np.abs(want).max(), (s, t)
            if t < 12:
                assert toks[t][s] == int(np.argmax(got))
                want = e.forwardDecode(toks[t][s]).copy()
        e.destroy()
