"""The attention over pages in every form that its plan can launch, and the
edges of what mllm_rope_kv_paged and mllm_attn_paged document
(include/mllm.h).  Tolerances: test_gpu_paged.ref_attn's and ref_rope's.
"""
import math

import numpy as np
import pytest

from mllm import abi
from test_gpu_paged import TYPES, Pool, p, ref_attn, ref_rope, run_attn, run_rope

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


# ---------------------------------------------------------------- the plan's forms
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
STORAGES = ["f32", "f16", "bf16"]
MALL = 256 << 20   # more cache than this is read past the caches
SHORT = 128 << 10  # a wave to a unit: rows of at most this many bytes a head ...
MANY = 512         # ... and more units than this


def most_heads(storage, hd):
    """Query heads of a workgroup at most: 16, or 8 where a lane has more than
    8 elements of a value."""
    es, lanes = SIZE[storage], 4
    while lanes * 16 < hd * es:
        lanes *= 2
    while lanes > 64 or hd % lanes or hd // lanes * es % 4:
        lanes //= 2
    return 16 if hd // lanes <= 8 else 8


def parts_of(pool, rows, heads, max_len):
    """The parts that the library's plan takes, from the workspace it asks for."""
    kv, at = pool.desc(), p(pool.k)
    rc = abi.lib().mllm_attn_paged(kv, rows, heads, at, at, at, max_len, 1.0, None, at, 0, None)  # refused: no out
    msg = abi.lib().mllm_last_error().decode()
    assert rc == 1
    if "needed" not in msg:
        assert "null pointer" in msg
        return 1
    rep, most = heads // pool.kv_heads, most_heads(pool.storage, pool.hd)
    part = (min(rep, most) * (pool.hd + 2) + 3) // 4 * 4 * 4
    units = rows * pool.kv_heads * -(-rep // most)
    parts, rest = divmod(int(msg.split(" bytes, ")[1].split()[0]) - 16384, units * part)
    assert rest == 0
    return parts


def holds(pool, q, seq, lens, heads, scale, max_len, some=None):
    o = run_attn(pool, q, seq, lens, heads, scale, max_len=max_len)
    some = list(range(len(lens))) if some is None else some
    seqs = range(len(lens)) if seq is None else seq
    ref, tol = ref_attn(q[some], pool, [seqs[r] for r in some], [lens[r] for r in some], heads, scale)
    assert (np.abs(o[some] - ref) <= tol).all(), float((np.abs(o[some] - ref) / np.maximum(tol, 1e-38)).max())


class LargePool(Pool):
    """A pool past the Infinity Cache's size, made on the device; the sequences'
    pages are drawn from all of it."""

    def __init__(self, hd, storage, page, seqs, cols, seed):
        self.page, self.hd, self.kv_heads, self.storage, self.strides = page, hd, 1, storage, (0, 0, 0)
        es = SIZE[storage]
        self.n = MALL // (2 * hd * es * page) + 9
        g = torch.Generator(device="cuda").manual_seed(seed)
        dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[storage]
        self.k, self.v = (torch.empty(self.n, 1, page, hd, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2))
        self.table = torch.randint(0, self.n, (seqs, cols), generator=g, device="cuda").to(torch.int32)
        self.kh, self.vh = self.k, self.v


def head_counts(storage, hd):
    """For the kernels of up to 4, 8 and (where there is one) 16 heads."""
    return [3, 7] + ([13] if most_heads(storage, hd) > 8 else [])


HDS = [32, 64, 96, 128, 160, 192, 224, 256]


@gpu
@pytest.mark.parametrize("hd", HDS)
@pytest.mark.parametrize("storage", STORAGES)
def test_attn_every_kernel_in_parts(storage, hd):
    """Rows in several parts, joined: lengths in the first part, at its end and in all of them."""
    g = torch.Generator().manual_seed(hd)
    rng = np.random.default_rng(hd)
    pool = Pool(g, 1, hd, 16, 5, 57, storage)
    lens = [900, 1, 0, 128, 611]
    for heads in head_counts(storage, hd) + [most_heads(storage, hd) + 2]:
        assert parts_of(pool, 5, heads, 900) > 1
        print(f"parts {storage} {hd} heads={heads}", flush=True)
        holds(pool, rng.standard_normal((5, heads, hd)).astype(np.float32), None, lens, heads, 1 / math.sqrt(hd), 900)


@gpu
@pytest.mark.parametrize("hd", HDS)
@pytest.mark.parametrize("storage", STORAGES)
def test_attn_every_kernel_of_one_wave(storage, hd):
    g = torch.Generator().manual_seed(hd + 1)
    rng = np.random.default_rng(hd + 1)
    top = min(150, SHORT // (2 * hd * SIZE[storage]))
    rows, seqs = MANY + 9, 24
    pool = Pool(g, 1, hd, 16, seqs, -(-top // 16), storage)
    seq = [int(v) for v in rng.integers(0, seqs, rows)]
    lens = [int(v) for v in rng.integers(0, top + 1, rows)]
    lens[:4] = [top, 0, 1, top - 1]
    for heads in head_counts(storage, hd):
        assert parts_of(pool, rows, heads, top) == 1
        print(f"one wave {storage} {hd} heads={heads}", flush=True)
        holds(pool, rng.standard_normal((rows, heads, hd)).astype(np.float32), seq, lens, heads, 1 / math.sqrt(hd), top,
              some=list(range(8)) + [rows // 2, rows - 1])


@gpu
@pytest.mark.parametrize("hd", HDS)
@pytest.mark.parametrize("storage", STORAGES)
def test_attn_every_kernel_past_the_caches(storage, hd):
    """More cache than the Infinity Cache holds, in long parts: a row of two
    parts and a bit, a short one, an empty one."""
    page = 128
    max_len = MALL // (3 * 2 * hd * SIZE[storage]) + 999
    pool = LargePool(hd, storage, page, 3, -(-max_len // page), hd)
    rng = np.random.default_rng(hd + 2)
    assert min(3 * max_len, pool.n * page) * 2 * hd * SIZE[storage] > MALL
    for heads in head_counts(storage, hd):
        parts = parts_of(pool, 3, heads, max_len)
        assert parts > 1
        lens = [2 * (max_len // parts) + 300, 70, 0]
        print(f"stream {storage} {hd} heads={heads} parts={parts} lens={lens}", flush=True)
        holds(pool, rng.standard_normal((3, heads, hd)).astype(np.float32), None, lens, heads, 1 / math.sqrt(hd), max_len)


@gpu
@pytest.mark.parametrize("storage,hd,heads,cols", [
    ("f16", 64, 3, 940), ("f32", 64, 3, 940), ("bf16", 128, 4, 940), ("f32", 128, 7, 700), ("f16", 64, 16, 940),
    ("bf16", 64, 13, 940), ("f16", 256, 8, 400)])
def test_attn_joins_of_more_than_64_parts(storage, hd, heads, cols):
    """A join takes its parts 64 at a time: all of them there, 65 and fewer."""
    g = torch.Generator().manual_seed(51)
    rng = np.random.default_rng(51)
    pool = Pool(g, 1, hd, 64, 1, cols, storage)
    top = cols * 64
    parts = parts_of(pool, 1, heads, top)
    assert parts > 64
    chunk = -(-top // parts)  # about: whole 128s
    for n in (top, top - 1, 65 * chunk + 7, 5 * chunk, 1):
        holds(pool, rng.standard_normal((1, heads, hd)).astype(np.float32), None, [n], heads, 1 / math.sqrt(hd), top)


@gpu
@pytest.mark.parametrize("storage,hd,heads", [("f16", 32, 8), ("f32", 32, 20), ("bf16", 32, 36), ("f16", 64, 32), ("f32", 64, 8)])
def test_attn_parts_of_more_than_2048_positions(storage, hd, heads):
    """A workgroup of four waves looks up 2048 places at a time."""
    g = torch.Generator().manual_seed(52)
    rng = np.random.default_rng(52)
    pool = Pool(g, 4, hd, 24, 6, 210, storage)
    rows, top = 64, 5000
    lens = [0, 1, 2047, 2048, 2049, 2200, 4095, 4096, 4097, 5000] + [int(v) for v in rng.integers(0, top + 1, rows - 10)]
    seq = [int(v) for v in rng.integers(0, 6, rows)]
    assert top // parts_of(pool, rows, heads, top) > 2048
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    holds(pool, q, seq, lens, heads, 1 / math.sqrt(hd), top, some=list(range(14)))


@gpu
@pytest.mark.parametrize("storage,heads,kvh,hd", [("f32", 9, 3, 64), ("f32", 4, 1, 128), ("f32", 15, 5, 64), ("bf16", 9, 3, 64)])
@pytest.mark.parametrize("lens", [[700], [3000], [257, 1500, 700]])
def test_attn_rows_of_a_chat_in_parts(storage, heads, kvh, hd, lens):
    """The engine's default storage and shapes at a chat's lengths."""
    g = torch.Generator().manual_seed(53)
    rng = np.random.default_rng(53)
    pool = Pool(g, kvh, hd, 16, len(lens), -(-max(lens) // 16), storage)
    assert parts_of(pool, len(lens), heads, max(lens)) > 1
    holds(pool, rng.standard_normal((len(lens), heads, hd)).astype(np.float32), None, lens, heads, 1 / math.sqrt(hd), max(lens))


@gpu
@pytest.mark.parametrize("top", [512, 700])
def test_attn_rows_that_fill_the_chip_are_not_split(top):
    """300 rows of 4 KV heads run in one part, without a workspace; one of them
    alone is split, and refused without one."""
    g = torch.Generator().manual_seed(54)
    rng = np.random.default_rng(54)
    rows, heads, alone = 300, 8, 900
    pool = Pool(g, 4, 64, 16, 20, -(-alone // 16), "f16")
    seq = [r % 20 for r in range(rows)]
    lens = [int(v) for v in rng.integers(0, top + 1, rows)]
    lens[0], lens[7] = top, top - 3
    q = rng.standard_normal((rows, heads, 64)).astype(np.float32)
    dev = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
    dq, ds, dl = dev(q.reshape(rows, -1), torch.float32), dev(seq, torch.int32), dev(lens, torch.int32)
    out, kv = torch.full((rows, heads * 64), 7.0, device="cuda"), pool.desc()
    abi.call("mllm_attn_paged", kv, rows, heads, p(dq), p(ds), p(dl), top, 0.125, p(out), None, 0, None)
    torch.cuda.synchronize()
    o = out.cpu().numpy().reshape(rows, heads, 64)
    some = [0, 7, 8, 150, 299]
    ref, tol = ref_attn(q[some], pool, [seq[r] for r in some], [lens[r] for r in some], heads, 0.125)
    assert (np.abs(o[some] - ref) <= tol).all()
    assert parts_of(pool, 1, heads, alone) > 1
    for i, r in enumerate(some[:2]):
        assert abi.lib().mllm_attn_paged(kv, 1, heads, p(dq), p(ds), p(dl), alone, 0.125, p(out), None, 0, None) == 1
        assert b"needed" in abi.lib().mllm_last_error()
        one = run_attn(pool, q[r:r + 1], [seq[r]], [lens[r]], heads, 0.125, max_len=alone)
        assert (np.abs(one[0] - ref[i]) <= tol[i]).all()


@gpu
@pytest.mark.parametrize("storage,hd", [("f32", 64), ("bf16", 128), ("f32", 256)])
@pytest.mark.parametrize("rows,n", [(1, 700), (1, 64), (600, 64), (150, 700)])
def test_attn_values_at_the_documented_bound(storage, hd, rows, n):
    """Values of 2^116 / length, of one sign in an element, under weights of
    nearly e^8: each wave's first 16 positions score 0, the others 255 / 32.
    The sums come to 2^127.4 and stay finite."""
    g = torch.Generator().manual_seed(61)
    rng = np.random.default_rng(61)
    pool = Pool(g, 4, hd, 16, 1, -(-n // 16), storage)
    many = rows > 100
    assert many or n == 64 or parts_of(pool, rows, 4, n) > 1
    big = math.floor(2.0 ** 116 / n / 2.0 ** 100) * 2.0 ** 100
    big = float(int(big / 2.0 ** (math.frexp(big)[1] - 8))) * 2.0 ** (math.frexp(big)[1] - 8)  # eight bits, for bf16
    v = torch.from_numpy(rng.choice([-big, big], (4, n, hd)))
    v[:, :, 0], v[:, :, 1] = big, -big
    pool.kh.zero_()
    for i in range(n):
        page, slot = int(pool.table[0, i // 16]), i % 16
        pool.kh[page, :, slot, 0] = 0.0 if (i if many else i % 128) < 64 and n > 64 or i < 16 else 255 / 32
        pool.vh[page, :, slot] = v[:, i].to(TYPES[storage]).cuda()
    q = np.zeros((rows, 4, hd), np.float32)
    q[:, :, 0] = 8.0
    some = [0, rows - 1]
    holds(pool, q, [0] * rows, [n] * rows, 4, 0.125, n, some=some)


@gpu
@pytest.mark.parametrize("inter", [0, 1])
def test_rope_angles_keep_double_precision(inter):
    """Heads of (1, 0) in each pair are (cos, sin) after the rotation.  The angle
    comes in double, so they are the float functions' values (1 step at most) and
    one addition (half a step): 1.5 steps of the value.  For values near 0 there
    are the part that two float parts of the angle leave, 2^-47, and the angle's
    own roundings in double, half a step of it each: 1 / (2 pi), its product with
    the frequency, that with the position, and the oracle's product."""
    hd, T = 64, 4096
    g = torch.Generator().manual_seed(71)
    rng = np.random.default_rng(71)
    pool = Pool(g, 1, hd, 1024, 1, 64, "f32")
    pos = rng.permutation(65536)[:T].astype(np.int32)
    freq = rng.uniform(0.0, 3.0, hd // 2).astype(np.float32)
    x = np.zeros((T, 3, hd), np.float32)
    i = np.arange(hd // 2)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + hd // 2)
    x[:, :, a] = 1.0
    q = run_rope(pool, x.reshape(T, -1), np.zeros(T, np.int32), pos, freq, hd, inter, None, None, 1).cpu().numpy()
    ang = pos.astype(np.float64)[:, None] * freq.astype(np.float64)
    for got, want in ((q[:, a], np.cos(ang)), (q[:, b], np.sin(ang))):
        err = np.abs(got - want)
        step = np.spacing(np.abs(want).astype(np.float32)).astype(np.float64)
        tol = 1.5 * step + 2.0 ** -47 + 4 * 2.0 ** -53 * ang
        assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))


@gpu
@pytest.mark.parametrize("rows", [3, 600])
def test_attn_no_positions_at_all(rows):
    """max_len 0: empty rows are 0, padding stays, any length is too long."""
    g = torch.Generator().manual_seed(81)
    pool = Pool(g, 2, 64, 16, 5, 1, "f16", fill=float("nan"))
    seq, lens = [r % 5 for r in range(rows)], [0] * rows
    seq[1], lens[2] = -1, 1
    o = run_attn(pool, np.ones((rows, 4, 64), np.float32), seq, lens, 4, 0.125, max_len=0)
    assert (o[1] == 7.0).all() and np.isnan(o[2]).all() and (np.delete(o, [1, 2], 0) == 0).all()


@gpu
@pytest.mark.parametrize("storage,low", [("f16", -20), ("f16", -15), ("bf16", -128)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attn_subnormal_keys_and_values(storage, low, which):
    """Keys or values below the type's least normal number count for what they are."""
    g = torch.Generator().manual_seed(91)
    rng = np.random.default_rng(91)
    pool = Pool(g, 2, 64, 16, 1, 20, storage)
    t = pool.k if which == "k" else pool.v
    t.copy_((t.double() * 2.0 ** low).to(t.dtype))
    up = min(-low, 100) if which == "k" else 0
    scale = 0.125 * 2.0 ** ((-low if which == "k" else 0) - up)
    q = (rng.standard_normal((1, 6, 64)) * 2.0 ** up).astype(np.float32)
    holds(pool, q, None, [310], 6, scale, 310)
