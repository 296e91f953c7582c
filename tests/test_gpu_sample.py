"""mllm_sample against the definition in float64 (include/mllm.h): the same
token for every row, and its probability within a float32 rounding."""
import math

import numpy as np
import pytest

from mllm import abi

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def p(t):
    return None if t is None else t.data_ptr()


def ref_row(z, temp, k, top_p, min_p, u):
    """(id, probability) of one row."""
    z = z.astype(np.float64)
    z[np.isnan(z)] = -np.inf
    best = int(np.argmax(z))
    if z[best] == -np.inf:
        return 0, 0.0
    if not temp > 0:
        return best, 1.0
    with np.errstate(all="ignore"):
        d = np.where(z == z[best], 0.0, z - z[best])
        w = np.exp(d / temp)
    w = np.where(z == -np.inf, 0.0, w)
    order = np.argsort(-z, kind="stable")
    n = len(z) if k <= 0 else min(k, len(z))
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order[:n]])])
        n = max(1, int(np.count_nonzero(before[:n] < max(top_p, 0) * before[n])))
    keep = order[:n]
    keep = keep[(w[keep] >= min_p) | (keep == order[0])]
    keep = np.sort(keep)
    cum = np.cumsum(w[keep])
    if u >= 1:
        j = int(np.nonzero(w[keep] >= 2.0 ** -44)[0][-1])
    else:
        j = min(int(np.searchsorted(cum, (u if u > 0 else 0.0) * cum[-1], side="right")), len(keep) - 1)
    return int(keep[j]), w[keep[j]] / cum[-1]


def run(z, temp=None, k=None, top_p=None, min_p=None, u=None, probs=True, stream=None):
    z = np.ascontiguousarray(z, np.float32)
    R, V = z.shape
    dev = lambda a, t: None if a is None else torch.from_numpy(np.broadcast_to(np.asarray(a, t), (R,)).copy()).cuda()  # noqa: E731
    dz = torch.from_numpy(z).cuda()
    a = [dev(temp, np.float32), dev(k, np.int32), dev(top_p, np.float32), dev(min_p, np.float32), dev(u, np.float32)]
    ids = torch.full((R,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((R,), -7.0, device="cuda") if probs else None
    print(f"sample {R}x{V} temp={temp is not None} k={k is not None} p={top_p is not None} m={min_p is not None}", flush=True)
    abi.call("mllm_sample", R, V, p(dz), *[p(t) for t in a], p(ids), p(pr), stream)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), pr.cpu().numpy() if probs else None


def check(z, temp=None, k=None, top_p=None, min_p=None, u=None):
    ids, pr = run(z, temp, k, top_p, min_p, u)
    R = len(z)
    at = lambda a, r, off: off if a is None else np.broadcast_to(np.asarray(a, np.float32), (R,))[r]  # noqa: E731
    for r in range(R):
        want, wp = ref_row(z[r], float(at(temp, r, 1.0)), int(at(k, r, 0)), float(at(top_p, r, 1.0)),
                           float(at(min_p, r, 0.0)), float(at(u, r, 0.0)))
        assert ids[r] == want, (r, ids[r], want)
        # a rounding to float32 and the weights' 2^-45
        assert abs(pr[r] - wp) <= wp * 2.0 ** -24 * 1.01 + 2.0 ** -44, (r, pr[r], wp)


VOCABS = [1, 2, 3, 63, 64, 255, 256, 257, 1000, 4097, 16384, 49152, 50257, 65536, 65537, 131072, 151937, 524288]


@gpu
@pytest.mark.parametrize("vocab", VOCABS)
def test_sample_vs_definition(vocab):
    rng = np.random.default_rng(vocab)
    R = 12
    z = (2.5 * rng.standard_normal((R, vocab))).astype(np.float32)
    u = rng.random(R).astype(np.float32)
    temp = rng.uniform(0.3, 1.6, R).astype(np.float32)
    check(z, u=u)
    check(z, temp=temp, u=u)
    check(z, temp=temp, k=rng.integers(1, 60, R), u=u)
    check(z, temp=temp, top_p=rng.uniform(0.3, 1.0, R), u=u)
    check(z, temp=temp, min_p=rng.uniform(0.0, 0.4, R), u=u)
    check(z, temp=temp, k=rng.integers(1, max(2, vocab), R), top_p=rng.uniform(0.5, 1.0, R),
          min_p=rng.uniform(0.0, 0.1, R), u=u)


@gpu
@pytest.mark.parametrize("levels", [1, 2, 5, 200])
@pytest.mark.parametrize("vocab", [300, 5000, 50257, 70001])
def test_sample_ties_by_index(vocab, levels):
    """Logits of a few values: the filters cut through tokens that tie."""
    rng = np.random.default_rng(vocab + levels)
    R = 16
    z = (rng.integers(0, levels, (R, vocab)) / 8.0 - 1).astype(np.float32)
    u = rng.random(R).astype(np.float32)
    check(z, k=rng.integers(1, vocab, R), u=u)
    check(z, top_p=rng.uniform(0.1, 1.0, R), u=u)
    check(z, k=rng.integers(1, vocab, R), top_p=rng.uniform(0.1, 1.0, R), min_p=np.full(R, 0.9), u=u)


@gpu
@pytest.mark.parametrize("vocab", [700, 50257, 100001])
def test_sample_masks_and_non_numbers(vocab):
    rng = np.random.default_rng(vocab)
    R = 12
    z = (2 * rng.standard_normal((R, vocab))).astype(np.float32)
    z[0, rng.random(vocab) < 0.9] = -np.inf
    z[1, :] = -np.inf
    z[2, :] = np.nan
    z[3, rng.random(vocab) < 0.5] = np.nan
    z[4, rng.random(vocab) < 0.5] = np.finfo(np.float32).min
    z[5, [5, 99, 600]] = np.inf
    z[6, :] = np.finfo(np.float32).min
    z[7, :] = np.where(rng.random(vocab) < 0.999, -1e9, z[7])
    z[8, :] = -np.inf
    z[8, vocab - 1] = -3.0
    z[9, :] = 3.0e38
    z[10, :] = np.where(rng.random(vocab) < 0.5, -0.0, 0.0)
    z[11, :] *= 1e-30
    u = rng.random(R).astype(np.float32)
    for kw in (dict(), dict(k=40), dict(top_p=0.7), dict(min_p=0.3), dict(k=500, top_p=0.9, min_p=0.01), dict(temp=0.0)):
        check(z, u=u, **kw)


@gpu
def test_sample_extreme_settings():
    rng = np.random.default_rng(3)
    R, V = 16, 3001
    z = (3 * rng.standard_normal((R, V))).astype(np.float32)
    u = rng.random(R).astype(np.float32)
    big = np.float32(3e38)
    for temp in (-1.0, np.nan, 1e-3, 1e-20, 1e-44, 50.0, 1e20, np.inf):
        check(z, temp=temp, u=u)
        check(z, temp=temp, k=17, top_p=0.5, u=u)
    for k in (-5, 0, 1, V - 1, V, V + 1, 2 ** 31 - 1):
        check(z, k=k, u=u)
    for tp in (-1.0, 0.0, 1e-30, 0.999999, 1.0, 2.0, big):
        check(z, top_p=tp, u=u)
    for mp in (-1.0, 0.0, 1e-20, 0.5, 1.0, 1.5, big):
        check(z, min_p=mp, u=u)
    for uu in (-1.0, 0.0, np.nan, 1e-45, 1 - 2.0 ** -24, 1.0, 5.0):
        check(z, u=uu)
        check(z, k=3, u=uu)


@gpu
def test_sample_wide_and_narrow_spreads():
    """Logits spread over the exponents (the histograms' worst case), or within
    a few steps of a float."""
    rng = np.random.default_rng(4)
    V = 20011
    rows = [np.sign(rng.standard_normal(V)) * 2.0 ** rng.uniform(-126, 3, V),
            2.0 ** rng.uniform(-140, -120, V),
            1000 + rng.integers(0, 8, V) * 2.0 ** -13,
            np.where(rng.random(V) < 0.5, 8.0, 8.0 - 2.0 ** rng.uniform(-20, 0, V)),
            -(2.0 ** rng.uniform(-30, 5, V)),
            np.linspace(-20, 20, V)]
    z = np.array(rows, np.float32)
    for seed in range(3):
        r = np.random.default_rng(seed)
        n = len(rows)
        u = r.random(n).astype(np.float32)
        check(z, k=r.integers(1, V, n), u=u)
        check(z, temp=0.7, top_p=r.uniform(0.05, 1, n), u=u)
        check(z, temp=1.3, k=r.integers(100, V, n), top_p=r.uniform(0.05, 1, n), u=u)


@gpu
def test_sample_rows_do_not_depend_on_the_batch_and_repeat():
    """A row's draw is the same alone, in a batch, twice, and without probs."""
    rng = np.random.default_rng(5)
    R, V = 400, 8001
    z = (2 * rng.standard_normal((R, V))).astype(np.float32)
    u = rng.random(R).astype(np.float32)
    a, pa = run(z, top_p=0.9, u=u)
    b, pb = run(z, top_p=0.9, u=u)
    assert np.array_equal(a, b) and np.array_equal(pa, pb)
    c, _ = run(z, top_p=0.9, u=u, probs=False)
    assert np.array_equal(a, c)
    for r in (0, 17, 399):
        d, pd = run(z[r:r + 1], top_p=0.9, u=u[r:r + 1])
        assert d[0] == a[r] and pd[0] == pa[r]


@gpu
def test_sample_frequencies():
    """40000 draws of one small distribution: each token's count within six
    standard deviations of its probability's."""
    z = np.array([[1.0, 0.0, -1.0, 2.0, 0.5]], np.float32)
    n = 40000
    u = (np.arange(n, dtype=np.float64) + 0.5) / n
    ids, _ = run(np.repeat(z, n, 0), u=u.astype(np.float32))
    w = np.exp(z[0].astype(np.float64))
    w /= w.sum()
    got = np.bincount(ids, minlength=5) / n
    assert (np.abs(got - w) <= 6 * np.sqrt(w * (1 - w) / n)).all()


@gpu
@pytest.mark.parametrize("temp", [1e37, 1.2e37, 1e38, 3e38, np.inf])
def test_sample_logits_further_apart_than_the_largest_float(temp):
    """At temperatures near the largest float, finite logits of both ends of
    the type weigh what the formula says; +inf still takes all, -inf nothing."""
    rng = np.random.default_rng(9)
    R, V = 24, 2003
    z = (3.2e38 * rng.uniform(-1, 1, (R, V))).astype(np.float32)
    z[:, 5], z[:, 77] = 3.3e38, -np.finfo(np.float32).max
    z[R - 1, 9] = np.inf
    z[R - 2, 100:] = -np.inf
    u = rng.random(R).astype(np.float32)
    check(z, temp=temp, u=u)
    check(z, temp=temp, k=rng.integers(1, V, R), u=u)
    check(z, temp=temp, top_p=rng.uniform(0.3, 1.0, R), u=u)
    check(z, temp=temp, min_p=rng.uniform(0.0, 0.05, R), u=u)
