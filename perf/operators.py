"""One decode step of several sequences, put together from operators on device
pointers (include/mllm.h), as cases that can be timed and checked:

    rope    mllm_rope_kv_paged: the rows of attn.qkv, normed and rotated, into
            q and the pages of the key-value cache
    attn    mllm_attn_paged: the attention of one new token per row over pages
    sample  mllm_sample: temperature, top-k, top-p, min-p and a given number

    listed()          the named cases
    draw(rng)         another case of the same ranges
    prepare(case, s)  inputs from the seed s
    run(state)        one pass: elementary torch operations, or with `own` the
                      framework's operators
    work(case)        the bytes and operations a pass cannot do without
    exact(case, s)    what run() returns, in 64 bits
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}  # include/mllm.h MLLM_F32, MLLM_F16, MLLM_BF16


# ---------------------------------------------------------------- the cases
def _rope(seqs, new, ctx, heads, kv_heads, hd, kv, page, rot=0, inter=False, norm=False, layout="hnd", theta=1e5,
          scale=1.0):
    """seqs sequences with `new` tokens each, the last at about position ctx;
    rot 0: the whole head; scale: positions compressed by it."""
    return dict(op="rope", seqs=seqs, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, hd=hd, kv=kv, page=page,
                rot=rot or hd, inter=inter, norm=norm, layout=layout, theta=theta, scale=scale)


def _attn(seqs, new, ctx, heads, kv_heads, hd, kv, page, ragged=True, layout="hnd"):
    """seqs sequences, `new` rows each (1: decode; k + 1: a speculation pass,
    each row one position longer), contexts up to ctx."""
    return dict(op="attn", seqs=seqs, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, hd=hd, kv=kv, page=page,
                ragged=ragged, layout=layout)


def _sample(rows, vocab, filters, ties=False, masked=0.0):
    return dict(op="sample", rows=rows, vocab=vocab, filters=filters, ties=ties, masked=masked)


def listed():
    return [
        # chat with one user: one token of the 135M shape, f32 cache
        dict(_rope(1, 1, 700, 9, 3, 64, "f32", 16), name="rope_decode_1"),
        # 64 users decode a token each: 360M shape, f16 cache
        dict(_rope(64, 1, 500, 15, 5, 64, "f16", 16), name="rope_decode_64"),
        # a prompt of odd length, 360M shape, pages of 64 slots by token
        dict(_rope(1, 1501, 1536, 15, 5, 64, "f16", 64, layout="nhd"), name="rope_prompt_1501"),
        # prompts of a larger model with normed queries and keys, neighbouring
        # pairs, half of the head rotated, positions compressed for long contexts
        dict(_rope(8, 1000, 4000, 32, 8, 128, "bf16", 32, rot=64, inter=True, norm=True, theta=1e6, scale=4.0),
             name="rope_norm_8000"),
        # one user in a chat: the 135M shape at 700 positions, f32 cache
        dict(_attn(1, 1, 700, 9, 3, 64, "f32", 16), name="attn_decode_1x700"),
        # a token and four drafts verified at 512 positions (prompt lookup)
        dict(_attn(1, 5, 516, 9, 3, 64, "f16", 16), name="attn_verify_5x512"),
        # 64 users at up to 2048 positions: 360M shape, f16 cache
        dict(_attn(64, 1, 2048, 15, 5, 64, "f16", 16), name="attn_decode_64x2048"),
        # two documents of 100000 positions, grouped heads of a larger model
        dict(_attn(2, 1, 100000, 32, 8, 128, "bf16", 64, ragged=False, layout="nhd"), name="attn_long_2x100000"),
        # one user: the usual chat settings (temperature, top-k, top-p)
        dict(_sample(1, 49152, "kp"), name="sample_1"),
        # a batch with every user's own settings, GPT-2's odd vocabulary,
        # logits that tie (they come from 8-bit mantissas)
        dict(_sample(64, 50257, "mix", ties=True), name="sample_mix_64x50257"),
        # top-p alone, a grammar masks a third of the tokens
        dict(_sample(200, 49152, "p", masked=0.3), name="sample_p_200x49152"),
        # the plain distribution of a large vocabulary, min-p
        dict(_sample(100, 131072, "minp"), name="sample_minp_100x131072"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "sample", "sample"])
    if op == "sample":
        rows = _log(rng, 1, 250)
        vocab = _log(rng, 1000, min(131072, 12000000 // rows))
        return _sample(rows, vocab, rng.choice(["k", "p", "kp", "minp", "none", "mix"]), ties=rng.random() < 0.3,
                       masked=rng.choice([0.0, 0.0, 0.5]))
    hd = rng.choice([64, 64, 64, 128, 128, 32, 96, 256])
    kv_heads = rng.randint(1, 8)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    kv = rng.choice(["f32", "f16", "f16", "bf16"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    layout = rng.choice(["hnd", "hnd", "nhd"])
    es = 4 if kv == "f32" else 2
    if op == "rope":
        seqs = _log(rng, 1, 64)
        most = max(2, 60000000 // ((heads + 2 * kv_heads) * hd * 4 * seqs))
        new = 1 if rng.random() < 0.4 else _log(rng, 1, min(2000, most))
        ctx = new + _log(rng, 1, max(2, 60000000 // (2 * seqs * kv_heads * hd * es)))
        return _rope(seqs, new, ctx, heads, kv_heads, hd, kv, page, rot=rng.choice([hd, hd, hd // 2, hd // 4]),
                     inter=rng.random() < 0.4, norm=rng.random() < 0.4, layout=layout,
                     theta=rng.choice([1e4, 1e5, 1e6]), scale=rng.choice([1.0, 1.0, 8.0]))
    seqs = _log(rng, 1, 100)
    new = rng.choice([1, 1, 1, 2, 5])
    ctx = new + _log(rng, 1, max(2, min(60000, 250000000 // (2 * seqs * new * kv_heads * hd * es))))
    return _attn(seqs, new, ctx, heads, kv_heads, hd, kv, page, ragged=rng.random() < 0.7, layout=layout)


# ---------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _lengths(c):
    """Each sequence's context, a part of the case: ragged from a quarter of
    ctx on, the first one whole."""
    r = random.Random(c["ctx"] * 131 + c["seqs"])
    lo = max(c["new"], c["ctx"] // 4)
    return [c["ctx"] if i == 0 or not c.get("ragged", True) else r.randint(lo, c["ctx"]) for i in range(c["seqs"])]


def _pages(c, g, lens):
    """A pool with room for every sequence and some free pages, its tables in
    the order in which a long-running server hands pages out: none."""
    cols = (max(lens) + c["page"] - 1) // c["page"]
    need = [(n + c["page"] - 1) // c["page"] for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEV)
    table = torch.zeros(c["seqs"], cols, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    shape = (total, c["kv_heads"], c["page"], c["hd"]) if c["layout"] == "hnd" else (total, c["page"], c["kv_heads"], c["hd"])
    k, v = (_normal(g, *shape).to(TYPES[c["kv"]]) for _ in range(2))
    return k, v, table


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    s = {"case": c}
    if c["op"] == "sample":
        R, V = c["rows"], c["vocab"]
        x = 2.5 * _normal(g, R, V)  # a long tail and some tokens that stand out
        some = torch.randint(0, V, (R, 64), generator=g, device=DEV)
        x.scatter_add_(1, some, 10.0 * torch.rand(R, 64, generator=g, device=DEV))
        if c["ties"]:
            x = x.to(torch.bfloat16).float()
        if c["masked"]:
            x = x.masked_fill(torch.rand(R, V, generator=g, device=DEV) < c["masked"], -math.inf)
        rand = lambda lo, hi: lo + (hi - lo) * torch.rand(R, generator=g, device=DEV)  # noqa: E731
        f = c["filters"]
        temp, k = rand(0.4, 1.3), torch.randint(10, 200, (R,), generator=g, device=DEV, dtype=torch.int32)
        p, m, u = rand(0.7, 0.99), rand(0.01, 0.2), rand(0.0, 1.0).clamp(max=1 - 2.0 ** -24)
        if f == "mix":  # each of them on for some rows, and some rows greedy
            on = torch.rand(4, R, generator=g, device=DEV)
            temp, k = torch.where(on[0] < 0.1, 0.0, temp), torch.where(on[1] < 0.5, 0, k).to(torch.int32)
            p, m = torch.where(on[2] < 0.5, 1.0, p), torch.where(on[3] < 0.5, 0.0, m)
        s.update(logits=x, temp=temp, k=k if f in ("k", "kp", "mix") else None, p=p if f in ("p", "kp", "mix") else None,
                 m=m if f in ("minp", "mix") else None, u=u)
        return s
    lens = _lengths(c)
    k, v, table = _pages(c, g, lens)
    s.update(k=k, v=v, table=table, kp=_heads_first(c, k), vp=_heads_first(c, v))
    ids = torch.arange(c["seqs"], device=DEV, dtype=torch.int32).repeat_interleave(c["new"])
    step = torch.arange(c["new"], device=DEV, dtype=torch.int32).repeat(c["seqs"])
    ends = torch.tensor(lens, device=DEV, dtype=torch.int32).repeat_interleave(c["new"])
    pos = ends - c["new"] + step  # the last tokens of each sequence
    T = c["seqs"] * c["new"]
    s["seq"] = ids
    if c["op"] == "rope":
        s["pos"] = pos
        s["qkv"] = _normal(g, T, (c["heads"] + 2 * c["kv_heads"]) * c["hd"])
        i = torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64)
        s["freq"] = (c["theta"] ** (-2.0 * i / c["rot"]) / c["scale"]).float()
        gains = 1.0 + 0.1 * _normal(g, 2, c["hd"])
        s["gq"], s["gk"] = (gains[0].contiguous(), gains[1].contiguous()) if c["norm"] else (None, None)
        return s
    s["len"] = pos + 1
    s["q"] = _normal(g, T, c["heads"] * c["hd"])
    return s


def _heads_first(c, pool):
    """The pool as [pages][kv heads][slots][hd], whatever its layout."""
    return pool if c["layout"] == "hnd" else pool.permute(0, 2, 1, 3)


# ---------------------------------------------------------------- the plain forms
def _plain_rope(s):
    c = s["case"]
    H, KV, D, R, T = c["heads"], c["kv_heads"], c["hd"], c["rot"], s["qkv"].shape[0]
    x = s["qkv"].view(T, H + 2 * KV, D)
    qk, v = x[:, :H + KV], x[:, H + KV:]
    if c["norm"]:
        gain = torch.cat([s["gq"].expand(H, D), s["gk"].expand(KV, D)])
        qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS) * gain
    a = s["pos"].double()[:, None] * s["freq"].double()
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    if c["inter"]:
        x1, x2 = qk[..., 0:R:2], qk[..., 1:R:2]
        turned = torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).flatten(-2)
    else:
        x1, x2 = qk[..., :R // 2], qk[..., R // 2:R]
        turned = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    qk = torch.cat([turned, qk[..., R:]], -1)
    pos = s["pos"].long()
    page, slot = s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]
    s["kp"][page, :, slot] = qk[:, H:].to(s["k"].dtype)
    s["vp"][page, :, slot] = v.to(s["v"].dtype)
    return {"q": qk[:, :H].reshape(T, H * D), "k": s["k"], "v": s["v"]}


def _plain_attn(s):
    c = s["case"]
    H, KV, D, T = c["heads"], c["kv_heads"], c["hd"], s["q"].shape[0]
    tab = s["table"][s["seq"].long()].long()
    k, v = (p[tab].float().permute(0, 2, 1, 3, 4).reshape(T, KV, -1, D) for p in (s["kp"], s["vp"]))
    q = s["q"].view(T, KV, H // KV, D)
    sc = torch.matmul(k, q.transpose(2, 3).contiguous()).transpose(2, 3) * (1.0 / math.sqrt(D))  # [T, KV, rep, positions]
    sees = torch.arange(sc.shape[-1], device=DEV) < s["len"][:, None, None, None]
    sc = torch.where(sees, sc, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(T, H * D)


def _plain_sample(s):
    z = s["logits"].double()
    R, V = z.shape
    greedy = s["temp"] <= 0
    t = torch.where(greedy, 1.0, s["temp"]).double()[:, None]
    w = torch.exp((z - z.amax(-1, keepdim=True)) / t)
    order = torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(V, device=DEV)
    keep = torch.ones_like(ws, dtype=torch.bool)
    if s["k"] is not None:
        keep = (rank < s["k"][:, None]) | (s["k"][:, None] <= 0)
    if s["p"] is not None:
        wk = ws * keep
        before = wk.cumsum(-1) - wk
        p = s["p"].double()[:, None]
        keep = keep & ((before < p * wk.sum(-1, keepdim=True)) | (p >= 1))
    if s["m"] is not None:
        keep = keep & (ws >= s["m"].double()[:, None])
    keep = torch.where(greedy[:, None], rank == 0, keep | (rank == 0))
    w = torch.zeros_like(w).scatter_(1, order, ws * keep)
    cum = w.cumsum(-1)
    total = cum[:, -1:]
    ids = (cum <= s["u"].double()[:, None] * total).sum(-1).clamp(max=V - 1)
    return {"ids": ids.to(torch.int32), "probs": (w.gather(1, ids[:, None]) / total)[:, 0].float()}


# ---------------------------------------------------------------- the framework's operators
def _p(t):
    return None if t is None else t.data_ptr()


def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    at = os.path.join(root, "microllm-lab_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from mllm import abi

    return abi


def _handle(abi, s):
    """What a server makes once for its pool: the description of the pages, and
    the outputs' and the workspace's memory."""
    c = s["case"]
    T = s["seq"].numel()
    H, S, D = c["kv_heads"], c["page"], c["hd"]
    strides = (H * S * D, S * D, D) if c["layout"] == "hnd" else (H * S * D, D, H * D)
    s["kv"] = abi.MllmKvPages(_p(s["k"]), _p(s["v"]), CODES[c["kv"]], H, D, s["k"].shape[0], S, *strides,
                              _p(s["table"]), *s["table"].shape)
    s["out"] = torch.empty(T, c["heads"] * D, dtype=torch.float32, device=DEV)
    if c["op"] == "attn":
        n = abi.lib().mllm_attn_paged_workspace(s["kv"], T, c["heads"], c["ctx"])
        s["ws"] = torch.zeros(max(1, n), dtype=torch.uint8, device=DEV)


def _own(s):
    c = s["case"]
    abi = _library()
    st = torch.cuda.current_stream().cuda_stream
    if c["op"] == "sample":
        R, V = s["logits"].shape
        ids, probs = torch.empty(R, dtype=torch.int32, device=DEV), torch.empty(R, dtype=torch.float32, device=DEV)
        abi.call("mllm_sample", R, V, _p(s["logits"]), _p(s["temp"]), _p(s["k"]), _p(s["p"]), _p(s["m"]), _p(s["u"]),
                 _p(ids), _p(probs), st)
        return {"ids": ids, "probs": probs}
    if "kv" not in s:
        _handle(abi, s)
    T, D = s["seq"].numel(), c["hd"]
    if c["op"] == "rope":
        abi.call("mllm_rope_kv_paged", s["kv"], T, c["heads"], _p(s["qkv"]), _p(s["seq"]), _p(s["pos"]), _p(s["freq"]),
                 c["rot"], int(c["inter"]), _p(s["gq"]), _p(s["gk"]), EPS, _p(s["out"]), st)
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    abi.call("mllm_attn_paged", s["kv"], T, c["heads"], _p(s["q"]), _p(s["seq"]), _p(s["len"]), c["ctx"],
             1.0 / math.sqrt(D), _p(s["out"]), _p(s["ws"]), s["ws"].numel(), st)
    return s["out"]


def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "attn": _plain_attn, "sample": _plain_sample}[s["case"]["op"]](s)


# ---------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + 28 * c["rows"], "flops": 4 * n}  # difference, quotient, exp, sum
    es = 4 if c["kv"] == "f32" else 2
    T, H, KV, D = c["seqs"] * c["new"], c["heads"], c["kv_heads"], c["hd"]
    if c["op"] == "rope":
        turned = T * (H + KV)
        return {"bytes": 4 * T * (2 * H + 2 * KV) * D + 2 * es * T * KV * D + 12 * T,
                "flops": turned * (3 * c["rot"] + (4 * D if c["norm"] else 0))}
    lens = _lengths(c)  # a sequence's rows read the same keys
    keys = sum(n - c["new"] + 1 + i for n in lens for i in range(c["new"]))
    return {"bytes": 2 * es * sum(lens) * KV * D + 8 * T * H * D + 4 * sum(-(-n // c["page"]) for n in lens),
            "flops": 4 * keys * H * D}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](s)


def _exact_rope(s):
    """The rotation as a product of complex numbers, a pair to each."""
    c = s["case"]
    H, KV, D, R, T = c["heads"], c["kv_heads"], c["hd"], c["rot"], s["qkv"].shape[0]
    x = s["qkv"].double().reshape(T, H + 2 * KV, D)
    if c["norm"]:
        for lo, hi, gain in ((0, H, s["gq"]), (H, H + KV, s["gk"])):
            h = x[:, lo:hi]
            x[:, lo:hi] = h * gain.double() * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    i = torch.arange(R // 2, device=DEV)
    a, b = (2 * i, 2 * i + 1) if c["inter"] else (i, i + R // 2)
    angle = s["pos"].double()[:, None, None] * s["freq"].double()
    z = torch.complex(x[:, :H + KV, a], x[:, :H + KV, b]) * torch.polar(torch.ones_like(angle), angle)
    x[:, :H + KV, a], x[:, :H + KV, b] = z.real, z.imag
    at = s["pos"].long()
    row = s["table"].long().gather(1, (at // c["page"]).reshape(c["seqs"], c["new"])).reshape(-1)
    out = {"q": x[:, :H].reshape(T, H * D)}
    for name, lo in (("k", H), ("v", H + KV)):
        pool = s[name].double()
        if c["layout"] == "hnd":
            for h in range(KV):
                pool[row, h, at % c["page"]] = x[:, lo + h]
        else:
            pool[row, at % c["page"]] = x[:, lo:lo + KV]
        out[name] = pool
    return out


def _exact_attn(s):
    """Row by row: the sequence's positions one after another, then its heads."""
    c = s["case"]
    H, KV, D = c["heads"], c["kv_heads"], c["hd"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, (q, n) in enumerate(zip(s["seq"].tolist(), s["len"].tolist())):
        pages = s["table"][q, :-(-n // c["page"])].long()
        rows = []
        for pool in (s["k"], s["v"]):
            p = pool[pages].double()
            p = p.transpose(1, 2) if c["layout"] == "hnd" else p
            rows.append(p.reshape(-1, KV, D)[:n])
        k, v = rows
        x = s["q"][r].double().reshape(KV, H // KV, D)
        o = []
        for h in range(KV):
            p = torch.softmax(x[h] @ k[:, h].T.contiguous() / math.sqrt(D), -1)
            o.append(p @ v[:, h].contiguous())
        out[r] = torch.cat(o).reshape(-1)
    return out


def _exact_sample(s):
    """Row by row on the host: the tokens in order of their logits, the
    prefix that each filter leaves, the first token whose sum passes u."""
    x = s["logits"].cpu().numpy().astype(np.float64)
    get = lambda n, off: s[n].double().cpu().numpy() if s[n] is not None else np.full(len(x), off)  # noqa: E731
    temp, ks, ps, ms, us = get("temp", 1.0), get("k", 0), get("p", 1.0), get("m", 0.0), get("u", 0.0)
    ids, probs = np.zeros(len(x), np.int32), np.zeros(len(x))
    for r, z in enumerate(x):
        if temp[r] <= 0:
            ids[r], probs[r] = int(np.argmax(z)), 1.0
            continue
        order = np.argsort(-z, kind="stable")
        w = np.exp((z[order] - z[order[0]]) / temp[r])
        n = min(int(ks[r]), len(z)) if ks[r] > 0 else len(z)
        if ps[r] < 1:
            before = np.concatenate([[0.0], np.cumsum(w[:n])])
            n = max(1, int(np.searchsorted(before[:n], ps[r] * before[n], side="left")))
        n = max(1, int(np.count_nonzero(w[:n] >= ms[r])))
        kept = np.sort(order[:n])
        w = np.exp((z[kept] - z[order[0]]) / temp[r])
        cum = np.cumsum(w)
        j = min(int(np.searchsorted(cum, us[r] * cum[-1], side="right")), n - 1)
        ids[r], probs[r] = kept[j], w[j] / cum[-1]
    return {"ids": ids, "probs": probs}
