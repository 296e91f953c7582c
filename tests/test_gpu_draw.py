"""mllm_draw: tokens drawn from a model's logits on the device, through the C ABI,
PetitGPT.generate(mode="sample") and the Node class, against mllm_sample's
definition on the same logits (test_gpu_sample.ref_row)."""
import ctypes as C
import json

import numpy as np
import pytest

from mllm import abi, pgw
from test_gpu_sample import ref_row
from test_js_host import NODE, run_node

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def bundle(kind="q4", arch="llama"):
    return pgw.make_model(pgw.small_config(arch), seed=11, kind=kind, std=0.3)


SETTINGS = [dict(), dict(temperature=0.7, topK=20), dict(temperature=1.3, topP=0.8), dict(minP=0.1),
            dict(temperature=0.9, topK=50, topP=0.9, minP=0.02), dict(temperature=0.0)]


def expect(logits, u, s):
    return ref_row(logits.copy(), float(np.float32(s.get("temperature", 1.0))), s.get("topK", 0),
                   float(np.float32(s.get("topP", 1.0))), float(np.float32(s.get("minP", 0.0))), float(np.float32(u)))


@gpu
@pytest.mark.parametrize("arch,kind,exec_mode", [("llama", "q4", None), ("llama", "q4", 1), ("llama", "q8", None),
                                                ("llama", "bf16", None), ("gpt2", "q4", None), ("gpt2", "f32", None)])
def test_draw_follows_every_kind_of_call(arch, kind, exec_mode):
    import mllm

    g = mllm.PetitGPT(pgw.parse_pgw(bundle(kind, arch)), exec_mode=exec_mode)
    rng = np.random.default_rng(4)
    with pytest.raises(abi.MllmError):
        g.draw(0.5)  # nothing has run

    def same(logits):
        for s in SETTINGS:
            u = float(rng.random(dtype=np.float32))
            want, prob = expect(logits, u, s)
            tok, p = g.draw(u, **s)
            assert tok == want and abs(p - prob) <= 2e-7, (s, u)

    same(g.forwardPrompt([5]).copy())
    g.resetCache()
    same(g.forwardPrompt([int(v) for v in rng.integers(0, 512, 21)]).copy())
    g.set_prefill(0)
    g.resetCache()
    same(g.forwardPrompt([int(v) for v in rng.integers(0, 512, 19)]).copy())
    same(g.forwardDecode(7).copy())
    rows, logits = g.forwardVerify([3, 9, 27], want_logits=True)
    same(logits[-1].copy())
    g.cacheLen = 10
    want = g.forwardDecode(3).copy()
    g.cacheLen = 10
    g.decodeStep(3)
    same(want)
    g.decodeChain(3, 2)
    with pytest.raises(abi.MllmError):
        g.draw(0.5)
    with pytest.raises(abi.MllmError):
        g.forwardDecode(-1)  # refused: the chain's state stays
    same(g.forwardDecode(3).copy())
    g.destroy()


@gpu
def test_generate_sample_and_null_prob():
    import mllm

    g = mllm.PetitGPT(pgw.parse_pgw(bundle()))
    prompt = [3, 14, 15, 92, 65]
    u = [float(v) for v in np.random.default_rng(6).random(16, dtype=np.float32)]
    it = iter(u)
    got = g.generate(prompt, maxNewTokens=16, mode="sample", temperature=0.8, topK=40, topP=0.9, random=lambda: next(it))
    g.resetCache()
    lg, want = g.forwardPrompt(prompt), []
    for v in u:
        want.append(expect(lg, v, dict(temperature=0.8, topK=40, topP=0.9))[0])
        if len(want) < 16:
            lg = g.forwardDecode(want[-1])
    assert got["generatedIds"] == want and got["mode"].endswith("sample")
    greedy = g.generate(prompt, maxNewTokens=8, mode="sample", temperature=0.0)
    assert greedy["generatedIds"] == g.generate(prompt, maxNewTokens=8)["generatedIds"]
    eos = greedy["generatedIds"][2]
    stopped = g.generate(prompt, maxNewTokens=8, mode="sample", temperature=0.0, eosId=eos)
    assert stopped["stopReason"] == "eos" and stopped["generatedIds"][-1] == eos
    tok = C.c_int32(0)
    assert abi.lib().mllm_draw(g._h, 1.0, 0, 1.0, 0.0, 0.5, C.byref(tok), None) == 0
    assert abi.lib().mllm_draw(g._h, 1.0, 0, 1.0, 0.0, 0.5, None, None) == 1
    g.destroy()


def test_draw_refuses_null():
    tok = C.c_int32(0)
    assert abi.lib().mllm_draw(None, 1.0, 0, 1.0, 0.0, 0.5, C.byref(tok), None) == 1


@gpu
@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_node_sample(tmp_path):
    import mllm

    b = bundle()
    (tmp_path / "m.pgw").write_bytes(b)
    u = [float(v) for v in np.random.default_rng(7).random(12, dtype=np.float32)]
    spec = {"prompt": [1, 2, 3, 4], "maxNewTokens": 12, "temperature": 0.75, "topK": 30, "topP": 0.875, "minP": 0.015625,
            "numbers": u}
    (tmp_path / "spec.json").write_text(json.dumps(spec))
    out = run_node("run_sample.mjs", str(tmp_path / "m.pgw"), str(tmp_path / "spec.json"))
    g = mllm.PetitGPT(pgw.parse_pgw(b))
    it = iter(u)
    want = g.generate([1, 2, 3, 4], maxNewTokens=12, mode="sample", temperature=0.75, topK=30, topP=0.875, minP=0.015625,
                      random=lambda: next(it))
    g.destroy()
    assert out["generatedIds"] == want["generatedIds"] and out["used"] == 12
    assert out["drawn"]["id"] == want["generatedIds"][0] and 0 < out["drawn"]["prob"] <= 1
    assert "no logits" in out["refused"]
