"""generate(mode="sample") in Python and Node beside the other modes."""
import json

import numpy as np
import pytest

from mllm import pgw
from test_gpu_draw import bundle, expect
from test_js_host import NODE, run_node

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("arch,kind,tokens", [("llama", "q4", 1), ("llama", "q4", 21), ("llama", "bf16", 21), ("gpt2", "q4", 5)])
def test_sampling_leaves_the_logits_on_the_device(arch, kind, tokens):
    """The prompt's row, too: the host's buffer is not written, and the tokens
    are those of the logits that forwardPrompt and forwardDecode bring."""
    import mllm

    g = mllm.PetitGPT(pgw.parse_pgw(bundle(kind, arch)))
    rng = np.random.default_rng(8)
    prompt = [int(v) for v in rng.integers(0, 512, tokens)]
    u = [float(v) for v in rng.random(6, dtype=np.float32)]
    it = iter(u)
    g._logits[:] = 7.0
    got = g.generate(prompt, maxNewTokens=6, mode="sample", temperature=0.75, topK=40, random=lambda: next(it))
    assert (g._logits == 7.0).all()
    g.resetCache()
    lg, want = g.forwardPrompt(prompt), []
    for v in u:
        want.append(expect(lg, v, dict(temperature=0.75, topK=40))[0])
        if len(want) < 6:
            lg = g.forwardDecode(want[-1])
    assert got["generatedIds"] == want
    g.destroy()


@gpu
@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_node_sampling_leaves_the_logits_on_the_device(tmp_path):
    b = bundle()
    (tmp_path / "m.pgw").write_bytes(b)
    spec = {"prompt": [1, 2, 3, 4], "maxNewTokens": 6, "temperature": 0.0, "numbers": [0.5] * 6}
    (tmp_path / "spec.json").write_text(json.dumps(spec))
    out = run_node("run_sample_modes.mjs", str(tmp_path / "m.pgw"), str(tmp_path / "spec.json"))
    assert out["kept"] and out["drawn"] == out["greedy"]


def repeating(kind):
    """A GPT-2 whose plain argmax repeats itself, so that the 3-gram block acts."""
    return pgw.make_model(pgw.small_config("gpt2"), seed=5, kind=kind)


@gpu
@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), 1e-50])  # the last is 0 in float32
@pytest.mark.parametrize("kind", ["q4", "f32"])
def test_gpt2_at_temperature_0_is_greedy(kind, temperature):
    import mllm

    g = mllm.PetitGPT(pgw.parse_pgw(repeating(kind)))
    prompt = [3, 14, 15, 92, 65]
    greedy = g.generate(prompt, maxNewTokens=24)
    got = g.generate(prompt, maxNewTokens=24, mode="sample", temperature=temperature, random=lambda: 0.5)
    assert got["generatedIds"] == greedy["generatedIds"] and got["mode"].endswith("sample")
    eos = greedy["generatedIds"][5]
    stopped = g.generate(prompt, maxNewTokens=24, mode="sample", temperature=temperature, eosId=eos)
    assert stopped["stopReason"] == "eos" and stopped["generatedIds"] == greedy["generatedIds"][:stopped_at(greedy, eos)]
    # the rule has something to do: the maxima alone are other tokens
    lg, plain = g.forwardPrompt(prompt), []
    for _ in range(24):
        plain.append(int(np.argmax(lg)))
        lg = g.forwardDecode(plain[-1])
    assert plain != greedy["generatedIds"]
    g.destroy()


def stopped_at(res, eos):
    return res["generatedIds"].index(eos) + 1


@gpu
@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_node_gpt2_at_temperature_0_is_greedy(tmp_path):
    import mllm

    b = repeating("q4")
    (tmp_path / "m.pgw").write_bytes(b)
    spec = {"prompt": [3, 14, 15, 92, 65], "maxNewTokens": 24, "temperature": 0.0, "numbers": [0.5] * 24}
    (tmp_path / "spec.json").write_text(json.dumps(spec))
    out = run_node("run_sample_modes.mjs", str(tmp_path / "m.pgw"), str(tmp_path / "spec.json"))
    g = mllm.PetitGPT(pgw.parse_pgw(b))
    assert out["drawn"] == out["greedy"] == g.generate(spec["prompt"], maxNewTokens=24)["generatedIds"]
    g.destroy()
