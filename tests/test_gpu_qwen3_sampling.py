"""Sampling in the Qwen3 engine on gfx950: every token is the one that the
definition draws, in 64 bits, from the oracle's logits (which the engine's equal
bit for bit) with the random number of its position."""
import json
import os
import subprocess

import numpy as np
import pytest

import oracle_lib as orc
import xpu_playground_amd as xpu
from checkpoint_util import write_checkpoint
from cache_util import values
from test_gpu_sample import expected
from xpu_playground_amd import qwen3

pytestmark = pytest.mark.gpu
MODES = [qwen3.GRAPH, qwen3.EAGER, qwen3.REFERENCE]
FILTERS = [dict(temperature=0.7), dict(temperature=1.5, top_k=40, top_p=0.9, min_p=0.02)]
M = (1 << 64) - 1


def mix64(z):
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9 & M
    z = (z ^ (z >> 27)) * 0x94D049BB133111EB & M
    return z ^ (z >> 31)


def number(seed, position):
    return (mix64((mix64(seed) + (position + 1) * 0x9E3779B97F4A7C15) & M) >> 40) * 2.0 ** -24


def drawn(cfg, prompt, new, max_seq, seed, temperature, top_k=0, top_p=1.0, min_p=0.0):
    m, out = orc.Model(cfg, seed=5, gain_std=0.1, max_seq=max_seq), []
    for p in range(len(prompt) + new - 1):
        token = int(prompt[p]) if p < len(prompt) else out[-1]
        _, logits = m.decode(token, p, want_logits=True)
        if p >= len(prompt) - 1:
            out.append(expected(values(logits, xpu.BF16), temperature, top_k, top_p, min_p, number(seed, p))[0])
    return out


@pytest.mark.parametrize("name,vocab", [("tiny", None), ("tiny", 20011), ("small", None)])
@pytest.mark.parametrize("how", FILTERS)
def test_generate(rt, name, vocab, how):
    cfg = orc.config(name, **({"vocab": vocab} if vocab else {}))
    prompt = orc.tokens(12, 9, cfg.vocab)
    want = drawn(cfg, prompt, 16, 64, 77, **how)
    eng = qwen3.Engine(qwen3.config_from(cfg), max_seq=64, seed=5, gain_std=0.1, runtime=rt)
    greedy = eng.generate(prompt, 16, stop_on_eos=False)[0].tolist()
    eng.set_sampling(seed=77, **how)
    for mode in MODES:
        for prefill in ("batched", "stepwise") if name == "small" and mode != qwen3.REFERENCE else (None,):
            print(f"{name} vocab {cfg.vocab} mode {mode} prefill {prefill}", flush=True)
            eng.set_mode(mode)
            if prefill:
                eng.set_prefill(prefill)
            assert eng.generate(prompt, 16, stop_on_eos=False)[0].tolist() == want
            # a token at a time, each call with all before it as its prompt
            if prefill != "batched":
                one = list(want[:3])
                one += eng.generate(list(prompt) + one, 1, stop_on_eos=False)[0].tolist()
                assert one == want[:4]
            assert eng.generate(prompt[:1], 0, stop_on_eos=False)[0].tolist() == []
    eng.set_sampling(seed=78, **how)
    assert eng.generate(prompt, 16, stop_on_eos=False)[0].tolist() != want
    eng.set_sampling(0)
    for mode in MODES:
        eng.set_mode(mode)
        assert eng.generate(prompt, 16, stop_on_eos=False)[0].tolist() == greedy
    eng.close()


def test_up_to_the_last_position(rt):
    cfg = orc.config("tiny")
    prompt = orc.tokens(3, 9, cfg.vocab)
    eng = qwen3.Engine(qwen3.config_from(cfg), max_seq=24, seed=5, gain_std=0.1, runtime=rt)
    eng.set_sampling(1.0, seed=3)
    want = drawn(cfg, prompt, 21, 24, 3, 1.0)
    for mode in MODES:
        eng.set_mode(mode)
        assert eng.generate(prompt, 21, stop_on_eos=False)[0].tolist() == want
    eng.close()


def test_non_finite_logits_raise(rt, tmp_path):
    cfg = orc.config("tiny")
    write_checkpoint(str(tmp_path), cfg, seed=1, gain_std=0.0, nan_embed=True)
    eng = qwen3.Engine(runtime=rt, model_dir=str(tmp_path), max_seq=16)
    eng.set_sampling(0.8)
    for mode in MODES:
        eng.set_mode(mode)
        with pytest.raises(xpu.XpuError, match="NaN"):
            eng.generate([3, 4], 4)
    eng.close()


def test_command_line(tmp_path):
    cfg = orc.config("tiny")
    prompt = orc.tokens(12, 5, cfg.vocab)
    ids = tmp_path / "ids.txt"
    ids.write_text(" ".join(map(str, prompt.tolist())) + "\n")
    with qwen3.Engine(qwen3.config_from(cfg), max_seq=64) as eng:
        eng.set_sampling(0.9, top_k=20, top_p=0.95, min_p=0.01, seed=6)
        want = eng.generate(prompt, 10, stop_on_eos=False)[0].tolist()
    exe = os.path.join(xpu.BUILD_DIR, "qwen3_hip")
    out = subprocess.run([exe, "--synthetic", "tiny", "--input-ids", str(ids), "--max-new-tokens", "10", "--max-seq-len", "64",
                          "--no-eos-stop", "--temperature", "0.9", "--top-k", "20", "--top-p", "0.95", "--min-p", "0.01",
                          "--sample-seed", "6"], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr
    assert json.loads(out.stdout)["generated_ids"] == want
    assert len(want) == 10 and np.unique(want).size > 1
