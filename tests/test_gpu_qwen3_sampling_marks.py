"""Sampling in the Qwen3 engine on gfx950 where some logits, not all, are not
finite: every mode refuses the step, as it does without sampling, whatever
xpu_sample would have drawn."""
import numpy as np
import pytest

import oracle_lib as orc
import xpu_playground_amd as xpu
from cache_util import codes, values
from checkpoint_util import write_checkpoint
from xpu_playground_amd import qwen3

pytestmark = pytest.mark.gpu
PROMPT = [3, 4, 9]


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("name", ["tiny", "small"])
def test_one_infinite_logit_raises(rt, tmp_path, name, sign):
    """One token's row of the embedding has a single value, so large that its
    product with the last hidden state passes FP32's range: its logit is one
    infinity, of this sign, and no other is touched."""
    import torch
    from safetensors.torch import load_file, save_file

    cfg = orc.config(name)
    write_checkpoint(str(tmp_path), cfg, seed=1, gain_std=0.0)
    with qwen3.Engine(runtime=rt, model_dir=str(tmp_path), max_seq=16) as eng:
        for p, token in enumerate(PROMPT):
            eng.decode(token, p)
        hidden = values(eng.hidden(), xpu.BF16)
        norm = orc.rmsnorm(codes(hidden, xpu.BF16), orc.fill_tensor(cfg, 1, 0.0, orc.W_FINALNORM, 0))
        norm = values(norm, xpu.BF16)
    j = int(np.abs(norm).argmax())
    assert abs(norm[j]) > 1.2
    path = str(tmp_path / "model.safetensors")
    tensors = load_file(path)
    head = "model.embed_tokens.weight" if cfg.tied else "lm_head.weight"
    row = 100
    tensors[head][row] = 0
    tensors[head][row, j] = 3.3e38 * sign * np.sign(norm[j])
    save_file(tensors, path)
    with qwen3.Engine(runtime=rt, model_dir=str(tmp_path), max_seq=16) as eng:
        for mode in (qwen3.GRAPH, qwen3.EAGER, qwen3.REFERENCE):
            eng.set_mode(mode)
            for prefill in ("batched", "stepwise") if name == "small" and mode != qwen3.REFERENCE else (None,):
                if prefill:
                    eng.set_prefill(prefill)
                for temperature in (0.0, 0.8):
                    eng.set_sampling(temperature, top_k=50, seed=4)
                    print(f"{name} sign {sign} mode {mode} prefill {prefill} temperature {temperature}", flush=True)
                    with pytest.raises(xpu.XpuError, match="NaN"):
                        eng.generate(PROMPT, 1)
                    with pytest.raises(xpu.XpuError, match="NaN"):
                        eng.generate(PROMPT, 4, stop_on_eos=False)
        logits = values(eng.logits(), xpu.BF16)
        assert np.isinf(logits).sum() >= 1 and not np.isnan(logits).any()
