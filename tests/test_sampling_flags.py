"""Refusals of the sampling options: of the engine's call, before it looks at the
engine, and of the command line, before it looks for a device."""
import os
import subprocess

import pytest

import xpu_playground_amd as xpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("args,word", [
    ((-0.5, 0, 1, 0), "temperature"), ((INF, 0, 1, 0), "temperature"), ((NAN, 0, 1, 0), "temperature"),
    ((1, 0, -1, 0), "top_p"), ((1, 0, NAN, 0), "top_p"), ((0, 0, NAN, 0), "top_p"), ((1, 0, 1, -0.1), "min_p"),
    ((1, 0, 1, 1.5), "min_p"), ((1, 0, 1, NAN), "min_p"), ((1, 5, 0.9, 0.1), "null engine"), ((0, 0, 1, 0), "null engine"),
])
def test_set_sampling_refuses(args, word):
    with pytest.raises(xpu.XpuError, match=word):
        xpu.check(xpu.library().xpu_qwen3_set_sampling(None, *args, 7))


@pytest.mark.parametrize("options,word", [
    (["--temperature", "-1"], "invalid value for --temperature"), (["--temperature", "inf"], "invalid value for --temperature"),
    (["--temperature", "nan"], "invalid value for --temperature"), (["--temperature", "1x"], "invalid value for --temperature"),
    (["--temperature"], "missing value"), (["--temperature", "1", "--top-k", "-3"], "invalid value for --top-k"),
    (["--temperature", "1", "--top-p", "-0.1"], "invalid value for --top-p"),
    (["--temperature", "1", "--min-p", "1.01"], "invalid value for --min-p"),
    (["--temperature", "1", "--sample-seed", "x"], "invalid value for --sample-seed"),
    (["--top-k", "5"], "--top-k needs --temperature"), (["--temperature", "0", "--top-p", "0.5"], "--top-p needs --temperature"),
    (["--sample-seed", "1"], "--sample-seed needs --temperature"),
])
def test_command_line_refuses(options, word):
    exe = os.path.join(xpu.BUILD_DIR, "qwen3_hip")
    out = subprocess.run([exe, "--synthetic", "tiny", "--input-ids", "-", "--max-new-tokens", "1", *options],
                         input="1 2 3\n", capture_output=True, text=True, timeout=120)
    assert out.returncode == 1 and word in out.stderr
