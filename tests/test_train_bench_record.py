"""The secondary benchmark's record tells a run with fused norms and positions from one without."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(*args):
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29599")
    return subprocess.run([sys.executable, "bench/train_bench.py", *args], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("config", ["resnet50-powersgd", "bert-large-dgc"])
def test_an_option_without_effect_is_refused(config):
    r = run("--config", config, "--fused", "--small")
    assert r.returncode == 2 and "--fused" in r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
def test_the_record_says_so(fused):
    r = run("--config", "llama-1.3b-fsdp", "--small", "--steps", "2", "--warmup", "3", "--no-e2e", *(["--fused"] if fused else []))
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads([v for v in r.stdout.splitlines() if v.startswith("{")][-1])
    assert line["config"]["fused"] is fused
