"""Ranks that train the same weights drop different elements: else the noise of dropout is not averaged over them."""
import json
import os
import socket
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# the example as it is, with what each call of the operator keeps written down
WRAPPER = """
import json, os, runpy, sys
sys.path.insert(0, {root!r})
import torch
from nangila import ops
from nangila.models import gpt2
made, plain, first = [], ops.dropout, gpt2.GPT2.__init__

def dropout(x, p, **options):
    state = torch.get_rng_state()
    kept = plain(torch.ones_like(x), p)
    torch.set_rng_state(state)
    made.append(hash(tuple(kept.detach().reshape(-1)[:4096].ne(0).tolist())))
    return plain(x, p, **options)

weights = []
def init(self, cfg):
    first(self, cfg)
    weights.append(float(sum(q.double().abs().sum() for q in self.parameters())))

ops.dropout, gpt2.GPT2.__init__ = dropout, init
sys.argv = ["examples/train_ddp_gpt2.py"] + {args!r}
try:
    runpy.run_path(os.path.join({root!r}, "examples", "train_ddp_gpt2.py"), run_name="__main__")
except SystemExit as e:
    assert not e.code
json.dump({{"masks": made, "weights": weights}}, open(os.path.join({out!r}, "rank" + os.environ["RANK"]), "w"))
"""


@pytest.mark.parametrize("compressor", ["predres", "powersgd"])
def test_masks_differ_between_ranks(tmp_path, compressor):
    path = tmp_path / "wrapped.py"
    path.write_text(WRAPPER.format(root=ROOT, out=str(tmp_path), args=["--tiny", "--steps", "4", "--warmup-steps", "2", "--micro-batch", "2", "--dropout", "0.2", "--compressor", compressor]))
    with socket.socket() as free:
        free.bind(("127.0.0.1", 0))
        port = str(free.getsockname()[1])
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="", OMP_NUM_THREADS="1", PYTHONHASHSEED="0")
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1", "--master-port", port, str(path)],
                       cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    a, b = (json.load(open(tmp_path / f"rank{rank}")) for rank in (0, 1))
    assert len(a["masks"]) == len(b["masks"]) >= 4 * 3 and a["weights"] == b["weights"]
    assert not set(a["masks"]) & set(b["masks"])
    assert len(set(a["masks"])) == len(a["masks"])  # nor does a rank use one twice
