"""What a layer's first call takes of the card's memory: its workspace and its
kernels, but not the array of the calls that allocate nothing (64 MiB)."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CODE = """
import torch
from moe_amd import synth
from moe_amd.layer import Context
host = synth.build_host_layer(synth.SHAPES["tiny_mixtral"], 3)
layer = synth.make_layer(Context(0), host)
x = torch.from_numpy(synth.activations(3, 4, host.shape.hidden)).cuda()
out = torch.empty_like(x)
torch.cuda.synchronize()
free = torch.cuda.mem_get_info()[0]
layer.feed_forward(x, out)
torch.cuda.synchronize()
print("taken", free - torch.cuda.mem_get_info()[0])
"""


def test_memory_of_the_first_call():
    got = subprocess.run([sys.executable, "-c", CODE], capture_output=True, text=True, timeout=100, cwd=Path(__file__).parent.parent)
    assert got.returncode == 0, got.stderr[-2000:]
    assert int(got.stdout.split("taken")[1]) < 48 << 20
