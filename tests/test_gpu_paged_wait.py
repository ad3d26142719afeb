"""A wait of the tensor-core attention over pages on a barrier where nothing arrives ends within seconds, and the word that the next call reads says which it was; the wait for the end of a part
lasts as long as its tiles go on.  The kernel's own barriers cannot be made to miss an arrival, so the waits are compiled into a program of their own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_waits_that_run_out(tmp_path):
    exe = str(tmp_path / "paged_wait")
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-I", os.path.join(os.path.dirname(HERE), "lm.rs_b200", "csrc"),
                           "-o", exe, os.path.join(HERE, "paged_wait.cu")])
    rows = [line.split("|") for line in subprocess.run([exe], check=True, capture_output=True, text=True, timeout=100).stdout.splitlines()]
    assert [r[0] for r in rows] == ["0", "1", "0", "1"] and [r[3] for r in rows] == ["0"] * 4   # (said once)
    ms = [int(r[1]) for r in rows]
    assert 2000 <= ms[0] < 10000 and ms[1] < 100 and 2000 <= ms[2] < 10000 and ms[3] >= 2500
    assert [r[2] for r in rows] == ["rows128_kernel gave up waiting for scores (device status 1290)", "", "rows128_kernel gave up waiting for the other rows of a part (device status 1296)", ""]


FIRST = """
import sys; sys.path.insert(0, sys.argv[1])
import torch
from lmrs_b200 import paged
g = torch.Generator("cuda"); g.manual_seed(1)
k, v, q = (torch.randn(*s, generator=g, device="cuda").bfloat16() for s in ((8, 64, 2, 64), (8, 64, 2, 64), (64, 8, 64)))
i32 = dict(dtype=torch.int32, device="cuda")
batch = paged.Batch(torch.tensor([400], **i32), torch.arange(8, **i32)[None], rows=torch.tensor([0, 64], **i32), max_rows=64)
pages, graph = paged.KVPages(k, v), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = paged.attention(pages, batch, q)
out.fill_(9.0)
graph.replay()
assert torch.equal(out, paged.attention(pages, batch, q)) and not (out == 9.0).all()
print("ok")
"""


def test_a_process_whose_first_call_is_captured():
    """(64 rows of a KV head's group go to the tensor cores)"""
    lib = os.path.join(os.path.dirname(HERE), "lm.rs_b200")
    assert subprocess.run([sys.executable, "-c", FIRST, lib], check=True, capture_output=True, text=True, timeout=200).stdout.strip() == "ok"
