"""A wait of the attention over 8-bit pages that runs out: what the CTA still had to do is NaN, all else is right, and the process' next call names the kernel and the wait.  The kernels' own copies and
products all arrive, so they are compiled into a program whose waits can be told that they have waited long enough."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
ROWS8, CODES128 = 6 << 8, 7 << 8
FREE, FULL, QUERIES, SCORES, WEIGHTS, VALUES = 1, 2, 9, 10, 11, 12   # (as dense_gemm.cuh numbers them)
WAITS = {FREE: "a free stage", FULL: "a stage's copies", QUERIES: "the split queries", SCORES: "scores", WEIGHTS: "softmax weights", VALUES: "weighted values"}


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("wait") / "paged8_wait")
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-I", os.path.join(os.path.dirname(HERE), "lm.rs_b200", "csrc"), "-o", exe, os.path.join(HERE, "paged8_wait.cu")])
    return exe


CASES = [  # head size, sequences, rows of each, prefix: waits that run out (kernel and wait, CTA, warp, waits of the kind before it)
    ((64, 300, 1, 0), [(ROWS8 + FULL, 3, 0, 1), (ROWS8 + FULL, 0, 0, 0), (ROWS8 + FULL, 100, 2, 3), (ROWS8 + FULL, 591, 0, 2)]),
    ((64, 300, 1, 500), [(ROWS8 + FULL, 3, 0, 1), (ROWS8 + FULL, 300, 0, 0), (ROWS8 + FULL, 400, 3, 2)]),
    ((256, 300, 6, 0), [(ROWS8 + FULL, 3, 0, 1), (ROWS8 + FULL, 200, 1, 0)]),
    ((64, 100, 70, 0), [(CODES128 + FULL, 3, 8, 1), (CODES128 + FULL, 4, 9, 0), (CODES128 + FULL, 5, 10, 5), (CODES128 + FREE, 6, 8, 9), (CODES128 + SCORES, 7, 1, 2), (CODES128 + WEIGHTS, 8, 10, 3), (CODES128 + VALUES, 9, 2, 0)]),
    ((128, 100, 40, 300), [(CODES128 + FULL, 30, 8, 4), (CODES128 + FULL, 140, 10, 0), (CODES128 + QUERIES, 10, 10, 1), (CODES128 + SCORES, 0, 0, 0)]),
    ((256, 60, 40, 200), [(CODES128 + FULL, 2, 5, 3), (CODES128 + FULL, 3, 10, 2), (CODES128 + FREE, 4, 7, 6), (CODES128 + SCORES, 50, 3, 1), (CODES128 + WEIGHTS, 60, 10, 0)]),
]


@pytest.mark.parametrize("case, waits", CASES, ids=str)
def test_a_wait_that_runs_out(program, case, waits):
    ran = subprocess.run([program, *(str(x) for x in case), *(str(x) for w in waits for x in w)], capture_output=True, text=True, timeout=100)
    assert ran.returncode == 0, ran.stdout + ran.stderr
    lines = [line.split("|") for line in ran.stdout.splitlines()]
    assert len(lines) == len(waits)
    for (what, *_), (nan, wrong, rows, said, words, after, same) in zip(waits, lines):
        kernel = {ROWS8: "rows8_kernel", CODES128: "codes128_kernel"}[what & ~255]
        assert int(wrong) == 0 and 0 < int(nan) < int(rows), (case, what, nan, wrong)
        assert said == "1" and "results of an earlier call are NaN: " + kernel in words and words.endswith(f" gave up waiting for {WAITS[what & 255]} (device status {what})")
        assert f"NaN: {kernel} gave up" in words   # (paged_attention, which reads the same word, says it in the same words)
        assert after == "0" and same == "1"   # (said once)


FIRST = """
import sys; sys.path.insert(0, sys.argv[1])
import torch
from lmrs_b200 import paged
g = torch.Generator("cuda"); g.manual_seed(1)
i32 = dict(dtype=torch.int32, device="cuda")
rows = int(sys.argv[2])
k, v, q = (torch.randn(rows, h, 64, generator=g, device="cuda").half() for h in (2, 2, 8))
pool = torch.zeros(8, 64, 2, 64, dtype=torch.int8, device="cuda")
pages = paged.QuantPages(pool, pool.clone(), torch.ones(8, 4, 2, device="cuda"), torch.ones(8, 4, 2, device="cuda"))
batch = paged.Batch(torch.tensor([rows], **i32), torch.arange(8, **i32)[None], rows=torch.tensor([0, rows], **i32), max_rows=rows)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    paged.append(pages, batch, k, v)
    out = paged.attention(pages, batch, q)
out.fill_(9.0)
graph.replay()
assert torch.equal(out, paged.attention(pages, batch, q)) and not (out == 9.0).all()
print("ok")
"""


@pytest.mark.parametrize("rows", [3, 300])
def test_a_process_whose_first_call_is_captured(rows):
    """(either kernel needs the word that it may say something in)"""
    lib = os.path.join(os.path.dirname(HERE), "lm.rs_b200")
    assert subprocess.run([sys.executable, "-c", FIRST, lib, str(rows)], check=True, capture_output=True, text=True, timeout=200).stdout.strip() == "ok"
