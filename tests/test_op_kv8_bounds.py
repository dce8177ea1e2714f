"""Row bounds that do not ascend, and counts at the ends of their types: skipped and reported, or refused."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest
import torch

from test_op_kv8 import L, M, SENTINEL, attend, batch, status  # noqa: F401 (L and M are fixtures)

ROOT = Path(__file__).resolve().parents[1]


def test_plan_counts(tmp_path):
    exe = tmp_path / "kv8_plan_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    "/usr/local/cuda/include", "-o", str(exe), str(ROOT / "tests" / "cpp" / "kv8_plan_test.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_head_counts_at_the_end_of_their_type(M):
    # counters that step by several heads would pass 2^31
    import test_op_refusals as T
    for heads in (2**31 - 1, 2**31 - 5, 2**30 + 1):
        a = M.RopeArgs(x=T.P, out=2 * T.P, pos=T.P, x_row_stride=8, x_head_stride=0, out_row_stride=8, out_head_stride=8, rows=1,
                       heads=heads, head_dim=8)
        T.refused(M, M.lib().mossgpu_rope_rotate(T.rope(M, rotary_dim=8), a, None), "above 2^30")
        a = T.append(M, q=T.P, q_out=2 * T.P, q_heads=heads, q_out_row_stride=64, q_out_head_stride=64)
        T.refused(M, M.lib().mossgpu_kv8_append(T.cache(M), T.seqs(M, rows=1), T.rope(M), a, None), "above 2^30")


@pytest.mark.parametrize("name", ["tokens", "logprob", "entropy", "top_ids", "top_logprobs"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_logprob_pointers(M, name, off):
    # every pointer that the device would read or write 4 bytes at
    import test_op_refusals as T
    a = dict(logits=T.P, tokens=T.P, logprob=T.P, entropy=T.P, top_ids=T.P, top_logprobs=T.P, row_stride=100, rows=2, vocab=100, top_k=4,
             temperature=1.0)
    T.refused(M, M.lib().mossgpu_token_logprobs(M.LogprobArgs(**{**a, name: T.P + off}), None), "aligned to its type")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,t", [(8192, torch.float32), (65536, torch.bfloat16), (65536, torch.float16)])
def test_rows_claimed_by_many_sequences(M, L, rows, t):
    # every other sequence claims all rows, with 2^18 positions: more tiles than the plan can count.  Nothing is
    # written, and the call says why.  (2, 16 and 16 mean rows of a sequence: the forms for few, some and many.)
    kvh, dim, n = 1, 64, 4096
    pages = 16384
    codes = torch.zeros(2 * kvh * 16 * dim, dtype=torch.uint8, device="cuda")
    scales = torch.ones(2 * kvh * 16, device="cuda")
    table = torch.zeros(1, pages, dtype=torch.int32, device="cuda")
    c = M.KV8Cache(codes.data_ptr(), scales.data_ptr(), table.data_ptr(), 1, 1, pages, kvh, dim, 0)
    group = 2 if t == torch.float16 else 1
    q = torch.zeros(rows, group, dim, dtype=t, device="cuda")
    out = torch.full_like(q, SENTINEL)
    keep, seqs = batch(M, [rows * (i % 2) for i in range(n + 1)], [0] * n, [16 * pages - rows] * n, rows)

    class Dev:
        def struct(self, _):
            return c

    attend(M, L, Dev(), seqs, q, out, 0.125)
    assert status(L) == 9
    assert (out == SENTINEL).all()
    # rows claimed twice, few enough to count: written or left, and none behind them
    keep, seqs = batch(M, [0, 40, 20, 60], [0, 0, 0], [5, 5, 5], 60)
    attend(M, L, Dev(), seqs, q[:60], out[:60], 0.125)
    assert status(L) == 0 and (out[60:] == SENTINEL).all() and ((out[:60] == 0) | (out[:60] == SENTINEL)).all()
