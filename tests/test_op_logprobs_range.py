"""Token log-probabilities (mossgpu_token_logprobs) at small temperatures and at logits of any size, in
every form of the kernel, against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_op_logprobs import M, check, logits, run  # noqa: F401 (M is a fixture)

pytestmark = pytest.mark.gpu

# rows and vocabularies of fp32 logits that reach: one CTA of 128 and of 512 threads and clusters, two or four
# vectors a thread; a warp a row, CTAs of 128 and 512 threads, more than eight vectors a thread, clusters of those
FORMS = [(5, 300), (4, 3900), (3, 30000), (2, 120000), (1300, 1024), (300, 4096), (76, 16384), (40, 32768), (24, 60000)]


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("temperature", [1e-4, 1e-5, 1e-6, 1e-7, 1e-8, 1e-12, 1e-20, 1e-36])
def test_small_temperatures(M, rows, vocab, temperature):
    # logits of up to 20 / 1e-36 stay within the range of fp32
    x, view, tok = logits(rows, vocab, torch.float32, 11)
    o = run(M, view, tok.cuda(), 5, temperature)
    check(x, tok, 5, temperature, o)
    assert torch.isfinite(o["ent"]).all() and (o["top"][:, 0] <= 0).all()


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale,shift", [(1e4, 0.0), (1e6, 0.0), (1e8, 0.0), (1e20, 0.0), (1.0, 3e4), (1.0, -3e4), (1.0, 1e6), (1.0, -1e6),
                                         (4.0, 1e8), (4.0, -1e8), (1e3, -1e20)])
def test_logits_of_any_size(M, rows, vocab, scale, shift):
    x, _, tok = logits(rows, vocab, torch.float32, 12)
    x = x * scale + shift
    o = run(M, x.cuda(), tok.cuda(), 5)
    check(x, tok, 5, 1.0, o)
    assert torch.isfinite(o["ent"]).all()


@pytest.mark.parametrize("t,scale", [(torch.float16, 1e3), (torch.float16, 1.5e4), (torch.bfloat16, 1e5), (torch.bfloat16, 1e9)])
@pytest.mark.parametrize("rows,vocab", [(5, 700), (3, 30000), (1300, 2048), (24, 128000)])
def test_large_16_bit_logits(M, t, scale, rows, vocab):
    x, _, tok = logits(rows, vocab, torch.float32, 13)
    x = (x.clamp(-4, 4) * scale).to(t)
    check(x, tok, 5, 0.7, run(M, x.cuda(), tok.cuda(), 5, 0.7))


def test_temperatures_that_are_refused(M):
    # 1 / T is finite and log2(e) / T is not: the maximum's own term would be 0 times infinity
    L = M.lib()
    for t in (3e-39, 4.2e-39, 1e-45):
        a = M.LogprobArgs(logits=1 << 20, entropy=1 << 20, row_stride=100, rows=2, vocab=100, temperature=t)
        assert L.mossgpu_token_logprobs(a, None) != 0 and b"temperature" in L.mossgpu_op_last_error()
    x = torch.zeros(1, 100, device="cuda")
    o = run(M, x, torch.zeros(1, dtype=torch.int32, device="cuda"), 1, 4.3e-39)
    assert abs(o["lp"][0] + torch.log(torch.tensor(100.0))) < 1e-5 and o["top"][0, 0] == o["lp"][0]


@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_lowest_value_below_large_logits(M, rows, vocab, t):
    # the distance to the maximum passes the range of fp32, its quotient by the temperature does not
    x, _, tok = logits(rows, vocab, torch.float32, 14)
    x = (x.clamp(0, 9) * 1e37).to(t)
    x[:, :3] = torch.finfo(t).min
    x[:, 3] = 3e38
    tok[:] = torch.arange(rows) % 4
    check(x, tok, 5, 8.0, run(M, x.cuda(), tok.cuda(), 5, 8.0))
