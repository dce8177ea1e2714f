"""Token log-probabilities, entropy and top alternatives (mossgpu_token_logprobs) against the
definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import moss_b200
    moss_b200.build()
    return moss_b200


def run(M, x, tok, k, temperature=1.0, want=("lp", "ent", "ids", "top")):
    """x: a device view [rows][vocab] whose last dimension is contiguous."""
    L = M.lib()
    rows, vocab = x.shape
    o = {"lp": torch.full((rows,), 77.0, device="cuda"), "ent": torch.full((rows,), 77.0, device="cuda"),
         "ids": torch.full((rows, k), -77, dtype=torch.int32, device="cuda"), "top": torch.full((rows, k), 77.0, device="cuda")}
    a = M.LogprobArgs(logits=x.data_ptr(), row_stride=x.stride(0), rows=rows, vocab=vocab, type=R.type_id(x.dtype),
                      top_k=k if "ids" in want or "top" in want else 0, temperature=temperature)
    if "lp" in want:
        a.tokens, a.logprob = tok.data_ptr(), o["lp"].data_ptr()
    if "ent" in want:
        a.entropy = o["ent"].data_ptr()
    if k and "ids" in want:
        a.top_ids = o["ids"].data_ptr()
    if k and "top" in want:
        a.top_logprobs = o["top"].data_ptr()
    assert L.mossgpu_token_logprobs(a, torch.cuda.current_stream().cuda_stream) == 0, L.mossgpu_op_last_error()
    torch.cuda.synchronize()
    return {n: v.cpu() for n, v in o.items()}


def order(x, k):
    """The k first ids by (value descending, id ascending), NaN last."""
    rows = []
    for r in x.float().numpy():
        key = np.where(np.isnan(r), -np.inf, r).astype(np.float64)
        nan = np.isnan(r)
        rows.append(np.lexsort((np.arange(len(r)), -key, nan))[:k])
    return torch.from_numpy(np.array(rows).reshape(len(x), k)).int()


def check(x, tok, k, temperature, o):
    y = x.double() / float(np.float32(temperature))
    top = y.amax(-1, keepdim=True)
    e = torch.where(y > -np.inf, torch.exp(y - top), 0.0)
    z = e.sum(-1, keepdim=True)
    logp = torch.where(y > -np.inf, y - top - torch.log(z), -np.inf)
    ids = order(x, k)
    assert torch.equal(o["ids"], ids)
    # (x - max) / T: two roundings and the inverse's (3 * 2^-24 of its size), ln Z: sums of positive terms, 2^-21,
    # its own rounding; entropy: the same of sum p |x - max| / T
    size = torch.where(y > -np.inf, (y - top).abs(), 0.0)
    tol = size * 2.0**-22 + torch.log(z).abs() * 2.0**-22 + 2.0**-20
    ok = tok.long().clamp(min=0)
    lp = torch.where(tok < 0, 0.0, logp.gather(1, ok[:, None])[:, 0])
    lp_tol = tol.gather(1, ok[:, None])[:, 0]
    for got, want, t in ((o["lp"], lp, lp_tol), (o["top"], logp.gather(1, ids.long()), tol.gather(1, ids.long())),
                         (o["ent"], -(e / z * torch.where(e > 0, logp, 0.0)).sum(-1),
                          2.0**-20 + ((e / z * size).sum(-1) + torch.log(z)[:, 0].abs()) * 2.0**-20)):
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine].double(), want[~fine])
        assert ((got.double() - want).abs()[fine] <= t[fine]).all()


def logits(rows, vocab, t, seed, lead=0, pad=0, banned=0.05):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 3
    x[torch.rand(rows, vocab, generator=g) < banned] = float("-inf")
    x = x.to(t)
    buf = torch.full((lead + rows * (vocab + pad) + 8,), float("nan"), dtype=t, device="cuda")  # what lies around is no logit
    view = buf[lead:].as_strided((rows, vocab), (vocab + pad, 1), lead)
    view.copy_(x)
    tok = torch.randint(-1, vocab, (rows,), generator=g, dtype=torch.int32)
    return x, view, tok


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("rows,vocab,k,lead,pad", [
    (1, 1, 1, 0, 0), (3, 2, 2, 1, 1), (5, 31, 7, 0, 0), (7, 40, 32, 3, 0), (4, 1000, 32, 5, 3), (19, 1024, 5, 0, 0), (3, 1024, 12, 1, 0),
    (6, 1025, 9, 0, 0), (5, 4089, 20, 0, 7), (2, 4096, 1, 0, 0), (3, 4097, 32, 7, 0), (9, 16384, 20, 0, 0), (2, 16377, 32, 1, 1),
    (2, 20001, 10, 0, 1), (3, 50257, 32, 0, 0), (2, 128001, 20, 3, 2), (1, 262145, 8, 0, 0), (1, 500000, 32, 1, 0), (300, 1024, 8, 0, 0)])
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_against_the_definition(M, t, rows, vocab, k, lead, pad, temperature):
    x, view, tok = logits(rows, vocab, t, rows + vocab, lead, pad)
    check(x, tok, k, temperature, run(M, view, tok.cuda(), k, temperature))


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("vocab", [64, 1024, 3000, 16384, 40000, 140000])
@pytest.mark.parametrize("kind", ["equal", "few", "rising", "falling", "two", "lowest", "one", "ties", "zeros"])
def test_shapes_of_rows(M, t, vocab, kind):
    g = torch.Generator().manual_seed(vocab)
    x = torch.full((4, vocab), float("-inf"))
    if kind == "equal":
        x[:] = -2.5
    elif kind == "few":  # fewer allowed tokens than alternatives asked for
        for r in range(4):
            x[r, torch.randint(0, vocab, (3 + 4 * r,), generator=g)] = torch.randn(3 + 4 * r, generator=g)
    elif kind in ("rising", "falling"):
        x[:] = torch.linspace(-20, 5, vocab) * (1 if kind == "rising" else -1)
    elif kind == "two":  # many at two values
        x[:] = torch.randint(0, 2, (4, vocab), generator=g).float()
    elif kind == "lowest":  # a mask of the type's lowest value
        x[:] = torch.finfo(t).min
        x[:, vocab // 2 :: 7] = torch.randn(4, len(range(vocab // 2, vocab, 7)), generator=g)
    elif kind == "one":
        x[:, vocab - 1] = 3.0
    elif kind == "ties":
        x[:] = torch.randint(-40, 40, (4, vocab), generator=g).float() / 4
    else:
        x[:] = torch.where(torch.rand(4, vocab, generator=g) < 0.5, 0.0, -0.0)
    x = x.to(t)
    tok = torch.tensor([0, vocab - 1, vocab // 2, -5], dtype=torch.int32)
    check(x, tok, 32, 1.0, run(M, x.cuda(), tok.cuda(), 32))


def test_empty_and_unsound_rows(M):
    for vocab in (40, 1024, 5000, 30000, 140000):
        x = torch.randn(5, vocab, generator=torch.Generator().manual_seed(1))
        x[0] = float("-inf")
        x[1, vocab // 3] = float("nan")
        x[2, vocab - 1] = float("inf")
        x[3] = float("nan")
        tok = torch.tensor([3, 4, 5, 6, vocab], dtype=torch.int32)
        o = run(M, x.cuda(), tok.cuda(), 20)
        assert torch.equal(o["ids"], order(x, 20))
        assert o["lp"][0] == float("-inf") and o["ent"][0] == 0 and (o["top"][0] == float("-inf")).all()
        for r in (1, 2, 3):
            assert torch.isnan(o["lp"][r]) and torch.isnan(o["ent"][r]) and torch.isnan(o["top"][r]).all()
        assert torch.isnan(o["lp"][4]) and torch.isfinite(o["ent"][4])  # a token past the vocabulary
        import ctypes as C
        code = C.c_int(0)
        assert M.lib().mossgpu_op_device_status(C.byref(code)) == 0 and code.value == 11
        # a negative token asks for none, whatever the row holds
        o = run(M, x.cuda(), torch.full((5,), -1, dtype=torch.int32).cuda(), 20)
        assert (o["lp"] == 0).all()
        assert M.lib().mossgpu_op_device_status(C.byref(code)) == 0 and code.value == 0


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 1e3, 1e30])
def test_temperatures(M, temperature):
    x, view, tok = logits(4, 2000, torch.float32, 3)
    o = run(M, view, tok.cuda(), 5, temperature)
    if temperature == 1e-30:  # all on the largest
        assert (o["ent"] == 0).all() and (o["top"][:, 0] == 0).all() and (o["top"][:, 1:] < -1e20).all()
    else:
        check(x, tok, 5, temperature, o)


def test_any_subset_of_the_outputs(M):
    x, view, tok = logits(6, 1500, torch.float32, 5)
    whole = run(M, view, tok.cuda(), 7)
    for want in (("lp",), ("ent",), ("ids",), ("top",), ("lp", "top"), ("ent", "ids")):
        o = run(M, view, tok.cuda(), 7, want=want)
        for n in o:
            assert torch.equal(o[n], whole[n]) if n in want else (o[n].abs() == 77).all()


def test_captured(M):
    x, view, tok = logits(8, 30000, torch.bfloat16, 5)
    tok = tok.cuda()
    want = run(M, view, tok, 6)
    L = M.lib()
    lp, ids = torch.zeros(8, device="cuda"), torch.zeros(8, 6, dtype=torch.int32, device="cuda")
    a = M.LogprobArgs(logits=view.data_ptr(), tokens=tok.data_ptr(), logprob=lp.data_ptr(), top_ids=ids.data_ptr(),
                      row_stride=view.stride(0), rows=8, vocab=30000, type=2, top_k=6, temperature=1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert L.mossgpu_token_logprobs(a, torch.cuda.current_stream().cuda_stream) == 0
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(lp.cpu(), want["lp"]) and torch.equal(ids.cpu(), want["ids"])


def test_engine_scores_a_frame(M, weights_path):
    # teacher-forced codes, the step's own codes and alternatives under the frame's logits, 3 streams
    eng = M.Engine(weights_path, max_streams=4, max_ctx=64)
    sids = [eng.open() for _ in range(3)]
    rng = np.random.default_rng(5)
    for i, sid in enumerate(sids):
        eng.fill_state_random(sid, 5 + 7 * i, i)
        eng.generate_begin(sid, i)
    p = M.SampleParams.make(greedy=True, repetition_penalty=1.2, min_frames=99)
    for forced in (rng.integers(0, 1024, (3, 16)).astype(np.int32), None):
        codes, stop, _, logits = eng.step(sids, p, forced=forced, want_logits=True)
        assert not stop.any()
        x = torch.from_numpy(logits.reshape(48, 1024))
        for asked in (forced, None):
            if asked is None:
                asked_codes = codes
            else:
                asked_codes = asked.copy()
                asked_codes[1, 3] = -1
            lp, ent, ids, top = eng.frame_logprobs(3, None if asked is None else asked_codes, top_k=6, temperature=0.9)
            o = {"lp": torch.from_numpy(lp.reshape(-1)), "ent": torch.from_numpy(ent.reshape(-1)),
                 "ids": torch.from_numpy(ids.reshape(48, 6)), "top": torch.from_numpy(top.reshape(48, 6))}
            check(x, torch.from_numpy(asked_codes.reshape(-1)), 6, 0.9, o)
    lp, ent, ids, top = eng.frame_logprobs(3)
    assert ids is None and top is None and (lp < 0).all() and (ent > 0).all()
    bad = np.full((3, 16), 1024, np.int32)
    for kw, text in ((dict(n=2), "number of streams"), (dict(n=3, codes=bad), "out of range"), (dict(n=3, top_k=33), "top_k"),
                     (dict(n=3, temperature=0.0), "temperature")):
        with pytest.raises(M.MossGpuError, match=text):
            eng.frame_logprobs(**kw)
    eng.step_frames(sids, p, 2)
    with pytest.raises(M.MossGpuError, match="number of streams"):
        eng.frame_logprobs(3)
    eng.close()
