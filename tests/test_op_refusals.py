"""Arguments that the rotary, 8-bit-cache, attention and log-probability entry points refuse, on
the CPU: a refused call returns non-zero with a message and reaches no device; and the index
arithmetic of the cache as a host program."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
P = 1 << 20  # an aligned address that no call may touch


@pytest.fixture(scope="module")
def M():
    import moss_b200
    moss_b200.build()
    return moss_b200


def refused(M, rc, text):
    msg = M.lib().mossgpu_op_last_error().decode()
    assert rc != 0 and text in msg, msg


def cache(M, **kw):
    d = dict(codes=P, scales=P, page_table=P, n_pages=8, n_slots=2, pages_per_slot=4, kv_heads=2, head_dim=64, format=0)
    return M.KV8Cache(**{**d, **kw})


def seqs(M, **kw):
    return M.SeqBatch(**{**dict(row_start=P, slot=P, ctx_len=P, n_seqs=2, rows=4), **kw})


def rope(M, **kw):
    return M.Rope(**{**dict(steps=P, rotary_dim=64, interleaved=0, magnitude=1.0), **kw})


def append(M, **kw):
    d = dict(k=P, v=P, k_row_stride=128, k_head_stride=64, v_row_stride=128, v_head_stride=64, type=0)
    return M.KV8AppendArgs(**{**d, **kw})


def attn(M, **kw):
    d = dict(q=P, out=2 * P, workspace=P, workspace_bytes=1 << 40, q_row_stride=256, q_head_stride=64, out_row_stride=256,
             out_head_stride=64, q_heads=4, type=0, scale=0.125)
    return M.AttentionKV8Args(**{**d, **kw})


CACHES = [(dict(codes=0), "NULL"), (dict(scales=0), "NULL"), (dict(page_table=0), "NULL"), (dict(codes=P + 8), "16-byte"),
          (dict(scales=P + 4), "16-byte"), (dict(page_table=P + 2), "aligned"), (dict(n_pages=0), "positive"),
          (dict(n_slots=-1), "positive"), (dict(pages_per_slot=0), "positive"), (dict(pages_per_slot=1 << 27), "2^26"),
          (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=1025), "kv_heads"), (dict(head_dim=96), "head_dim"), (dict(format=2), "format")]
BATCHES = [(dict(n_seqs=-1), "n_seqs"), (dict(n_seqs=4097), "n_seqs"), (dict(rows=-1), "rows"), (dict(row_start=0), "NULL"),
           (dict(slot=0), "NULL"), (dict(ctx_len=0), "NULL"), (dict(ctx_len=P + 1), "aligned")]


@pytest.mark.parametrize("kw,text", CACHES)
def test_cache_refusals(M, kw, text):
    L = M.lib()
    refused(M, L.mossgpu_kv8_append(cache(M, **kw), seqs(M), None, append(M), None), text)
    refused(M, L.mossgpu_kv8_read(cache(M, **kw), seqs(M), M.KV8ReadArgs(k=P), None), text)
    refused(M, L.mossgpu_attention_kv8(cache(M, **kw), seqs(M), attn(M), None), text)


@pytest.mark.parametrize("kw,text", BATCHES)
def test_batch_refusals(M, kw, text):
    L = M.lib()
    refused(M, L.mossgpu_kv8_append(cache(M), seqs(M, **kw), None, append(M), None), text)
    refused(M, L.mossgpu_kv8_read(cache(M), seqs(M, **kw), M.KV8ReadArgs(k=P), None), text)
    refused(M, L.mossgpu_attention_kv8(cache(M), seqs(M, **kw), attn(M), None), text)


def test_null_descriptors(M):
    L = M.lib()
    refused(M, L.mossgpu_kv8_append(None, seqs(M), None, append(M), None), "cache")
    refused(M, L.mossgpu_kv8_append(cache(M), None, None, append(M), None), "seqs")
    refused(M, L.mossgpu_kv8_append(cache(M), seqs(M), None, None, None), "args")
    refused(M, L.mossgpu_kv8_read(cache(M), seqs(M), None, None), "args")
    refused(M, L.mossgpu_attention_kv8(cache(M), seqs(M), None, None), "args")
    refused(M, L.mossgpu_rope_rotate(None, M.RopeArgs(), None), "NULL")
    refused(M, L.mossgpu_rope_rotate(rope(M), None, None), "NULL")
    refused(M, L.mossgpu_token_logprobs(None, None), "NULL")


@pytest.mark.parametrize("kw,text", [
    (dict(k=0), "NULL"), (dict(v=0), "NULL"), (dict(type=3), "type"), (dict(type=-1), "type"), (dict(k=P + 2), "aligned"),
    (dict(q=P, q_out=P, q_heads=2), "without a rope"), (dict(pos=P + 1), "aligned")])
def test_append_refusals(M, kw, text):
    refused(M, M.lib().mossgpu_kv8_append(cache(M), seqs(M), None, append(M, **kw), None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=P, q_heads=2), "NULL"), (dict(q=P, q_out=P), "q_heads"),
    (dict(q=P, q_out=2 * P, q_heads=2, q_out_row_stride=64, q_out_head_stride=64), "overlap"),
    (dict(q=P, q_out=P, q_heads=2, q_row_stride=256, q_head_stride=64, q_out_row_stride=128, q_out_head_stride=64), "in place")])
def test_append_query_refusals(M, kw, text):
    refused(M, M.lib().mossgpu_kv8_append(cache(M), seqs(M), rope(M), append(M, **kw), None), text)


@pytest.mark.parametrize("kw,text", [(dict(steps=0), "NULL"), (dict(steps=P + 4), "aligned"), (dict(rotary_dim=0), "rotary_dim"),
                                     (dict(rotary_dim=63), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"),
                                     (dict(magnitude=float("nan")), "magnitude")])
def test_rope_refusals(M, kw, text):
    L = M.lib()
    a = dict(x=P, out=2 * P, pos=P, x_row_stride=64, x_head_stride=64, out_row_stride=64, out_head_stride=64, rows=2, heads=1,
             head_dim=64)
    refused(M, L.mossgpu_rope_rotate(rope(M, **kw), M.RopeArgs(**a), None), text)
    refused(M, L.mossgpu_kv8_append(cache(M), seqs(M), rope(M, **kw), append(M), None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(rows=-1), "rows"), (dict(heads=-2), "heads"), (dict(head_dim=260), "head_dim"), (dict(head_dim=4), "head_dim"),
    (dict(head_dim=68), "head_dim"), (dict(type=7), "type"), (dict(x=0), "NULL"), (dict(out=0), "NULL"), (dict(pos=0), "NULL"),
    (dict(pos=P + 2), "aligned"), (dict(x=P + 2), "aligned"), (dict(out_row_stride=63), "overlap"),
    (dict(out=P, out_row_stride=128), "in place")])
def test_rope_argument_refusals(M, kw, text):
    a = dict(x=P, out=2 * P, pos=P, x_row_stride=64, x_head_stride=64, out_row_stride=64, out_head_stride=64, rows=2, heads=1,
             head_dim=64, type=0)
    refused(M, M.lib().mossgpu_rope_rotate(rope(M), M.RopeArgs(**{**a, **kw}), None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(workspace=0), "NULL"), (dict(workspace=P + 8), "16-byte"),
    (dict(workspace_bytes=100), "workspace too small"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"),
    (dict(type=5), "type"), (dict(scale=float("inf")), "scale"), (dict(mask=P), "mask_words"), (dict(mask_words=1), "mask_words"),
    (dict(mask=P + 2, mask_words=1), "aligned"), (dict(out=P), "out must not be q"), (dict(out_head_stride=32), "overlap"),
    (dict(q=P + 1), "aligned")])
def test_attention_refusals(M, kw, text):
    refused(M, M.lib().mossgpu_attention_kv8(cache(M), seqs(M), attn(M, **kw), None), text)


def test_attention_refuses_what_its_plan_cannot_count(M):
    c = cache(M, pages_per_slot=1 << 26)
    refused(M, M.lib().mossgpu_attention_kv8(c, seqs(M, rows=1000), attn(M), None), "split the call")
    wide = dict(q_heads=64, q_row_stride=4096, out_row_stride=4096, workspace_bytes=1 << 62)
    refused(M, M.lib().mossgpu_attention_kv8(cache(M, kv_heads=1), seqs(M, rows=1 << 25), attn(M, **wide), None), "2^30")
    refused(M, M.lib().mossgpu_attention_kv8(cache(M), seqs(M, rows=1 << 29), attn(M, **wide), None), "2^33")


def test_workspace_bytes(M):
    L = M.lib()
    assert L.mossgpu_attention_kv8_workspace_bytes(None, 4, 4) == 0
    assert L.mossgpu_attention_kv8_workspace_bytes(cache(M), 3, 4) == 0
    assert L.mossgpu_attention_kv8_workspace_bytes(cache(M), 4, 0) == 0
    small, large = (L.mossgpu_attention_kv8_workspace_bytes(cache(M), 2, n) for n in (1, 10000))
    assert 0 < small < large < 64 << 20


@pytest.mark.parametrize("kw,text", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=500001), "vocab"), (dict(type=4), "type"), (dict(top_k=33), "top_k"),
    (dict(top_k=-1), "top_k"), (dict(vocab=5, top_k=6, top_ids=P), "top_k"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=1e-40), "temperature"), (dict(row_stride=99), "row_stride"), (dict(logits=0), "NULL"),
    (dict(logits=P + 2), "aligned"), (dict(tokens=0), "together"), (dict(logprob=0), "together"), (dict(top_k=3), "top_k"),
    (dict(top_ids=P), "top_k"), (dict(tokens=0, logprob=0), "nothing")])
def test_logprob_refusals(M, kw, text):
    a = dict(logits=P, tokens=P, logprob=P, row_stride=100, rows=2, vocab=100, temperature=1.0)
    refused(M, M.lib().mossgpu_token_logprobs(M.LogprobArgs(**{**a, **kw}), None), text)


def test_nothing_to_do_is_no_error(M):
    L = M.lib()
    for kw in (dict(n_seqs=0), dict(rows=0)):
        assert L.mossgpu_kv8_append(cache(M), seqs(M, **kw), None, append(M, k=0, v=0), None) == 0
        assert L.mossgpu_kv8_read(cache(M), seqs(M, **kw), M.KV8ReadArgs(), None) == 0
        assert L.mossgpu_attention_kv8(cache(M), seqs(M, **kw), attn(M, q=0, out=0, workspace=0), None) == 0
    assert L.mossgpu_rope_rotate(rope(M), M.RopeArgs(rows=0, heads=3, head_dim=64), None) == 0
    assert L.mossgpu_token_logprobs(M.LogprobArgs(rows=0, vocab=10, temperature=1.0), None) == 0


def test_rope_steps(M):
    import kv8_ref as R
    import numpy as np
    for rot, base in ((2, 10000.0), (64, 10000.0), (128, 500000.0), (254, 10000.0)):
        steps, mag = M.rope_steps(rot, base)
        f = R.freqs(rot, base)
        want = R.steps_of(f)
        # pow and the division by 2 pi: a few ulp of a double
        assert mag == 1.0 and (np.abs(steps.astype(np.float64) - want.astype(np.float64)) <= 8 * 2.0**-53 * want.astype(np.float64) + 1).all()
    steps, _ = M.rope_steps(64, 10000.0, M.RopeScaling(1, 4.0))
    assert np.allclose(steps.astype(np.float64), R.steps_of(R.freqs(64) / 4).astype(np.float64), rtol=1e-14)
    steps, _ = M.rope_steps(64, 10000.0, M.RopeScaling(2, 4.0))
    assert np.allclose(steps.astype(np.float64), R.steps_of(R.freqs(64, 10000.0 * 4.0 ** (64 / 62))).astype(np.float64), rtol=1e-13)
    steps, mag = M.rope_steps(64, 10000.0, M.RopeScaling(3, 8.0, 4096.0, 1.0, 32.0))
    f = R.freqs(64)
    keep = np.clip((4096.0 * f / (2 * np.pi) - 1.0) / 31.0, 0, 1)
    assert np.allclose(steps.astype(np.float64), R.steps_of(f * keep + f / 8 * (1 - keep)).astype(np.float64), rtol=1e-13)
    assert abs(mag - (0.1 * np.log(8.0) + 1.0)) < 1e-7


def test_rope_steps_refusals(M):
    for args, text in (((63, 1e4, None), "rotary_dim"), ((0, 1e4, None), "rotary_dim"), ((258, 1e4, None), "rotary_dim"),
                       ((64, 1.0, None), "base"), ((64, float("nan"), None), "base"), ((64, 1e4, M.RopeScaling(4, 2.0)), "kind"),
                       ((64, 1e4, M.RopeScaling(1, 0.5)), "factor"), ((2, 1e4, M.RopeScaling(2, 2.0)), "rotary_dim"),
                       ((64, 1e4, M.RopeScaling(3, 2.0, 0.0, 1.0, 32.0)), "ramp"),
                       ((64, 1e4, M.RopeScaling(3, 2.0, 4096.0, 32.0, 1.0)), "ramp")):
        with pytest.raises(M.MossGpuError, match=text):
            M.rope_steps(*args)


def test_cache_index_arithmetic(tmp_path):
    exe = tmp_path / "kv8_index_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    "/usr/local/cuda/include", "-o", str(exe), str(ROOT / "tests" / "cpp" / "kv8_index_test.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
