"""Engine.frame_logprobs after sampled frames: the logits written channel by channel, of one stream to a
batch on the tensor cores, against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_op_logprobs import M, check  # noqa: F401 (M is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 3, 20])
def test_sampled_frames(M, weights_path, n):
    eng = M.Engine(weights_path, max_streams=n, max_ctx=64)
    sids = [eng.open() for _ in range(n)]
    for i, sid in enumerate(sids):
        eng.fill_state_random(sid, 5 + i % 20, i)
        eng.generate_begin(sid, i)
    p = M.SampleParams.make(temperature=0.9, top_k=50, top_p=0.95, repetition_penalty=1.3, min_frames=99, greedy=False)
    for frame in range(3):
        codes, stop, _, logits = eng.step(sids, p, want_logits=True)
        assert not stop.any()
        x = torch.from_numpy(logits.reshape(n * 16, 1024))
        lp, ent, ids, top = eng.frame_logprobs(n, top_k=7, temperature=1.1)
        o = {"lp": torch.from_numpy(lp.reshape(-1)), "ent": torch.from_numpy(ent.reshape(-1)),
             "ids": torch.from_numpy(ids.reshape(n * 16, 7)), "top": torch.from_numpy(top.reshape(n * 16, 7))}
        check(x, torch.from_numpy(codes.reshape(-1).astype(np.int32)), 7, 1.1, o)
    eng.close()
