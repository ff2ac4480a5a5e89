"""Weights under speculative decoding: a step verifies its drafts with the plain
call, and adds up the accepted rows alone afterwards, their queries gathered and
the contexts as before.  Rejected drafts then weigh nothing, whatever they hold."""
import pytest
import torch

import test_gpu_accumulate_attention as A
import test_gpu_window_attention as W
from test_gpu_accumulate_attention import NAN

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("heads", [(8, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("accepted", [[1, 5, 3, 2], [1, 1, 1, 1], [5, 5, 5, 5], [0, 4, 0, 5]])
def test_accepted_rows_alone(cuda_device, heads, accepted):
    Hq, Hkv, hd = heads
    ctx = [300, 1, 2100, 77]
    s = A.make([(5, c) for c in ctx], Hq, Hkv, hd, seed=3)
    s["window"], s["sinks"] = 1 << 30, 0
    ws = W.call(s)  # the verification
    W.verify(s)
    assert torch.equal(s["weights"], s["before"])
    rows = [5 * b + i for b, k in enumerate(accepted) for i in range(k)]
    t = dict(s, lens=list(zip(accepted, ctx)), T=len(rows), q=s["q"][rows].contiguous(),
             out=torch.full((len(rows), Hq, hd), 7.0, dtype=torch.float16, device=DEV),
             off=torch.tensor([sum(accepted[:b]) for b in range(5)], dtype=torch.int32, device=DEV))
    for b, (k, c) in enumerate(t["lens"]):  # rejected drafts' keys and values are still in the cache
        for slot in range(c + k, c + 5):
            s["kv"][int(s["tables"][b, slot // 16]), :, :, slot % 16] = NAN
    wa = A.call(t)
    A.verify(t)
    del ws, wa
