"""How the prompt and shared-prefix attention cut their key ranges, read from the
workspace: 256 bytes, then six int32 a sequence (pieces of the shared prefix,
first row, stride; pieces of the own range, first row, stride)."""
import pytest
import torch

import test_gpu_prompt_attention as P
import test_gpu_shared_prefix as X

pytestmark = pytest.mark.gpu


def pieces(ws, sequences):
    torch.cuda.synchronize()
    return ws[256:256 + 24 * sequences].view(torch.int32).view(sequences, 6)[:, [0, 3]].tolist()


@pytest.mark.parametrize("prompt", [2800, 2900])
def test_a_long_range_is_cut_beside_many_short_ones(cuda_device, prompt):
    """A token on 100,000 slots beside 250 sequences of 5 rows, in calls of less
    and of more than 4096 rows: one CTA would walk 782 key tiles for it."""
    lens = [(5, 600)] * 250 + [(prompt, 0), (1, 100000)]
    s = P.make(lens, 32, 8, 128, seed=2)
    ws = P.call(s)
    got = pieces(ws, len(lens))
    assert got[251][1] >= 16
    off = s["off"].tolist()
    for b in (0, 1, 249, 250, 251):
        P.close(s["out"][off[b]:off[b + 1]], *P.want(s, b), f"sequence {b}")
    del ws


@pytest.mark.parametrize("groups,R,own,alone", [
    ([(200, 30)], 21, 90, ()), ([(40, 12), (0, 3), (60, 5)], 64, 33, (70, 5)),  # more rows than there is room for duals
    ([(3, 4)], 5, 40, (90,)), ([], 5, 0, (3, 40, 0, 200)), ([], 64, 0, (150,) * 60), ([], 3, 0, (900, 5000) * 30)])
def test_shared_prefixes_in_the_room_there_is(cuda_device, groups, R, own, alone):
    """Calls of many rows, of short tables (16 pages at most) and of no groups."""
    n = sum(g for g, _ in groups)
    s = X.make(groups, [(own * b) % (own + 1) for b in range(n)], R, 8, 2, 64, seed=R + n, alone=alone)
    ws = X.call(s)
    X.verify(s)
    del ws
