"""specdec_attention_accumulate of many rows where values are at their limits:
the weights come from scores that are computed a second time, with the operands
of the product exchanged, and from (m, 1 / l) that the final rows, the merge of
their pieces or the merge of pieces with infinities leave.

Bounds are test_gpu_accumulate_attention's.  A row's weights have to add up to 1
whatever its scores' size, as the scores of the sum l and those of the weights
are the same 32 bits: exponents taken apart from a product of up to 4096 are off
by 2^-13 (a rounding of the product that one of both does not make), and the rest
is 2^-20 (division, exponentials, sums of n weights by 2^-24 of the sum for each
of their log2 n levels and the running sums)."""
import math

import pytest
import torch

from test_gpu_accumulate_attention import NAN, call, make, verify

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

HEADS = [(8, 2, 64), (32, 8, 128)]
# in pieces; of one tile pair each in more items than SMs; without room for pieces
LENS = [[(40, 300), (130, 2000)], [(40, 300)] * 40, [(40, 100), (33, 220)]]


def key(s, b, slot, plane, head):
    return s["kv"][int(s["tables"][b, slot // 16]), plane, head, slot % 16]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS)
def test_a_nan_key(cuda_device, heads, lens):
    """The rows that see it are NaN, and so are the weights of what they see; the other heads and sequences keep theirs."""
    Hq, Hkv, hd = heads
    G = Hq // Hkv
    s = make(lens, *heads, seed=4)
    clean = s["kv"].clone()
    n, c = lens[-1]
    at = c + 7  # seen by rows 7 .. n - 1 of the last sequence
    lo = int(s["off"][-2])
    key(s, len(lens) - 1, at, 0, 1)[3] = NAN
    ws = call(s)
    torch.cuda.synchronize()
    out, w = s["out"].clone(), s["weights"].clone()
    assert bool(torch.isnan(out[lo + 7:, G:2 * G]).all()) and bool(torch.isnan(w[-1, 1, :n + c]).all())
    rest = torch.ones(out.shape[:2], dtype=torch.bool, device=DEV)
    rest[lo + 7:, G:2 * G] = False
    assert bool(torch.isfinite(out[rest]).all())
    rest = torch.ones(w.shape[:2], dtype=torch.bool, device=DEV)
    rest[-1, 1] = False
    assert bool(torch.isfinite(w[rest]).all()) and torch.equal(w[-1, 1, n + c:], s["before"][-1, 1, n + c:])
    # without it the same call: what it does not reach has the same bits
    s["kv"].copy_(clean)
    s["weights"].copy_(s["before"])
    call(s, ws)
    verify(s)
    assert torch.equal(s["weights"][rest], w[rest])
    s["out"][lo + 7:, G:2 * G] = out[lo + 7:, G:2 * G] = 0
    assert torch.equal(s["out"], out)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS)
def test_infinities_and_nan_of_v(cuda_device, heads, lens):
    """They reach the outputs, not the weights."""
    s = make(lens, *heads, seed=5)
    last = len(lens) - 1
    n, c = lens[-1]
    key(s, 0, 2, 1, 0)[5] = math.inf
    key(s, last, c + n // 2, 1, 1)[3] = NAN
    key(s, last, c // 2, 1, 1)[9] = -math.inf
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS)
def test_keys_of_minus_infinity_weigh_nothing(cuda_device, heads, lens):
    s = make(lens, *heads, seed=6)
    s["q"].view(s["q"].shape[0], -1, heads[2])[:, :, 7].abs_().add_(0.5)
    for slot in (0, 31, lens[0][1] + 5):
        key(s, 0, slot, 0, 0)[7] = -math.inf
    ws = call(s)
    verify(s)
    assert torch.equal(s["weights"][0, 0, 31], s["before"][0, 0, 31])
    del ws


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS)
def test_a_row_that_one_slot_takes(cuda_device, heads, lens):
    s = make(lens, *heads, seed=9)
    s["q"].fill_(100.0)
    for b in range(len(lens)):
        s["kv"][int(s["tables"][b, 0]), 0, :, 3] = 60.0
    ws = call(s)
    verify(s)
    for b, (n, _) in enumerate(lens):
        gained = s["weights"][b, :, 3].double() - s["before"][b, :, 3].double()
        assert float((gained - n * heads[0] // heads[1]).abs().max()) < n * 2.0 ** -10, b
    del ws


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS + [[(1, 3000), (6, 300)], [(1, 700)] * 40])
@pytest.mark.parametrize("size", [1.0, 5.0, 16.0, 45.0, 300.0, 3000.0])
def test_large_scores_close_to_one_another(cuda_device, heads, lens, size):
    """Products of a size that keeps few bits behind the point: sums in another order would differ, and the weights of a
    row would not add up to 1."""
    Hq, Hkv, hd = heads
    s = make(lens, *heads, seed=int(size))
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    base = torch.randn((hd,), generator=g, device=DEV)
    # the largest score is hd * size^2 / sqrt(hd), and neighbours of a key differ by about a step of fp16 in each channel
    s["q"].view(s["q"].shape[0], Hq, hd)[:] = (base * size * (1 + 0.01 * torch.randn((s["q"].shape[0], Hq, 1), generator=g, device=DEV))).half()
    noise = torch.randn(s["kv"][:, 0].shape, generator=g, device=DEV)
    s["kv"][:, 0] = (base * size * (1 + 2.0 ** -11 * noise)).half()
    s["weights"].zero_()
    ws = call(s)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(s["out"][:int(s["off"][-1])]).all())
    total = s["weights"].double().sum(2)
    for b, (n, _) in enumerate(lens):
        rows = n * Hq // Hkv
        off = float((total[b] - rows).abs().max())
        assert off <= rows * (2.0 ** -13 + 2.0 ** -20 * 16), f"sequence {b}: {off / rows}"
    del ws
