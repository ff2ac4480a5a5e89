"""specdec_attention_prompt and specdec_attention_shared_prefix where values are
at their limits: weights far below a row's largest, infinities and NaN in slots
that every row sees, values and scores near the ends of their types."""
import math

import pytest
import torch

import test_gpu_prompt_attention as P
import test_gpu_shared_prefix as X
from attn_plain import close, rows_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def slots_of(s, b, plane, n):
    """K or V [Hkv, n, hd] of sequence b's first n slots (a copy)."""
    pages = s["tables"][b, :(n + 15) // 16].long()
    return s["kv"][pages, plane].permute(1, 0, 2, 3).reshape(s["Hkv"], -1, s["hd"])[:, :n].clone()


def put_slots(s, b, plane, x):
    n = x.shape[1]
    pages = s["tables"][b, :(n + 15) // 16].long()
    full = s["kv"][pages, plane].permute(1, 0, 2, 3).reshape(s["Hkv"], -1, s["hd"])
    full[:, :n] = x.half()
    s["kv"][pages, plane] = full.reshape(s["Hkv"], -1, 16, s["hd"]).permute(1, 0, 2, 3)


def put_scores(s, b, x):
    """Makes the scores of every row of sequence b against its slots x[j], up to
    the keys' rounding: channel 0 alone counts."""
    k = slots_of(s, b, 0, x.numel())
    k[:] = 0
    k[:, :, 0] = (x * math.sqrt(s["hd"]) / 8.0)[None]
    put_slots(s, b, 0, k)
    s["q"].view(-1, s["q"].shape[-1] // s["hd"], s["hd"])[:, :, 0] = 8.0


def put_value(s, b, slot, value, head, column):
    s["kv"][int(s["tables"][b, slot // 16]), 1, head, slot % 16, column] = value


# ------------------------------------------------------------- small weights
def small_weights_bound(s, q, b, seen):
    """As attn_plain's bound, but for weights that are subnormal in fp16: P holds
    2^7 times a weight (the row's largest weight is at least 1), so that what a
    weight loses is at most half a subnormal step, 2^-25, over 2^7."""
    o, tol = rows_plain(q, s["kv"], s["tables"][b], seen)
    n = seen.shape[1]
    v = slots_of(s, b, 1, n).double().abs()
    G = s["Hq"] // s["Hkv"]
    S = torch.stack([seen.double() @ v[h // G] for h in range(s["Hq"])], 1)
    return o, tol - (2.0 ** -25 - 2.0 ** -32) * S


@pytest.mark.parametrize("lens", [[(1, 131072)], [(300, 20000)]])
@pytest.mark.parametrize("below", [22.3, 25.2])
def test_many_small_weights(cuda_device, lens, below):
    """One key of weight 1 and many thousands of 2^-22 to 2^-25: their sum is
    what the output holds, as the large key's value is zero."""
    s = P.make(lens, 8, 2, 64, seed=11)
    (n, c), = lens
    x = torch.full((n + c,), -below * math.log(2.0), device=DEV)
    x[7] = 0.0
    put_scores(s, 0, x)
    v = slots_of(s, 0, 1, n + c).abs() + 0.5
    v[:, 7] = 0.0
    put_slots(s, 0, 1, v)
    ws = P.call(s)
    torch.cuda.synchronize()
    q = s["q"][:n].reshape(n, 8, 64)
    seen = torch.arange(n + c, device=DEV)[None] <= c + torch.arange(n, device=DEV)[:, None]
    close(s["out"][:n], *small_weights_bound(s, q, 0, seen))
    del ws


def test_many_small_weights_under_a_shared_prefix(cuda_device):
    s = X.make([(3, 2500)], [5, 30, 0], 4, 8, 2, 64, seed=12)
    for b in range(3):
        n = s["ctx_host"][b] + 4
        x = torch.full((n,), -24.4 * math.log(2.0), device=DEV)
        x[7] = 0.0
        put_scores(s, b, x)
        v = slots_of(s, b, 1, n)
        v[:, :] = v.abs() + 0.5
        v[:, 7] = 0.0
        put_slots(s, b, 1, v.clamp(max=3))
    ws = X.call(s)
    torch.cuda.synchronize()
    for b in range(3):
        n = s["ctx_host"][b] + 4
        seen = torch.arange(n, device=DEV)[None] <= s["ctx_host"][b] + torch.arange(4, device=DEV)[:, None]
        close(s["out"][b], *small_weights_bound(s, s["q"][b], b, seen), f"sequence {b}")
    del ws


# ------------------------------------------- infinities and NaN that rows see
def some_bad_values(s, b, slots):
    """An infinity, its opposite (both in one column as well) and a NaN of head
    0 and the last in the given slots."""
    last, hd = s["Hkv"] - 1, s["hd"]
    for head in {0, last}:
        put_value(s, b, slots[0], math.inf, head, 0)
        put_value(s, b, slots[1], -math.inf, head, hd - 1)
        put_value(s, b, slots[2], math.nan, head, 5)
        put_value(s, b, slots[0], math.inf, head, 33)
        put_value(s, b, slots[1], -math.inf, head, 33)


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (5, 1, 128)])
@pytest.mark.parametrize("lens", [[(40, 900)], [(200, 5)], [(1, 6000)], [(1, 300), (3, 4000)], [(600, 1500)]])
@pytest.mark.parametrize("weight", ["ordinary", "small", "none"])
def test_infinities_and_nan_of_slots_that_all_rows_see(cuda_device, heads, lens, weight):
    """They reach every row, whatever their weight: 2^-30 (nothing in fp16) and
    2^-300 (nothing in 32 bits) are weights."""
    s = P.make(lens, *heads, seed=13)
    for b, (n, c) in enumerate(lens):
        slots = [c // 3, c // 2, min(c, 3)]
        if weight != "ordinary":
            x = torch.randn(n + c, device=DEV)
            x[slots] = -30 * math.log(2.0) if weight == "small" else -300 * math.log(2.0)
            put_scores(s, b, x)
        some_bad_values(s, b, slots)
    ws = P.call(s)
    P.verify(s)
    del ws


def test_a_cache_of_nan(cuda_device):
    """Every value of a long context NaN: rows that see it are NaN, in time."""
    s = P.make([(300, 5000), (1, 8000), (70, 0)], 8, 2, 128, seed=14)
    for b, c in ((0, 5000), (1, 8000)):
        v = slots_of(s, b, 1, c)
        v[:] = math.nan
        put_slots(s, b, 1, v)
    ws = P.call(s)
    P.verify(s)
    del ws


@pytest.mark.parametrize("R", [1, 5])
@pytest.mark.parametrize("weight", ["ordinary", "small", "none"])
def test_infinities_and_nan_of_a_shared_prefix(cuda_device, R, weight):
    s = X.make([(4, 70), (2, 9)], [9, 0, 200, 33, 500, 3], R, 8, 2, 128, seed=15, alone=(700,))
    for b in range(7):
        n = s["ctx_host"][b] + R
        slots = [100, 130, 3]
        if weight != "ordinary":
            x = torch.randn(n, device=DEV) if b in (0, 4, 6) else torch.zeros(n, device=DEV)
            if b in (0, 4, 6):
                x[slots] = -30 * math.log(2.0) if weight == "small" else -300 * math.log(2.0)
                put_scores(s, b, x)
        if b in (0, 4, 6):
            some_bad_values(s, b, slots)
    ws = X.call(s)
    X.verify(s)
    del ws


@pytest.mark.parametrize("lens", [[(1, 6000)], [(40, 900)], [(3, 4000), (1, 50)]])
@pytest.mark.parametrize("large_first", [False, True])
def test_a_nan_key_of_little_weight_beside_large_scores(cuda_device, lens, large_first):
    """A NaN score makes its rows NaN, also where the keys around it weigh
    nothing against the row's others."""
    s = P.make(lens, 8, 2, 64, seed=16)
    n, c = lens[0]
    x = torch.zeros(n + c, device=DEV)
    (x[:c // 2] if large_first else x[c // 2:]).fill_(250.0)
    put_scores(s, 0, x)
    slot = c - c // 4 if large_first else 19
    s["kv"][int(s["tables"][0, slot // 16]), 0, 1, slot % 16, 9] = math.nan
    ws = P.call(s)
    P.verify(s)
    assert bool(torch.isnan(s["out"][:n, 4:]).all()) and not bool(torch.isnan(s["out"][:n, :4]).any())
    del ws


# --------------------------------------------------- the ends of the types
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("lens", [[(60, 700)], [(1, 5000), (1, 40), (2, 300)], [(500, 0)]])
def test_the_largest_values(cuda_device, heads, lens):
    """All values 65504: a mean of them is 65504 and no infinity."""
    s = P.make(lens, *heads, seed=17)
    for b, (n, c) in enumerate(lens):
        v = slots_of(s, b, 1, n + c)
        v[:] = 65504.0
        v[:, :, 1::2] = -65504.0
        put_slots(s, b, 1, v)
    ws = P.call(s)
    P.verify(s)
    del ws


@pytest.mark.parametrize("lens", [[(200, 300)], [(2, 3000)] * 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_the_largest_values_with_one_key_of_most_weight(cuda_device, lens, hd):
    """One weight, of every fraction between 1 and 2, carries the rows: half its
    rounding to fp16 would take 65504 over the next step, to infinity."""
    s = P.make(lens, 8, 2, hd, seed=20)
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    for b, (n, c) in enumerate(lens):
        x = torch.full((n + c,), -30.0, device=DEV)
        x[3], x[200] = 0.0, 3.55
        put_scores(s, b, x)
        k = slots_of(s, b, 0, n + c)
        k[:, 200, 1] = 1.0
        put_slots(s, b, 0, k)
        v = slots_of(s, b, 1, n + c)
        v[:] = 65504.0
        put_slots(s, b, 1, v)
    q = s["q"].view(-1, 8, hd)
    q[:, :, 1] = (torch.rand(q.shape[:2], generator=g, device=DEV) * math.sqrt(hd) * 0.2).half()
    ws = P.call(s)
    P.verify(s)
    del ws


def test_the_largest_values_under_a_shared_prefix(cuda_device):
    s = X.make([(4, 40)], [9, 0, 200, 33], 5, 8, 2, 128, seed=18, alone=(60,))
    for b in range(5):
        v = slots_of(s, b, 1, s["ctx_host"][b] + 5)
        v[:] = -65504.0
        put_slots(s, b, 1, v)
    ws = X.call(s)
    X.verify(s)
    del ws


@pytest.mark.parametrize("size", [900.0, 7000.0, 40000.0])
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("lens", [[(60, 700)], [(1, 5000), (1, 40), (2, 300)], [(500, 0)]])
def test_very_large_scores(cuda_device, size, heads, lens):
    """Scores up to 2^37, a quarter of the largest apart: the softmax is the mean
    of the largest score's values.  (Each of q and k is one number in all
    channels, so equal keys have equal scores, however a product rounds.)"""
    s = P.make(lens, *heads, seed=19)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    s["q"].fill_(size)
    s["q"].view(-1, heads[0], heads[2])[:, 1::2] = -size
    for b, (n, c) in enumerate(lens):
        k = slots_of(s, b, 0, n + c)
        k[:] = (torch.randint(-4, 5, (n + c,), generator=g, device=DEV) * size / 4)[None, :, None]
        put_slots(s, b, 0, k)
    ws = P.call(s)
    P.verify(s)
    del ws
