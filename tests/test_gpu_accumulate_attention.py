"""specdec_attention_accumulate: causal attention of packed rows that adds up
what weight each slot received, against the definition in 64 bits.

The output's bounds are attn_plain's.  A weight comes from scores, exponents and
sums in 32 bits: as there, 2^-13 of itself, and 2^-22 for its exponential and the
division; adding up rounds by 2^-24 of the running sum for each of the rows and
heads, and of what was there: with at most 2^10 of them in these tests, 2^-14 of
the sum and 2^-24 of the base's and the result's sizes."""
import math

import pytest
import torch

import specdec as S
from attn_plain import close, rows_plain
from test_gpu_window_attention import MIXED, NAN, make as make_window

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(lens, Hq, Hkv, hd, seed=0, more=0, **kw):
    s = make_window(lens, Hq, Hkv, hd, 1 << 30, 0, seed, **kw)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed + 1)
    s["ldw"] = s["tables"].shape[1] * 16 + more
    s["weights"] = torch.rand((max(1, len(lens)), Hkv, s["ldw"]), generator=g, device=DEV)
    s["before"] = s["weights"].clone()
    return s


def workspace(s):
    n = S.lib().specdec_attention_accumulate_workspace_bytes(len(s["lens"]), s["T"], s["Hq"], s["Hkv"], s["hd"],
                                                             s["tables"].shape[1])
    return torch.full((max(1, n),), 0xFF, dtype=torch.uint8, device=DEV)  # NaN bits: nothing is read unwritten


def call(s, ws=None, stream=None, out=None):
    ws = workspace(s) if ws is None else ws
    out = s["out"] if out is None else out
    st = (stream or torch.cuda.current_stream()).cuda_stream
    S.check(S.lib().specdec_attention_accumulate(
        s["q"].data_ptr(), s["q"].shape[1], s["kv"].data_ptr(), s["nb"], s["Hkv"], s["hd"], s["tables"].data_ptr(),
        s["tables"].shape[1], s["ctx"].data_ptr(), s["off"].data_ptr(), len(s["lens"]), s["T"], s["Hq"],
        s["weights"].data_ptr(), s["ldw"], out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), st))
    return ws


def weights_of(q, kv, table, seen):
    """[Hkv, slots] in 64 bits."""
    n, Hq, hd = q.shape
    Hkv = kv.shape[2]
    pages = table[:(seen.shape[1] + 15) // 16].long()
    w = torch.zeros((Hkv, seen.shape[1]), dtype=torch.float64, device=DEV)
    for h in range(Hq):
        k = kv[pages, 0, h // (Hq // Hkv)].double().reshape(-1, hd)[:seen.shape[1]]
        x = torch.where(seen, q[:, h].double() @ torch.where(seen.any(0)[:, None], k, 0.0).T / math.sqrt(hd), -math.inf)
        top = x.amax(1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        w[h // (Hq // Hkv)] += (p / p.sum(1, keepdim=True).clamp(min=1e-300)).sum(0)
    return w


def verify(s, out=None, what="", times=1):
    torch.cuda.synchronize()
    out = s["out"] if out is None else out
    rest = torch.ones(s["weights"].shape, dtype=torch.bool, device=DEV)
    for b, (n, c) in enumerate(s["lens"]):
        lo = int(s["off"][b])
        L = min(n + c, s["tables"].shape[1] * 16)
        q = s["q"][lo:lo + n, :s["Hq"] * s["hd"]].reshape(n, s["Hq"], s["hd"])
        see = torch.arange(L, device=DEV)[None] <= c + torch.arange(n, device=DEV)[:, None]
        o, tol = rows_plain(q, s["kv"], s["tables"][b], see)
        close(out[lo:lo + n], o, tol, f"{what} sequence {b}")
        if n == 0 or L == 0:
            continue
        w = weights_of(q, s["kv"], s["tables"][b], see) * times
        base = s["before"][b, :, :L].double()
        bound = (2.0 ** -13 + 2.0 ** -14) * w + times * 2.0 ** -23 * (base + w)
        over = ((s["weights"][b, :, :L].double() - base - w).abs() / bound).max()
        assert float(over) <= 1.0, f"{what} weights of sequence {b}: {float(over)} of the bound"
        rest[b, :, :L] = False
    assert torch.equal(s["weights"][rest], s["before"][rest]), "weights of slots that no row sees"
    end = int(s["off"][-1])
    assert bool((out[end:] == 7.0).all()), "rows behind the last sequence were written"


HEADS = [(8, 2, 64), (32, 8, 128), (5, 1, 128), (3, 3, 64), (40, 8, 128), (32, 1, 64), (1, 1, 128), (17, 1, 64)]


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
@pytest.mark.parametrize("lens", [
    [(1, 0)], [(1, 40)], [(16, 0)], [(17, 15)], [(1, 127), (1, 128), (1, 129), (2, 15)],
    [(0, 5), (3, 0), (0, 0), (130, 7), (1, 300)], [(65, 0), (64, 64), (63, 1)]])
def test_lengths(cuda_device, Hq, Hkv, hd, lens):
    s = make(lens, Hq, Hkv, hd, seed=hd + len(lens), more=4 * len(lens))
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("lens,heads", [
    ([(1, 9000)], (8, 2, 64)), ([(1, 5000), (1, 100), (3, 2049)], (32, 8, 128)), ([(2, 4000)] * 3, (5, 1, 128)),
    ([(32, 3000)], (8, 8, 64)), ([(1, 700)] * 40, (32, 8, 128)), ([(16, 2000), (16, 1), (16, 555)], (40, 8, 128)),
    ([(1, 40000)], (4, 1, 64)), ([(5, 1000)] * 7, (40, 8, 128))])
def test_long(cuda_device, lens, heads):
    s = make(lens, *heads, seed=len(lens))
    ws = call(s)
    verify(s)
    del ws


def test_steps_add_up(cuda_device):
    s = make([(1, 300), (3, 77)], 8, 2, 64, seed=5)
    ws = workspace(s)
    for _ in range(4):
        call(s, ws)
    verify(s, times=4)
    # the weights of a row sum to 1 for each head
    gained = (s["weights"].double() - s["before"].double()).sum((1, 2))
    assert abs(float(gained[0]) - 4 * 8) < 1e-3 and abs(float(gained[1]) - 4 * 24) < 1e-3


def test_strides_and_padding(cuda_device):
    s = make([(70, 3), (5, 200), (1, 30)], 8, 2, 64, seed=2, tail_rows=9, wide=40, pad=264, more=8)
    big = torch.full((s["T"], 10, 64), 7.0, dtype=torch.float16, device=DEV)
    ws = call(s, out=big)
    verify(s, out=big[:, :8])
    assert bool((big[:, 8:] == 7.0).all())
    del ws


def test_tables_shorter_than_the_sequence(cuda_device):
    s = make([(40, 100), (1, 130), (3, 20)], 8, 2, 64, seed=6)
    s["tables"] = s["tables"][:, :7].contiguous()
    ws = call(s)
    verify(s)
    del ws


def test_nan_reaches_the_weights_of_the_rows_that_see_it(cuda_device):
    """A NaN key makes the rows that see it NaN, and the weights of all that these rows see; other heads and
    sequences, and slots of other rows alone, keep theirs."""
    s = make([(3, 200), (1, 60)], 8, 2, 64, seed=4)
    s["kv"][int(s["tables"][0, 201 // 16]), 0, 1, 201 % 16, 3] = NAN  # seen by rows 1 and 2
    ws = call(s)
    torch.cuda.synchronize()
    assert bool(torch.isnan(s["out"][1:3, 4:]).all()) and bool(torch.isfinite(s["out"][0]).all())
    assert bool(torch.isfinite(s["out"][:, :4]).all()) and bool(torch.isfinite(s["out"][3]).all())
    w = s["weights"]
    assert bool(torch.isnan(w[0, 1, :203]).all()) and bool(torch.isfinite(w[0, 0]).all()) and bool(torch.isfinite(w[1]).all())
    assert torch.equal(w[0, 1, 203:], s["before"][0, 1, 203:])
    # in V: the outputs, not the weights
    s = make([(3, 200), (1, 60)], 8, 2, 64, seed=4)
    s["kv"][int(s["tables"][0, 201 // 16]), 1, 1, 201 % 16, 3] = NAN
    s["kv"][int(s["tables"][0, 0]), 1, 0, 2, 5] = math.inf
    ws = call(s)
    torch.cuda.synchronize()
    assert bool(torch.isnan(s["out"][1:3, 4:, 3]).all()) and bool((s["out"][:3, :4, 5] == math.inf).all())
    assert bool(torch.isfinite(s["weights"]).all())
    verify(s)
    del ws


def test_a_row_that_one_slot_takes(cuda_device):
    """Scores of thousands: the weight of the largest is 1, the others' are 0."""
    s = make([(1, 700), (6, 300)], 8, 2, 64, seed=9)
    s["q"].fill_(100.0)
    for b, at in ((0, 700), (1, 3)):
        s["kv"][int(s["tables"][b, at // 16]), 0, :, at % 16] = 60.0
    ws = call(s)
    verify(s)
    assert abs(float(s["weights"][1, 0, 3] - s["before"][1, 0, 3]) - 24) < 1e-4
    del ws


@pytest.mark.parametrize("lens", [[(1, 3000)] * 9, [(16, 700), (1, 2500)]])
def test_same_bits_again(cuda_device, lens):
    s = make(lens, 32, 8, 128, seed=8)
    ws = call(s)
    torch.cuda.synchronize()
    first, w = s["out"].clone(), s["weights"].clone()
    for _ in range(5):
        ws.fill_(0xFF)
        s["weights"].copy_(s["before"])
        call(s, ws)
        torch.cuda.synchronize()
        assert torch.equal(first, s["out"]) and torch.equal(w, s["weights"])


def test_streams_graphs_and_two_calls_at_once(cuda_device):
    a = make([(1, 900), (10, 300)], 8, 2, 64, seed=1)
    b = make([(1, 700)] * 6, 32, 8, 128, seed=2)
    wa, wb = call(a), call(b)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s, w, st in ((a, wa, one), (b, wb, two)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call(s, w, st)
        graphs.append(graph)
    a["ctx"].copy_(torch.tensor([850, 280], dtype=torch.int32))
    a["lens"] = [(1, 850), (10, 280)]
    for s in (a, b):
        s["weights"].copy_(s["before"])
        s["out"].fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(one):
            graphs[0].replay()
        with torch.cuda.stream(two):
            graphs[1].replay()
    verify(a, what="graph", times=3)
    verify(b, what="graph", times=3)


def test_many_sequences(cuda_device):
    for n in (150, 1024):
        s = make([(1 + (i % 7 == 0), (37 * i) % 90) for i in range(n)], 4, 2, 64, seed=n)
        ws = call(s)
        verify(s)
        del ws


def test_bounds_that_no_caller_should_give(cuda_device):
    s = make([(3, 50), (20, 30), (1, 80)], 8, 2, 64, seed=4, wide=9)
    s["kv"] = torch.nan_to_num(s["kv"], nan=0.5)
    guard = torch.full((1 << 16,), 5.0, dtype=torch.float16, device=DEV)
    for ctx in ([-5, 1 << 30, 80], [(1 << 31) - 1, 0, -(1 << 31)]):
        for off in ([0, 3, 23, 24], [0, 24, 5, 24], [-9, 7, 7, 1 << 30], [24, 24, 24, 24], [9, 6, 3, 0], [0, 1 << 30, -3, 24]):
            s["ctx"].copy_(torch.tensor(ctx, dtype=torch.int64).int())
            s["off"].copy_(torch.tensor(off, dtype=torch.int32))
            ws = call(s)
            torch.cuda.synchronize()
    assert bool((guard == 5.0).all())
    del ws


def test_host_and_foreign_memory_is_refused(cuda_device):
    s = make([(3, 20)], 8, 2, 64, seed=13)
    ws = call(s)
    for name in ("kv", "tables", "ctx", "off", "q", "out", "weights"):
        t = dict(s)
        t[name] = s[name].cpu()
        with pytest.raises(S.SpecdecError, match="not memory of the current device"):
            call(t, ws)
    with pytest.raises(S.SpecdecError, match="workspace"):
        call(s, ws.cpu())
    torch.cuda.synchronize()


@pytest.mark.parametrize("wide", [1100, 90000])
def test_tables_far_wider_than_the_sequences(cuda_device, wide):
    heads = (32, 8, 128) if wide == 1100 else (8, 2, 64)
    lens = [(1 + (i % 9 == 0), (37 * i) % 700) for i in range(64)] if wide == 1100 else [(1, 5000), (3, 40), (0, 7), (2, 999)]
    s = make(lens, *heads, seed=wide % 91, wide=wide)
    ws = call(s)
    verify(s)
    del ws


def test_scores_past_what_is_kept(cuda_device):
    """Tables so wide that the rows' scores would take more than 1 GiB: they are computed again."""
    s = make([(1, 300), (2, 50)], 8, 2, 64, seed=3, wide=800000)
    ws = call(s)
    assert ws.numel() < 3 << 30
    verify(s)
    del ws


def test_many_rows_beside_many_sequences(cuda_device):
    """One CTA goes through several runs of a sequence's slots."""
    s = make([(0, 3)] * 1000 + [(4200, 0)] + [(0, 0)] * 23, 32, 4, 64, seed=5)
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("G", [1, 3, 5, 7, 8, 12, 16, 31, 32])
@pytest.mark.parametrize("lens", [[(1, 700), (2, 130)], [(40, 300), (3, 90)]])
def test_head_groups(cuda_device, G, lens):
    s = make(lens, 2 * G, 2, 64 if G % 2 else 128, seed=G)
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("lens,heads", [([(1, 5)] * 40, (32, 8, 128)), ([(4, 20)] * 12, (40, 8, 128)),
                                        ([(0, 30)] * 3 + [(200, 0)], (8, 2, 64))])
def test_what_follows_a_captured_call_sees_its_results(cuda_device, lens, heads):
    # tables of several runs, sequences of one: nothing is left for the last kernel of the call to do
    s = make(lens, *heads, seed=8, wide=1 << 8)
    ws = call(s)
    torch.cuda.synchronize()
    kept, gained = torch.empty_like(s["out"]), torch.empty_like(s["weights"])
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        s["out"].fill_(7.0)
        s["weights"].copy_(s["before"])
        call(s, ws, torch.cuda.current_stream())
        kept.copy_(s["out"])
        gained.copy_(s["weights"])
    for _ in range(5):
        kept.zero_()
        gained.zero_()
        graph.replay()
        torch.cuda.synchronize()
        s["weights"].copy_(gained)
        verify(s, out=kept)


@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 2, 64), (32, 8, 128), (5, 1, 128), (3, 3, 64), (16, 1, 64)])
@pytest.mark.parametrize("lens", MIXED)
@pytest.mark.parametrize("wide", [0, 5000])
def test_a_long_sequence_among_short_ones(cuda_device, Hq, Hkv, hd, lens, wide):
    s = make(lens, Hq, Hkv, hd, seed=Hq, wide=wide, tail_rows=3)
    ws = workspace(s)
    for _ in range(2):
        call(s, ws)
    verify(s, times=2)
