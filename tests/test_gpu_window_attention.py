"""specdec_attention_window: causal attention of packed rows that see a window
and the first tokens, against the definition in 64 bits (bounds in attn_plain)."""
import pytest
import torch

import specdec as S
from attn_plain import close, rows_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN = float("nan")


def seen_by(n, c, window, sinks, slots):
    """[n, slots]: what the rows of a sequence see."""
    p = c + torch.arange(n, device=DEV)[:, None]
    j = torch.arange(slots, device=DEV)[None]
    return (j <= p) & ((j < sinks) | (j > p - window))


def make(lens, Hq, Hkv, hd, window, sinks, seed=0, spare=3, wide=0, tail_rows=0, pad=0, gone=True, sharp=1.5):
    """lens: (rows, cached) of each sequence.  Slots that no row sees hold NaN,
    and with `gone` the pages of such slots alone are given back: their entries
    are -1 or far outside the pool."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    off = [0]
    for n, _ in lens:
        off.append(off[-1] + n)
    T = off[-1] + tail_rows
    need = [(n + c + 15) // 16 for n, c in lens]
    nb = sum(need) + spare
    order = torch.randperm(nb, generator=g, device=DEV)
    width = max(1, max(need, default=1), wide)
    tables = torch.full((max(1, len(lens)), width), -1, dtype=torch.int32, device=DEV)
    kv = torch.full((nb, 2, Hkv, 16, hd), NAN, dtype=torch.float16, device=DEV)
    at = 0
    for b, (n, c) in enumerate(lens):
        pages = order[at:at + need[b]]
        at += need[b]
        x = torch.randn((2, Hkv, n + c, hd), generator=g, device=DEV, dtype=torch.float32)
        any_row = seen_by(n, c, window, sinks, n + c).any(0) if n else torch.zeros(n + c, dtype=torch.bool, device=DEV)
        x[:, :, ~any_row] = NAN
        full = torch.full((2, Hkv, need[b] * 16, hd), NAN, device=DEV)
        full[:, :, :n + c] = x
        kv[pages] = full.reshape(2, Hkv, need[b], 16, hd).permute(2, 0, 1, 3, 4).half()
        used = torch.zeros(need[b] * 16, dtype=torch.bool, device=DEV)
        used[:n + c] = any_row
        used = used.reshape(-1, 16).any(1)
        none = torch.where(torch.arange(need[b], device=DEV) % 2 == 0, -1, 1 << 30)
        tables[b, :need[b]] = (torch.where(used, pages, none) if gone else pages).int()
    q = torch.randn((max(T, 1), Hq * hd + pad), generator=g, device=DEV) * sharp
    q[off[-1]:] = NAN
    return dict(lens=lens, Hq=Hq, Hkv=Hkv, hd=hd, T=T, nb=nb, tables=tables, kv=kv, q=q.half(), window=window, sinks=sinks,
                ctx=torch.tensor([c for _, c in lens] or [0], dtype=torch.int32, device=DEV),
                off=torch.tensor(off, dtype=torch.int32, device=DEV),
                out=torch.full((max(T, 1), Hq, hd), 7.0, dtype=torch.float16, device=DEV))


def workspace(s):
    n = S.lib().specdec_attention_window_workspace_bytes(len(s["lens"]), s["T"], s["Hq"], s["Hkv"], s["hd"],
                                                         s["tables"].shape[1])
    return torch.full((max(1, n),), 0xFF, dtype=torch.uint8, device=DEV)  # NaN bits: nothing is read unwritten


def call(s, ws=None, stream=None, out=None):
    ws = workspace(s) if ws is None else ws
    out = s["out"] if out is None else out
    st = (stream or torch.cuda.current_stream()).cuda_stream
    S.check(S.lib().specdec_attention_window(
        s["q"].data_ptr(), s["q"].shape[1], s["kv"].data_ptr(), s["nb"], s["Hkv"], s["hd"], s["tables"].data_ptr(),
        s["tables"].shape[1], s["ctx"].data_ptr(), s["off"].data_ptr(), len(s["lens"]), s["T"], s["Hq"], s["window"],
        s["sinks"], out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), st))
    return ws  # held by the caller until the kernels have run


def verify(s, out=None, what=""):
    torch.cuda.synchronize()
    out = s["out"] if out is None else out
    for b, (n, c) in enumerate(s["lens"]):
        lo = int(s["off"][b])
        L = min(n + c, s["tables"].shape[1] * 16)
        q = s["q"][lo:lo + n, :s["Hq"] * s["hd"]].reshape(n, s["Hq"], s["hd"])
        table = s["tables"][b].clone()
        table[(table < 0) | (table >= s["nb"])] = 0
        see = seen_by(n, c, s["window"], s["sinks"], L)
        o, tol = rows_plain(q, s["kv"], table, see)
        close(out[lo:lo + n], o, tol, f"{what} sequence {b}")
    end = int(s["off"][-1])
    assert bool((out[end:] == 7.0).all()), "rows behind the last sequence were written"


HEADS = [(8, 2, 64), (32, 8, 128), (5, 1, 128), (3, 3, 64), (40, 8, 128), (8, 1, 128)]


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
@pytest.mark.parametrize("lens", [
    [(1, 0)], [(1, 40)], [(17, 15)], [(1, 127), (1, 128), (1, 129), (2, 15)],
    [(0, 5), (3, 0), (0, 0), (130, 7), (1, 300)], [(65, 0), (64, 64), (63, 1)], [(5, 700)] * 3])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (129, 17)])
def test_lengths(cuda_device, Hq, Hkv, hd, lens, window, sinks):
    s = make(lens, Hq, Hkv, hd, window, sinks, seed=hd + len(lens))
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 33, 100, 127, 128, 129, 500, 10000, (1 << 31) - 1])
@pytest.mark.parametrize("sinks", [0, 1, 4, 15, 16, 17, 40, 300, (1 << 31) - 1])
def test_windows_and_sinks(cuda_device, window, sinks):
    """Borders within pages and on them, sinks that reach the window, one row and many."""
    s = make([(1, 421), (3, 190), (70, 333), (1, 3), (200, 0)], 8, 2, 64, window, sinks, seed=window % 1000 + sinks % 97)
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("Hq,Hkv,hd", [(128, 1, 64), (64, 1, 128), (48, 1, 64), (100, 1, 64), (1, 1, 64), (33, 1, 128), (17, 1, 64)])
def test_head_groups(cuda_device, Hq, Hkv, hd):
    s = make([(7, 50), (150, 0), (1, 90)], Hq, Hkv, hd, 37, 5, seed=Hq)
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("lens,heads,window,sinks", [
    ([(1, 9000)], (8, 2, 64), 4000, 4), ([(1, 5000), (1, 100), (3, 2049)], (32, 8, 128), 1500, 20),
    ([(2, 4000)] * 3, (5, 1, 128), 2048, 0), ([(300, 2000)], (8, 8, 64), 1024, 16), ([(1, 700)] * 40, (32, 8, 128), 333, 3),
    ([(1111, 0), (9, 70), (1050, 33)], (8, 2, 64), 256, 4), ([(900, 100)], (32, 8, 128), 300, 130),
    ([(1, 40000)], (4, 1, 64), 30000, 600)])
def test_long(cuda_device, lens, heads, window, sinks):
    s = make(lens, *heads, window, sinks, seed=len(lens), gone=False)
    s["kv"] = torch.nan_to_num(s["kv"], nan=0.5)
    ws = call(s)
    verify(s)
    del ws


def test_a_window_past_the_context_is_prompt_attention(cuda_device):
    s = make([(1, 200), (33, 100), (4, 0)], 8, 2, 64, 1 << 20, 0, seed=5)
    ws = call(s)
    verify(s)
    n = S.lib().specdec_attention_prompt_workspace_bytes(3, s["T"], 8, 2, 64, s["tables"].shape[1])
    w2, out = torch.empty(n, dtype=torch.uint8, device=DEV), torch.zeros_like(s["out"])
    S.check(S.lib().specdec_attention_prompt(
        s["q"].data_ptr(), s["q"].shape[1], s["kv"].data_ptr(), s["nb"], 2, 64, s["tables"].data_ptr(),
        s["tables"].shape[1], s["ctx"].data_ptr(), s["off"].data_ptr(), 3, s["T"], 8, out.data_ptr(), out.stride(0),
        w2.data_ptr(), n, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    # two roundings to fp16, and of the weights, apart
    assert bool(((out.double() - s["out"].double()).abs() <= 2.0 ** -9 * out.double().abs() + 2.0 ** -8).all())
    del ws


def test_strides_and_padding(cuda_device):
    s = make([(70, 3), (5, 200), (1, 30)], 8, 2, 64, 50, 6, seed=2, tail_rows=9, wide=40, pad=264)
    big = torch.full((s["T"], 10, 64), 7.0, dtype=torch.float16, device=DEV)
    ws = call(s, out=big)
    verify(s, out=big[:, :8])
    assert bool((big[:, 8:] == 7.0).all())
    s["off"] += 2  # rows in front of the first sequence's
    s["q"] = torch.cat([torch.full_like(s["q"][:2], NAN), s["q"][:-2]])
    big.fill_(7.0)
    ws = call(s, out=big)
    verify(s, out=big[:, :8])
    assert bool((big[:2] == 7.0).all())
    del ws


def test_tables_shorter_than_the_sequence(cuda_device):
    """Slots past the table's end do not exist; rows that see no others give zeros."""
    s = make([(40, 100), (1, 140)], 8, 2, 64, 20, 0, seed=6, gone=False)
    s["kv"] = torch.nan_to_num(s["kv"], nan=0.25)
    s["tables"] = s["tables"][:, :7].contiguous()
    ws = call(s)
    verify(s)
    assert bool((s["out"][40] == 0).all()) and bool((s["out"][39] == 0).all())
    del ws


@pytest.mark.parametrize("rows", [1, 6, 140])
def test_nan_and_infinity_reach_the_rows_that_see_them(cuda_device, rows):
    """In V and K of slots that some rows see and others do not, and of sinks."""
    for at, value in ((0, float("inf")), (3, NAN), (4, NAN), (199, -float("inf")), (175, NAN), (176, NAN), (200, float("inf")), (205, NAN)):
        for plane in (0, 1):
            s = make([(rows, 200), (2, 60)], 8, 2, 64, 25, 4, seed=rows + at, gone=False)
            s["kv"] = torch.nan_to_num(s["kv"], nan=0.5)
            if at >= rows + 200:
                continue
            s["kv"][int(s["tables"][0, at // 16]), plane, 1, at % 16, 9 if plane else slice(None)] = value if plane else NAN
            ws = call(s)
            torch.cuda.synchronize()
            q = s["q"].reshape(-1, 8, 64)
            see = seen_by(rows, 200, 25, 4, rows + 200)
            hit = see[:, at]
            got = s["out"][:rows].float()
            if plane == 0:  # a NaN key: the whole row of its group's heads
                assert bool(torch.isnan(got[hit][:, 4:]).all()) and bool(torch.isfinite(got[~hit]).all())
                assert bool(torch.isfinite(got[:, :4]).all())
            else:
                want = got[hit][:, 4:, 9]
                assert bool((torch.isnan(want) if value != value else want == value).all())
                got[hit.nonzero()[:, 0][:, None], torch.arange(4, 8, device=DEV), 9] = 0.0
                assert bool(torch.isfinite(got).all())
            k = torch.where(torch.isfinite(s["kv"]), s["kv"], 0.0)
            if plane == 1:
                o, tol = rows_plain(q[:rows], k, s["tables"][0], see)
                o[hit.nonzero()[:, 0][:, None], torch.arange(4, 8, device=DEV), 9] = 0.0
                close(got, o, tol, f"slot {at}")
            o, tol = rows_plain(q[rows:rows + 2], k, s["tables"][1], seen_by(2, 60, 25, 4, 62))
            close(s["out"][rows:rows + 2], o, tol, "the other sequence")
            del ws


@pytest.mark.parametrize("lens", [[(1, 3000)] * 5, [(3, 900), (1, 20)], [(300, 500)]])
def test_large_scores(cuda_device, lens):
    """Scores of thousands: one slot takes a row, also where it is the first or the last of the window."""
    s = make(lens, 8, 2, 64, 700, 4, seed=9, sharp=90.0, gone=False)
    s["kv"] = torch.nan_to_num(s["kv"], nan=0.0)
    s["kv"][:, 0] *= 4
    ws = call(s)
    torch.cuda.synchronize()
    for b, (n, c) in enumerate(s["lens"]):
        lo = int(s["off"][b])
        o, _ = rows_plain(s["q"][lo:lo + n].reshape(n, 8, 64), s["kv"], s["tables"][b], seen_by(n, c, 700, 4, n + c))
        # 64 additions, each off by 2^-24 of partial sums below 2^15, through sqrt(64): x is off by less than 2^-6, a weight
        # by 2^-6 of itself, before and behind the division, and by its rounding
        most = float(s["kv"][:, 1].abs().max())
        assert bool(((s["out"][lo:lo + n].double() - o).abs() <= (2.0 ** -5 + 2.0 ** -9) * most).all())
        assert bool(torch.isfinite(s["out"][lo:lo + n]).all())
    del ws


def test_many_small_weights(cuda_device):
    """One slot of weight 1 among 30,000 whose weights fp16 alone would lose: their sum is 2^-10.2."""
    s = make([(1, 30000)], 8, 2, 64, 1 << 20, 0, seed=1)
    s["q"].zero_()
    s["q"][:, ::64] = 8.0
    s["kv"].zero_()
    s["kv"][:, 0, :, :, 0] = -17.328  # x = -17.328, weight 2^-25
    s["kv"][:, 1] = 1.0
    page = int(s["tables"][0, 1000])
    s["kv"][page, 0, :, 5, 0] = 0.0
    s["kv"][page, 1, :, 5] = 0.0
    ws = call(s)
    verify(s)
    total = 30000 * 2.718281828459045 ** float(torch.tensor(-17.328, dtype=torch.float16))
    total /= 1 + total
    assert abs(float(s["out"][0, 0, 0]) - total) <= 2.0 ** -10 * total + 2.0 ** -25
    del ws


def test_the_largest_values(cuda_device):
    """Means of 65504 stay finite."""
    for lens in ([(1, 500)], [(40, 300)], [(1, 9000)]):
        s = make(lens, 8, 2, 64, 600, 4, seed=3, gone=False)
        s["kv"] = torch.nan_to_num(s["kv"], nan=0.0)
        s["kv"][:, 1] = 65504.0
        ws = call(s)
        torch.cuda.synchronize()
        n = lens[0][0]
        assert bool((s["out"][:n].double() - 65504.0).abs().max() <= 65504 * (2.0 ** -10 + 2.0 ** -13))
        assert bool(torch.isfinite(s["out"][:n]).all())
        del ws


@pytest.mark.parametrize("lens", [[(1, 3000)] * 9, [(33, 700), (1, 2500)]])
def test_same_bits_again(cuda_device, lens):
    s = make(lens, 32, 8, 128, 1024, 4, seed=8)
    ws = call(s)
    torch.cuda.synchronize()
    first = s["out"].clone()
    for _ in range(5):
        ws.fill_(0xFF)
        call(s, ws)
        torch.cuda.synchronize()
        assert torch.equal(first, s["out"])


def test_streams_graphs_and_two_calls_at_once(cuda_device):
    a = make([(1, 900), (40, 300)], 8, 2, 64, 128, 4, seed=1, gone=False)
    b = make([(1, 700)] * 6, 32, 8, 128, 400, 20, seed=2, gone=False)
    for s in (a, b):
        s["kv"] = torch.nan_to_num(s["kv"], nan=0.5)
    wa, wb = call(a), call(b)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s, w, st in ((a, wa, one), (b, wb, two)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call(s, w, st)
        graphs.append(graph)
    # other lengths in the same memory
    a["ctx"].copy_(torch.tensor([850, 280], dtype=torch.int32))
    a["lens"] = [(1, 850), (40, 280)]
    a["out"].fill_(7.0)
    b["out"].fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(one):
            graphs[0].replay()
        with torch.cuda.stream(two):
            graphs[1].replay()
    verify(a, what="graph")
    verify(b, what="graph")


def test_many_sequences(cuda_device):
    for n in (150, 1024):
        s = make([(1 + (i % 7 == 0), (37 * i) % 90) for i in range(n)], 4, 2, 64, 33, 2, seed=n)
        ws = call(s)
        verify(s)
        del ws


def test_bounds_that_no_caller_should_give(cuda_device):
    """Lengths and bounds out of range or order: the call ends, and writes rows of the buffer only."""
    s = make([(3, 50), (20, 30), (1, 80)], 8, 2, 64, 20, 4, seed=4, wide=9)
    guard = torch.full((1 << 16,), 5.0, dtype=torch.float16, device=DEV)
    for ctx in ([-5, 1 << 30, 80], [(1 << 31) - 1, 0, -(1 << 31)]):
        for off in ([0, 3, 23, 24], [0, 24, 5, 24], [-9, 7, 7, 1 << 30], [24, 24, 24, 24], [9, 6, 3, 0], [0, 1 << 30, -3, 24]):
            s["ctx"].copy_(torch.tensor(ctx, dtype=torch.int64).int())
            s["off"].copy_(torch.tensor(off, dtype=torch.int32))
            ws = call(s)
            torch.cuda.synchronize()
    assert bool((guard == 5.0).all())


def test_host_and_foreign_memory_is_refused(cuda_device):
    s = make([(3, 20)], 8, 2, 64, 16, 4, seed=13)
    ws = call(s)
    for name in ("kv", "tables", "ctx", "off", "q", "out"):
        t = dict(s)
        t[name] = s[name].cpu()
        with pytest.raises(S.SpecdecError, match="not memory of the current device"):
            call(t, ws)
    with pytest.raises(S.SpecdecError, match="workspace"):
        call(s, ws.cpu())
    torch.cuda.synchronize()


@pytest.mark.parametrize("wide", [1100, 90000])
def test_tables_far_wider_than_the_sequences(cuda_device, wide):
    """Where a CTA for every run of the table would find nothing, the pages are cut by the lengths in device memory."""
    heads = (32, 8, 128) if wide == 1100 else (8, 2, 64)
    lens = [(1 + (i % 9 == 0), (37 * i) % 700) for i in range(64)] if wide == 1100 else [(1, 5000), (3, 40), (0, 7), (2, 999)]
    for window, sinks in ((1 << 20, 0), (300, 20)):
        s = make(lens, *heads, window, sinks, seed=wide % 91, wide=wide)
        ws = call(s)
        verify(s)
        first = s["out"].clone()
        ws.fill_(0xFF)
        call(s, ws)
        torch.cuda.synchronize()
        assert torch.equal(first, s["out"])
        del ws


def test_long_calls_under_wide_tables(cuda_device):
    """Pages enough for a second wave of ranges."""
    s = make([(1, 1500 + 7 * i) for i in range(64)], 8, 8, 64, 1 << 20, 0, seed=3, wide=1100, gone=False)
    ws = call(s)
    verify(s)
    del ws


# few rows on average, most of them in one or two sequences
MIXED = [[(1, 300)] * 30 + [(33, 500)], [(0, 40)] * 12 + [(90, 100)], [(1, 90)] * 6 + [(8, 300), (9, 300)] + [(1, 5)] * 6 + [(20, 0)]]


@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 2, 64), (32, 8, 128), (5, 1, 128), (3, 3, 64), (16, 1, 64)])
@pytest.mark.parametrize("lens", MIXED)
@pytest.mark.parametrize("wide", [0, 5000])
def test_a_long_sequence_among_short_ones(cuda_device, Hq, Hkv, hd, lens, wide):
    s = make(lens, Hq, Hkv, hd, 120, 5, seed=Hq, wide=wide, tail_rows=3)
    ws = call(s)
    verify(s)
    del ws


def test_rows_that_move_between_sequences_of_a_captured_call(cuda_device):
    lens = [[(4, 300)] * 20, [(1, 300)] * 19 + [(61, 300)], [(0, 300)] * 10 + [(8, 300)] * 10, [(80, 300)] + [(0, 300)] * 19]
    s = make([(80, 300)] * 20, 32, 8, 128, 100, 4, gone=False)
    s["kv"] = torch.nan_to_num(s["kv"], nan=0.5)
    s["T"], s["lens"] = 80, lens[0]
    s["q"], s["out"] = s["q"][:80].contiguous(), s["out"][:80].contiguous()

    def bounds(x):
        s["off"].copy_(torch.tensor([sum(n for n, _ in x[:i]) for i in range(21)], dtype=torch.int32))
    bounds(lens[0])
    ws = call(s)
    torch.cuda.synchronize()
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        call(s, ws, torch.cuda.current_stream())
    for x in lens[1:] + lens:
        bounds(x)
        s["lens"] = x
        s["out"].fill_(7.0)
        ws.fill_(0xFF)
        graph.replay()
        verify(s, what=str(x[-1]))
