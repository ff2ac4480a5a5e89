"""specdec_attention_prompt: causal attention of packed rows over the paged
pool, against the definition in 64 bits."""
import math

import pytest
import torch

import specdec as S
from attn_plain import close, rows_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(lens, Hq, Hkv, hd, seed=0, spare=3, wide=0, tail_rows=0, fused=False, sharp=1.0):
    """lens: (rows, cached) of each sequence.  Unused pages, table ends and the
    slots behind every sequence hold NaN."""
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
    kv = torch.full((nb, 2, Hkv, 16, hd), float("nan"), dtype=torch.float16, device=DEV)
    at = 0
    for b, (n, c) in enumerate(lens):
        tables[b, :need[b]] = order[at:at + need[b]].int()
        at += need[b]
        x = torch.randn((2, Hkv, n + c, hd), generator=g, device=DEV, dtype=torch.float32)
        pad = torch.full((2, Hkv, need[b] * 16, hd), float("nan"), device=DEV)
        pad[:, :, :n + c] = x
        kv[tables[b, :need[b]].long()] = pad.reshape(2, Hkv, need[b], 16, hd).permute(2, 0, 1, 3, 4).half()
    width_q = (Hq + 2 * Hkv) * hd if fused else Hq * hd
    buf = torch.randn((max(T, 1), width_q), generator=g, device=DEV) * 1.5 * sharp
    buf[off[-1]:] = float("nan")
    return dict(lens=lens, Hq=Hq, Hkv=Hkv, hd=hd, T=T, nb=nb, tables=tables, kv=kv, q=buf.half(),
                ctx=torch.tensor([c for _, c in lens] or [0], dtype=torch.int32, device=DEV),
                off=torch.tensor(off, dtype=torch.int32, device=DEV),
                out=torch.full((max(T, 1), Hq, hd), 7.0, dtype=torch.float16, device=DEV))


def workspace(s):
    n = S.lib().specdec_attention_prompt_workspace_bytes(len(s["lens"]), s["T"], s["Hq"], s["Hkv"], s["hd"],
                                                         s["tables"].shape[1])
    return torch.full((max(1, n),), 0xFF, dtype=torch.uint8, device=DEV)  # NaN bits: nothing is read unwritten


def call(s, ws=None, stream=None, out=None):
    ws = workspace(s) if ws is None else ws
    out = s["out"] if out is None else out
    st = torch.cuda.current_stream().cuda_stream if stream is None else stream.cuda_stream
    S.check(S.lib().specdec_attention_prompt(
        s["q"].data_ptr(), s["q"].shape[1], s["kv"].data_ptr(), s["nb"], s["Hkv"], s["hd"], s["tables"].data_ptr(),
        s["tables"].shape[1], s["ctx"].data_ptr(), s["off"].data_ptr(), len(s["lens"]), s["T"], s["Hq"],
        out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), st))
    return ws  # held by the caller until the kernels have run


def want(s, b):
    n, c = s["lens"][b]
    lo = int(s["off"][b])
    q = s["q"][lo:lo + n, :s["Hq"] * s["hd"]].reshape(n, s["Hq"], s["hd"])
    L = min(n + c, s["tables"].shape[1] * 16)
    slot = torch.arange(L, device=DEV)
    seen = slot[None] <= c + torch.arange(n, device=DEV)[:, None]
    return rows_plain(q, s["kv"], s["tables"][b], seen)


def verify(s, out=None, what=""):
    torch.cuda.synchronize()
    out = s["out"] if out is None else out
    for b, (n, _) in enumerate(s["lens"]):
        lo = int(s["off"][b])
        o, tol = want(s, b)
        close(out[lo:lo + n], o, tol, f"{what} sequence {b}")
    end = int(s["off"][-1])
    assert bool((out[end:] == 7.0).all()), "rows behind the last sequence were written"


HEADS = [(8, 2, 64), (32, 8, 128), (5, 1, 128), (3, 3, 64), (40, 8, 128), (8, 1, 128)]


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
@pytest.mark.parametrize("lens", [
    [(1, 0)], [(1, 40)], [(16, 0)], [(17, 15)], [(1, 127), (1, 128), (1, 129), (2, 15)],
    [(0, 5), (3, 0), (0, 0), (130, 7), (1, 300)], [(65, 0), (64, 64), (63, 1)], [(257, 129)]])
def test_lengths(cuda_device, Hq, Hkv, hd, lens):
    s = make(lens, Hq, Hkv, hd, seed=hd + len(lens))
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("Hq,Hkv,hd", [(128, 1, 64), (64, 1, 128), (48, 1, 64), (100, 1, 64), (1, 1, 64)])
def test_head_groups(cuda_device, Hq, Hkv, hd):
    s = make([(7, 50), (150, 0)], Hq, Hkv, hd, seed=Hq)
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("lens,heads", [([(1, 9000)], (8, 2, 64)), ([(1, 5000), (1, 100), (3, 2049)], (32, 8, 128)),
                                        ([(2, 4000)] * 3, (5, 1, 128)), ([(300, 3000)], (8, 8, 64)),
                                        ([(1, 700)] * 40, (32, 8, 128))])
def test_long_caches_with_few_rows(cuda_device, lens, heads):
    s = make(lens, *heads, seed=len(lens))
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("heads", [(8, 2, 64), (32, 8, 128)])
def test_long_prompts(cuda_device, heads):
    s = make([(1111, 0), (9, 70), (2050, 33)], *heads, seed=4)
    ws = call(s)
    verify(s)
    del ws


def test_fused_rows_and_padding(cuda_device):
    """Queries inside the [q | k | v] rows, a wider output, rows of no sequence
    in front of the buffer's end."""
    s = make([(70, 3), (5, 200)], 8, 2, 64, seed=2, fused=True, tail_rows=9, wide=40)
    big = torch.full((s["T"], 10, 64), 7.0, dtype=torch.float16, device=DEV)
    ws = call(s, out=big)
    torch.cuda.synchronize()
    assert bool((big[:, 8:] == 7.0).all())
    verify(s, out=big[:, :8])
    del ws


def test_large_scores_in_rising_order(cuda_device):
    """Scores from -90 to 90 whose maximum grows along the keys (the running
    maximum moves at every tile), and the same falling."""
    for sign in (1.0, -1.0):
        s = make([(40, 900), (1, 2500)], 8, 2, 64, seed=3, sharp=0.05)
        for b, (n, c) in enumerate(s["lens"]):
            ramp = torch.linspace(-1, 1, n + c, device=DEV) * sign
            pages = s["tables"][b, :(n + c + 15) // 16].long()
            k = s["kv"][pages, 0].permute(1, 0, 2, 3).reshape(2, -1, 64)
            k[:, :n + c, 0] = (ramp * 60).half()
            s["kv"][pages, 0] = k.reshape(2, -1, 16, 64).permute(1, 0, 2, 3)
        s["q"].view(-1, 8, 64)[:, :, 0] = 12.0
        ws = call(s)
        verify(s)
        del ws


def test_nan_and_infinity_of_later_tokens_reach_later_rows_only(cuda_device):
    for hd, Hq, Hkv in ((64, 8, 2), (128, 8, 2)):
        s = make([(200, 5), (40, 0)], Hq, Hkv, hd, seed=9)
        for b, tok, plane, val in ((0, 5 + 130, 1, float("nan")), (0, 5 + 60, 1, float("inf")),
                                   (0, 5 + 61, 1, float("-inf")), (1, 39, 1, float("inf"))):
            page = int(s["tables"][b, tok // 16])
            s["kv"][page, plane, 0, tok % 16, 3] = val
            s["kv"][page, plane, 1, tok % 16, hd - 1] = val
        ws = call(s)
        verify(s)
        # a NaN key makes the rows that see it NaN, and no other
        s = make([(200, 5)], Hq, Hkv, hd, seed=9)
        page = int(s["tables"][0, (5 + 77) // 16])
        s["kv"][page, 0, 0, (5 + 77) % 16, 0] = float("nan")
        ws = call(s)
        torch.cuda.synchronize()
        G = Hq // Hkv
        assert bool(torch.isnan(s["out"][77:, :G]).all())
        assert not bool(torch.isnan(s["out"][:77]).any()) and not bool(torch.isnan(s["out"][:, G:]).any())
        del ws


def test_tables_shorter_than_the_sequence(cuda_device):
    """Slots past max_blocks * 16 do not exist."""
    s = make([(50, 100)], 8, 2, 64, seed=1)
    s["tables"] = s["tables"][:, :8].contiguous()
    ws = call(s)
    verify(s)
    del ws


def test_table_entries_outside_the_pool_read_block_0(cuda_device):
    s = make([(3, 60)], 8, 2, 64, seed=1)
    s["kv"].nan_to_num_(nan=0.5)
    bad = s["tables"].clone()
    bad[0, 1], bad[0, 2] = 1 << 30, -5
    s["tables"][0, 1], s["tables"][0, 2] = 0, 0
    o = want(s, 0)
    s["tables"] = bad
    ws = call(s)
    torch.cuda.synchronize()
    close(s["out"], *o)
    del ws


@pytest.mark.parametrize("lens", [[(300, 0), (20, 77)], [(1, 4000), (1, 3000)]])
def test_same_bits_again(cuda_device, lens):
    s = make(lens, 32, 8, 128, seed=6)
    ws = call(s)
    torch.cuda.synchronize()
    first = s["out"].clone()
    for _ in range(3):
        s["out"].fill_(7.0)
        call(s, ws)
        torch.cuda.synchronize()
        assert torch.equal(first, s["out"])


def test_streams_graphs_and_two_calls_at_once(cuda_device):
    a = make([(1, 6000)], 8, 2, 64, seed=1)
    b = make([(90, 500), (1, 3000)], 32, 8, 128, seed=2)
    wa, wb = call(a), call(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        call(a, wa, s1)
        call(b, wb, s2)
    verify(a)
    verify(b)
    # captured, then replayed with other lengths in the same buffers
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        call(a, wa)
    with torch.cuda.graph(gb):
        call(b, wb)
    a["lens"] = [(1, 37)]
    a["ctx"].fill_(37)
    a["out"].fill_(7.0)
    b["lens"] = [(20, 500), (71, 2000)]
    b["off"][1] = 20
    b["ctx"][1] = 2000
    b["out"].fill_(7.0)
    b["kv"].nan_to_num_(nan=0.25)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        ga.replay()
    with torch.cuda.stream(s2):
        gb.replay()
    verify(a)
    verify(b)


def test_agrees_with_the_verify_attention(cuda_device):
    """The same rows through specdec_attention (chain mask) and this call."""
    B, R, Hq, Hkv, hd = 3, 20, 8, 2, 64
    s = make([(R, 100), (R, 16), (R, 333)], Hq, Hkv, hd, seed=8)
    s["kv"].nan_to_num_(nan=0.0)
    ws = call(s)
    mask = torch.tensor([(2 << r) - 1 for r in range(R)], dtype=torch.int64, device=DEV)
    other = torch.empty_like(s["out"])
    S.check(S.lib().specdec_attention(s["q"].data_ptr(), s["kv"].data_ptr(), s["nb"], Hkv, hd, s["tables"].data_ptr(),
                                      s["tables"].shape[1], s["ctx"].data_ptr(), mask.data_ptr(), B, R, Hq,
                                      other.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    for b in range(B):
        o, tol = want(s, b)
        close(s["out"][b * R:(b + 1) * R], o, tol)
        close(other[b * R:(b + 1) * R], o, tol)
    del ws


def test_no_rows(cuda_device):
    s = make([(0, 5), (0, 0)], 8, 2, 64)
    ws = call(s)
    verify(s)
    assert math.isclose(float(s["out"][0, 0, 0]), 7.0)
    del ws


@pytest.mark.parametrize("n", [200, 1024])
def test_many_sequences(cuda_device, n):
    """More sequences than the plan keeps at hand: single tokens, empty ones, short prompts, a long cache."""
    lens = [((7 * b) % 4, (37 * b) % 150) for b in range(n)]
    lens[5], lens[n - 1] = (1, 3000), (90, 11)
    s = make(lens, 8, 2, 64, seed=n)
    ws = call(s)
    verify(s)
    del ws


def test_pools_past_32_bits(cuda_device):
    """Pages whose offset passes 2^31 elements."""
    s = make([(3, 700), (70, 100)], 8, 8, 128, seed=1)
    blocks = 70000
    big = torch.zeros((blocks, 2, 8, 16, 128), dtype=torch.float16, device=DEV)
    big[blocks - s["nb"]:] = s["kv"]
    s["tables"] = torch.where(s["tables"] >= 0, s["tables"] + (blocks - s["nb"]), -1).int()
    s["kv"], s["nb"] = big, blocks
    ws = call(s)
    verify(s)
    del ws


def test_a_cut_range_of_which_a_tile_has_nothing(cuda_device):
    """Pieces of the longest tile's range are empty for the first tiles."""
    s = make([(2000, 0)], 8, 1, 128, seed=3)
    ws = call(s)
    verify(s)
    del ws


def test_host_pointers_are_refused(cuda_device):
    s = make([(3, 60)], 8, 2, 64)
    ws = workspace(s)
    host = torch.zeros(1 << 16, dtype=torch.float16)
    for name in ("q", "kv", "out"):
        t = dict(s)
        t[name] = host.view(-1, s[name].shape[-1]) if name == "q" else host
        if name == "out":
            t["out"] = host[:3 * 8 * 64].view(3, 8, 64)
        with pytest.raises(S.SpecdecError) as e:
            call(t, ws)
        assert e.value.code == S.EINVAL and "device" in str(e.value)
    call(s, ws)
    verify(s)


@pytest.mark.parametrize("name", ["tables", "ctx", "off"])
def test_host_tables_and_lengths_are_refused(cuda_device, name):
    s = make([(3, 60), (1, 400)], 8, 2, 64)
    with pytest.raises(S.SpecdecError) as e:
        call(dict(s, **{name: s[name].cpu()}))
    assert e.value.code == S.EINVAL and "device" in str(e.value)
    with pytest.raises(S.SpecdecError) as e:
        call(s, workspace(s).cpu())
    assert e.value.code == S.EINVAL and "device" in str(e.value)
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("lens", [
    [(4700, 0), (1, 30000), (3, 2000), (0, 50), (1, 5)],
    [(7, 300)] * 700,  # as many results as there is no room for
    [(1, 3000)] * 60 + [(4200, 100)] + [(1, 700)] * 70,
])
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 1, 128)])
def test_long_ranges_of_few_rows_beside_many(cuda_device, lens, heads):
    s = make(lens, *heads, seed=5)
    ws = call(s)
    verify(s)
    del ws
