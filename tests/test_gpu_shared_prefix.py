"""specdec_attention_shared_prefix: verify rows of sequences whose tables begin
with the same pages, against the definition in 64 bits."""
import pytest
import torch

import specdec as S
from attn_plain import close, rows_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def chain(R):
    return [(2 << r) - 1 for r in range(R)]


def tree(R):
    bits = [1]
    for r in range(1, R):
        bits.append(bits[(r - 1) // 2] | 1 << r)
    return bits


def make(groups, own, R, Hq, Hkv, hd, masks=None, seed=0, alone=()):
    """groups: (sequences, shared pages) each; own: context tokens of each
    sequence behind its shared pages; alone: sequences of no group, behind.
    Everything that no row sees holds NaN."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    off = [0]
    for n, _ in groups:
        off.append(off[-1] + n)
    B = off[-1] + len(alone)
    own = list(own) + list(alone)
    assert len(own) == B
    shared = [p for n, p in groups for _ in range(n)] + [0] * len(alone)
    ctx = [16 * shared[b] + own[b] for b in range(B)]
    mine = [(ctx[b] + R + 15) // 16 - shared[b] for b in range(B)]
    nb = sum(p for _, p in groups) + sum(mine) + 2
    order = torch.randperm(nb, generator=g, device=DEV).int()
    wide = max(shared[b] + mine[b] for b in range(B)) + 1
    tables = torch.full((B, wide), -1, dtype=torch.int32, device=DEV)
    kv = torch.randn((nb, 2, Hkv, 16, hd), generator=g, device=DEV).half()
    at = 0
    for gi, (n, p) in enumerate(groups):
        for b in range(off[gi], off[gi + 1]):
            tables[b, :p] = order[at:at + p]
        at += p
    for b in range(B):
        tables[b, shared[b]:shared[b] + mine[b]] = order[at:at + mine[b]]
        at += mine[b]
        end = ctx[b] + R
        if end % 16:
            kv[int(tables[b, end // 16]), :, :, end % 16:] = float("nan")
    kv[order[at:].long()] = float("nan")
    masks = chain(R) if masks is None else masks
    return dict(B=B, R=R, Hq=Hq, Hkv=Hkv, hd=hd, nb=nb, tables=tables, kv=kv, masks=masks, ctx_host=ctx,
                ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV),
                mask=torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device=DEV),
                goff=torch.tensor(off, dtype=torch.int32, device=DEV),
                pages=torch.tensor([p for _, p in groups] or [0], dtype=torch.int32, device=DEV), ng=len(groups),
                q=(torch.randn((B, R, Hq, hd), generator=g, device=DEV) * 1.5).half(),
                out=torch.full((B, R, Hq, hd), 7.0, dtype=torch.float16, device=DEV))


def workspace(s):
    n = S.lib().specdec_attention_shared_prefix_workspace_bytes(s["B"], s["R"], s["ng"], s["Hq"], s["Hkv"], s["hd"],
                                                                s["tables"].shape[1])
    return torch.full((max(1, n),), 0xFF, dtype=torch.uint8, device=DEV)


def call(s, ws=None, stream=None):
    ws = workspace(s) if ws is None else ws
    st = torch.cuda.current_stream().cuda_stream if stream is None else stream.cuda_stream
    S.check(S.lib().specdec_attention_shared_prefix(
        s["q"].data_ptr(), s["kv"].data_ptr(), s["nb"], s["Hkv"], s["hd"], s["tables"].data_ptr(),
        s["tables"].shape[1], s["ctx"].data_ptr(), s["mask"].data_ptr(), s["goff"].data_ptr(), s["pages"].data_ptr(),
        s["ng"], s["B"], s["R"], s["Hq"], s["out"].data_ptr(), ws.data_ptr(), ws.numel(), st))
    return ws


def verify(s, what=""):
    torch.cuda.synchronize()
    R = s["R"]
    bits = torch.tensor([[m >> i & 1 for i in range(R)] for m in s["masks"]], device=DEV) == 1
    for b in range(s["B"]):
        c = s["ctx_host"][b]
        L = min(c + R, s["tables"].shape[1] * 16)
        seen = torch.ones((R, c + R), dtype=torch.bool, device=DEV)
        seen[:, c:] = bits
        o, tol = rows_plain(s["q"][b], s["kv"], s["tables"][b], seen[:, :L])
        close(s["out"][b], o, tol, f"{what} sequence {b}")


@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 2, 64), (32, 8, 128), (5, 1, 128), (40, 8, 128), (4, 4, 64), (64, 1, 64)])
@pytest.mark.parametrize("R", [1, 5, 16])
def test_one_group(cuda_device, Hq, Hkv, hd, R):
    s = make([(4, 9)], [0, 1, 33, 200], R, Hq, Hkv, hd, seed=R)
    ws = call(s)
    verify(s)
    del ws


@pytest.mark.parametrize("R,masks", [(64, tree(64)), (21, tree(21)), (64, chain(64)), (7, chain(7))])
@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 2, 64), (10, 2, 128)])
def test_groups_and_masks(cuda_device, R, masks, Hq, Hkv, hd):
    """Groups of 3, 0 and 2 sequences, one that shares nothing, and two
    sequences of no group."""
    s = make([(3, 5), (0, 4), (2, 17), (1, 0)], [10, 0, 100, 31, 16, 64], R, Hq, Hkv, hd, masks, seed=R, alone=(40, 0))
    ws = call(s)
    verify(s)
    del ws


def test_long_prefix_few_rows(cuda_device):
    s = make([(3, 520)], [5, 300, 17], 1, 8, 2, 64, seed=1)
    ws = call(s)
    verify(s)
    s = make([(2, 300), (1, 257)], [5, 3000, 17], 4, 32, 8, 128, seed=1)
    ws2 = call(s)
    verify(s)
    del ws, ws2


def test_many_sequences(cuda_device):
    own = [(7 * b) % 130 for b in range(70)]
    s = make([(70, 33)], own, 5, 8, 2, 128, seed=1)
    ws = call(s)
    verify(s)
    del ws


def test_rows_that_see_little_or_nothing(cuda_device):
    """Masks of zero: with no context the row sees nothing and gives zeros,
    with context it sees that alone; groups whose members have no context."""
    masks = [0, 1, 0b10, 0b110, 0]
    s = make([(2, 0), (2, 1)], [0, 0, 0, 3], 5, 8, 2, 64, masks, seed=2)
    ws = call(s)
    verify(s)
    assert bool((s["out"][0, 0] == 0).all()) and bool((s["out"][1, 4] == 0).all())
    del ws


def test_shared_pages_past_a_members_context(cuda_device):
    """A group's announced pages are cut at its shortest context: nothing past
    a row's context is seen through the prefix."""
    s = make([(3, 6)], [0, 20, 40], 3, 8, 2, 64, seed=3)
    s["pages"][0] = 50  # more than any context holds
    ws = call(s)
    verify(s)
    s["ctx_host"][1] = 16 * 3 + 7
    s["ctx"][1] = 16 * 3 + 7
    call(s, ws)
    verify(s)
    s["ctx_host"][2] = 0
    s["ctx"][2] = 0
    call(s, ws)
    verify(s)
    s["pages"][0] = -4
    call(s, ws)
    verify(s)


def test_nan_of_unseen_new_rows(cuda_device):
    """A NaN value of one tree node reaches its descendants only."""
    R = 13
    s = make([(3, 4)], [9, 17, 0], R, 8, 2, 64, tree(R), seed=5)
    for b, node, val in ((0, 3, float("nan")), (1, 12, float("inf")), (2, 5, float("-inf"))):
        tok = s["ctx_host"][b] + node
        s["kv"][int(s["tables"][b, tok // 16]), 1, 1, tok % 16, 9] = val
    ws = call(s)
    verify(s)
    del ws


def test_streams_graphs_and_same_bits(cuda_device):
    a = make([(6, 40)], [5] * 6, 5, 32, 8, 128, seed=1)
    b = make([(2, 300), (2, 9)], [100, 5, 77, 900], 1, 8, 2, 64, seed=2)
    wa, wb = call(a), call(b)
    torch.cuda.synchronize()
    first = a["out"].clone(), b["out"].clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        call(a, wa, s1)
        call(b, wb, s2)
    torch.cuda.synchronize()
    assert torch.equal(first[0], a["out"]) and torch.equal(first[1], b["out"])
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        call(a, wa)
    with torch.cuda.graph(gb):
        call(b, wb)
    a["pages"][0] = 3  # less is shared than before: the same result
    a["out"].fill_(7.0)
    b["ctx"][3] = 9 * 16 + 33
    b["ctx_host"][3] = 9 * 16 + 33
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        ga.replay()
    with torch.cuda.stream(s2):
        gb.replay()
    verify(a)
    verify(b)


def test_agrees_with_the_verify_attention(cuda_device):
    s = make([(4, 12)], [3, 50, 16, 100], 6, 8, 2, 64, seed=8)
    s["kv"].nan_to_num_(nan=0.0)
    ws = call(s)
    verify(s)
    S.check(S.lib().specdec_attention(s["q"].data_ptr(), s["kv"].data_ptr(), s["nb"], 2, 64, s["tables"].data_ptr(),
                                      s["tables"].shape[1], s["ctx"].data_ptr(), s["mask"].data_ptr(), 4, 6, 8,
                                      s["out"].data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream))
    verify(s, "specdec_attention")
    del ws


def test_more_sequences_than_the_plan_keeps(cuda_device):
    own = [(11 * b) % 90 for b in range(300)]
    s = make([(120, 8), (3, 0), (150, 21), (1, 4)], own[:274], 3, 8, 2, 64, seed=4, alone=own[274:])
    ws = call(s)
    verify(s)
    s = make([(1024, 3)], [b % 40 for b in range(1024)], 1, 4, 4, 64, seed=4)
    ws2 = call(s)
    verify(s)
    del ws, ws2


def test_new_rows_without_slots(cuda_device):
    """A table that ends with the shared pages: the new rows' slots do not
    exist, the rows see the prefix alone (and zeros where there is none)."""
    s = make([(3, 6)], [0, 0, 0], 4, 8, 2, 64, seed=5, alone=(0,))
    s["tables"] = s["tables"][:, :6].contiguous()
    ws = call(s)
    verify(s)
    s["ctx_host"][3] = 6 * 16
    s["ctx"][3] = 6 * 16
    s["tables"][3] = s["tables"][0]
    call(s, ws)
    verify(s)


def test_no_groups(cuda_device):
    s = make([], [], 5, 8, 2, 64, seed=6, alone=(3, 40, 0, 700))
    s["goff"] = s["pages"] = torch.empty(0, dtype=torch.int32, device=DEV)  # null pointers
    assert s["goff"].data_ptr() == 0
    ws = call(s)
    verify(s)
    del ws


def test_groups_that_overlap_or_decrease_stay_in_bounds(cuda_device):
    """Bounds that no caller should give: the call ends, and memory around the
    workspace's and the output's is untouched."""
    s = make([(2, 4), (2, 4)], [30, 5, 9, 100], 2, 8, 2, 64, seed=7)
    need = S.lib().specdec_attention_shared_prefix_workspace_bytes(4, 2, 2, 8, 2, 64, s["tables"].shape[1])
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device=DEV)
    for off in ([0, 4, 0], [3, 1, 4], [-5, 9, 2], [4, 4, 4], [0, 1 << 30, -1]):
        s["goff"].copy_(torch.tensor(off))
        call(s, ws[:need])
        torch.cuda.synchronize()
        assert bool((ws[need:] == 0x5A).all())
    s["goff"].copy_(torch.tensor([0, 2, 4]))
    call(s, ws[:need])
    verify(s)


@pytest.mark.parametrize("name", ["tables", "ctx", "mask", "goff", "pages"])
def test_host_pointers_are_refused(cuda_device, name):
    s = make([(3, 4)], [5, 20, 40], 2, 8, 2, 64)
    with pytest.raises(S.SpecdecError) as e:
        call(dict(s, **{name: s[name].cpu()}))
    assert e.value.code == S.EINVAL and "device" in str(e.value)
    ws = call(s)
    verify(s)
    del ws


def test_misaligned_pointers_are_refused(cuda_device):
    s = make([(3, 4)], [5, 20, 40], 2, 8, 2, 64)
    ws = workspace(s)
    for at, step in ((5, 2), (7, 2), (8, 4), (9, 2), (10, 2)):  # tables, ctx_len, mask, group_off, shared_blocks
        args = [s["q"].data_ptr(), s["kv"].data_ptr(), s["nb"], s["Hkv"], s["hd"], s["tables"].data_ptr(),
                s["tables"].shape[1], s["ctx"].data_ptr(), s["mask"].data_ptr(), s["goff"].data_ptr(),
                s["pages"].data_ptr(), s["ng"], s["B"], s["R"], s["Hq"], s["out"].data_ptr(), ws.data_ptr(),
                ws.numel(), torch.cuda.current_stream().cuda_stream]
        args[at] += step
        with pytest.raises(S.SpecdecError) as e:
            S.check(S.lib().specdec_attention_shared_prefix(*args))
        assert e.value.code == S.EINVAL and "aligned" in str(e.value)
    call(s, ws)
    verify(s)
