"""specdec_qk_norm_rope_kv against the definition in 64 bits.

Bound, element by element: the output's rounding, 2^-11 |y| (2^-25 where fp16 is
subnormal), and what 32 bits lose: a sum of hd squares is off by less than hd
2^-24 of itself and the root by half of that, eight further roundings of 2^-24
(square root and reciprocal 2^-22), so less than 2^-16 of |a c| + |b s| (of |y|
where nothing turns)."""
import math

import pytest
import torch

import specdec as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(lens, Hq, Hkv, hd, half=False, rot=None, seed=0, wide=0, spare_rows=0, pad=0, far=0, own_pos=True):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    off = [0]
    for n, _ in lens:
        off.append(off[-1] + n)
    T = off[-1] + spare_rows
    need = [(n + c + 15) // 16 for n, c in lens]
    width = max(1, max(need, default=1), wide)
    nb = sum(need) + 3
    order = torch.randperm(nb, generator=g, device=DEV).int()
    tables = torch.full((max(1, len(lens)), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        tables[b, :k] = order[at:at + k]
        at += k
    rot = hd if rot is None else rot
    x = torch.randn((max(1, T), (Hq + 2 * Hkv) * hd + pad), generator=g, device=DEV)
    x[:, 5::37] *= 6
    max_pos = max(1, far + max((n + c for n, c in lens), default=1))
    angle = torch.arange(max_pos, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
        -2.0 * torch.arange(max(1, rot // 2), device=DEV, dtype=torch.float64) / max(1, rot))
    pos = torch.randint(0, max_pos, (max(1, T),), generator=g, device=DEV, dtype=torch.int32) if own_pos else None
    return dict(lens=lens, Hq=Hq, Hkv=Hkv, hd=hd, T=T, rot=rot, nb=nb, tables=tables, max_pos=max_pos,
                x=x.half() if half else x, half=int(half), qn=1 + 0.3 * torch.randn(hd, generator=g, device=DEV),
                kn=1 + 0.3 * torch.randn(hd, generator=g, device=DEV), cos=angle.cos().float(), sin=angle.sin().float(),
                pos=pos, off=torch.tensor(off, dtype=torch.int32, device=DEV),
                ctx=torch.tensor([c for _, c in lens] or [0], dtype=torch.int32, device=DEV),
                kv=torch.full((nb, 2, Hkv, 16, hd), 3.0, dtype=torch.float16, device=DEV),
                q=torch.full((max(1, T), Hq, hd), 7.0, dtype=torch.float16, device=DEV), eps=1e-5)


def call(s, stream=None):
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    st = (stream or torch.cuda.current_stream()).cuda_stream
    S.check(S.lib().specdec_qk_norm_rope_kv(
        p(s["x"]), s["half"], s["x"].stride(0), p(s["qn"]), p(s["kn"]), s["eps"], p(s["cos"]), p(s["sin"]),
        s["max_pos"], s["rot"], p(s["pos"]), p(s["kv"]), s["nb"], s["Hkv"], s["hd"], p(s["tables"]),
        s["tables"].shape[1], p(s["ctx"]), p(s["off"]), len(s["lens"]), s["T"], s["Hq"], p(s["q"]), s["q"].stride(0), st))


def want(s):
    """(q, kv) in 64 bits with bounds, from a pool and an output that were filled with 3 and 7."""
    Hq, Hkv, hd, rot = s["Hq"], s["Hkv"], s["hd"], s["rot"]
    q = torch.full((s["q"].shape[0], Hq, hd), 7.0, dtype=torch.float64, device=DEV)
    kv = torch.full(s["kv"].shape, 3.0, dtype=torch.float64, device=DEV)
    tq, tkv = torch.zeros_like(q), torch.zeros_like(kv)
    for b, (n, c) in enumerate(s["lens"]):
        for i in range(n):
            r, slot = int(s["off"][b]) + i, c + i
            x = s["x"][r, :(Hq + 2 * Hkv) * hd].double().reshape(-1, hd)
            y, scale = x.clone(), x.abs()
            for lo, hi, w in ((0, Hq, s["qn"]), (Hq, Hq + Hkv, s["kn"])):
                if w is not None:
                    y[lo:hi] = x[lo:hi] / torch.sqrt((x[lo:hi] ** 2).mean(1, keepdim=True) + s["eps"]) * w.double()
            scale = y.abs()
            if rot:
                p = slot if s["pos"] is None else int(s["pos"][r])
                p = min(max(p, 0), s["max_pos"] - 1)
                co, si = s["cos"][p].double(), s["sin"][p].double()
                a, d = y[:Hq + Hkv, :rot // 2].clone(), y[:Hq + Hkv, rot // 2:rot].clone()
                y[:Hq + Hkv, :rot // 2], y[:Hq + Hkv, rot // 2:rot] = a * co - d * si, d * co + a * si
                scale[:Hq + Hkv, :rot // 2] = (a * co).abs() + (d * si).abs()
                scale[:Hq + Hkv, rot // 2:rot] = (d * co).abs() + (a * si).abs()
            tol = 2.0 ** -11 * y.abs() + 2.0 ** -16 * scale + 2.0 ** -25
            q[r], tq[r] = y[:Hq], tol[:Hq]
            page = int(s["tables"][b, slot // 16]) if slot < 16 * s["tables"].shape[1] else -1
            if 0 <= page < s["nb"]:
                kv[page, 0, :, slot % 16], tkv[page, 0, :, slot % 16] = y[Hq:Hq + Hkv], tol[Hq:Hq + Hkv]
                kv[page, 1, :, slot % 16], tkv[page, 1, :, slot % 16] = y[Hq + Hkv:], tol[Hq + Hkv:]
    return q, tq, kv, tkv


def verify(s):
    torch.cuda.synchronize()
    q, tq, kv, tkv = want(s)
    assert bool(((s["q"].double() - q).abs() <= tq).all()), "queries"
    assert bool(((s["kv"].double() - kv).abs() <= tkv).all()), "the pool (or a slot of no row was written)"


HEADS = [(8, 2, 64), (32, 8, 128), (40, 8, 128), (5, 1, 128), (3, 3, 64), (1, 1, 64), (64, 1, 128)]


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lens", [[(1, 0)], [(1, 40)], [(17, 15), (0, 3), (1, 127)], [(5, 2), (70, 0), (33, 31)]])
def test_lengths(cuda_device, Hq, Hkv, hd, half, lens):
    s = make(lens, Hq, Hkv, hd, half, seed=len(lens) + hd)
    call(s)
    verify(s)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rot", [0, 16, 32, 48, 64, 112])
def test_parts_of_a_head_that_turn(cuda_device, hd, rot):
    if rot > hd:
        rot -= 64
    s = make([(9, 4), (2, 30)], 6, 3, hd, rot=rot, seed=rot)
    if rot == 0:
        s["cos"] = s["sin"] = None
    call(s)
    verify(s)


@pytest.mark.parametrize("none", ["qn", "kn", "both"])
def test_without_norms(cuda_device, none):
    s = make([(9, 4), (2, 30)], 8, 2, 128, seed=3)
    for k in ("qn", "kn") if none == "both" else (none,):
        s[k] = None
    call(s)
    verify(s)


def test_positions_are_slots_by_default_and_stay_in_the_tables(cuda_device):
    s = make([(9, 4), (20, 100)], 8, 2, 64, seed=4, own_pos=False)
    call(s)
    verify(s)
    s = make([(9, 4), (20, 100)], 8, 2, 64, seed=5)
    s["pos"][3], s["pos"][7], s["pos"][11] = -9, 1 << 30, s["max_pos"]
    call(s)
    verify(s)


def test_strides_and_rows_of_no_sequence(cuda_device):
    """A wider projection, a wider output, rows in front of the first sequence's and behind the last one's."""
    s = make([(6, 4), (3, 100)], 8, 2, 64, seed=6, pad=24, spare_rows=5)
    s["off"] += 2
    s["T"] = 14
    big = torch.full((14, 10, 64), 7.0, dtype=torch.float16, device=DEV)
    s["q"] = big
    call(s)
    torch.cuda.synchronize()
    q, tq, kv, tkv = want(s)
    assert bool(((big[:, :8].double() - q).abs() <= tq).all()) and bool((big[:, 8:] == 7.0).all())
    assert bool((big[:2] == 7.0).all()) and bool((big[11:] == 7.0).all())
    assert bool(((s["kv"].double() - kv).abs() <= tkv).all())


def test_slots_without_a_page_write_nothing(cuda_device):
    """Entries outside the pool, and slots past the table's end: the queries are written all the same."""
    s = make([(20, 10), (5, 14), (9, 40)], 8, 2, 64, seed=7)
    s["tables"][0, 1], s["tables"][1, 1], s["tables"][2, 3] = s["nb"], -7, 1 << 30
    s["ctx"][2] = 58
    s["lens"] = [(20, 10), (5, 14), (9, 58)]
    call(s)
    verify(s)


def test_bounds_that_no_caller_should_give(cuda_device):
    """Negative contexts, bounds past the rows and out of order: nothing out of range is touched."""
    s = make([(9, 4), (2, 30), (7, 3)], 8, 2, 64, seed=8)
    guard = torch.full((4, 1 << 16), 5.0, dtype=torch.float16, device=DEV)
    s["ctx"][0], s["ctx"][1] = -3, 1 << 30
    for off in ([0, 100, 5, 18], [-4, 9, 11, 1 << 30], [18, 18, 18, 18], [3, 2, 1, 0]):
        s["off"].copy_(torch.tensor(off, dtype=torch.int32))
        call(s)
        torch.cuda.synchronize()
    assert bool((guard == 5.0).all())


def test_large_and_small_values(cuda_device):
    """Rows of zeros, of tiny and of large values; v past fp16's range becomes infinite as a rounding does."""
    s = make([(6, 0)], 4, 2, 128, seed=9)
    s["x"][0], s["x"][1] = 0.0, s["x"][1] * 1e-12
    s["x"][2] *= 1e12
    s["x"][2, 6 * 128:] = 1.0
    s["x"][3, 6 * 128] = 1e6
    call(s)
    torch.cuda.synchronize()
    page = int(s["tables"][0, 0])
    assert float(s["kv"][page, 1, 0, 3, 0]) == math.inf
    s["kv"][page, 1, 0, 3, 0] = 3.0
    q, tq, kv, tkv = want(s)
    kv[page, 1, 0, 3, 0] = 3.0
    assert bool(((s["q"].double() - q).abs() <= tq).all()) and bool(((s["kv"].double() - kv).abs() <= tkv).all())


def test_many_sequences(cuda_device):
    lens = [(i % 3, (7 * i) % 50) for i in range(1000)]
    s = make(lens, 2, 1, 64, seed=10)
    call(s)
    verify(s)


def test_streams_and_graphs(cuda_device):
    s = make([(3, 20), (1, 7)], 8, 2, 64, seed=11)
    call(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(s, side)
    # other rows and lengths in the same memory
    t = make([(1, 30), (2, 11)], 8, 2, 64, seed=12)
    s["x"][:3].copy_(t["x"][:3])
    s["off"].copy_(t["off"])
    s["ctx"].copy_(t["ctx"])
    s["lens"] = t["lens"]
    s["q"].fill_(7.0)
    s["kv"].fill_(3.0)
    s["tables"][:, 2:] = -1
    graph.replay()
    s["q"][3:] = 7.0
    verify(s)


def test_host_and_foreign_memory_is_refused(cuda_device):
    s = make([(3, 20)], 8, 2, 64, seed=13)
    call(s)
    for name in ("x", "qn", "kn", "cos", "sin", "pos", "kv", "tables", "ctx", "off", "q"):
        t = dict(s)
        t[name] = s[name].cpu()
        with pytest.raises(S.SpecdecError, match="not memory of the current device"):
            call(t)
    torch.cuda.synchronize()
