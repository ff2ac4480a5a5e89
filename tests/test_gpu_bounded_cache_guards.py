"""The operators of a bounded cache with bounds, lengths, tables and requests that
no caller should give: everything that a call writes lies between guards."""
import pytest
import torch

import specdec as S
import test_gpu_accumulate_attention as A
import test_gpu_kv_evict as E
import test_gpu_qk_norm_rope as N
import test_gpu_window_attention as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MARGIN = 1 << 18  # bytes on each side


class Guarded:
    """Tensors in the middle of larger buffers."""

    def __init__(self):
        self.all = []

    def like(self, t):
        size = t.numel() * t.element_size()
        whole = torch.full((2 * MARGIN + (size + 255) // 256 * 256,), 0xA5, dtype=torch.uint8, device=DEV)
        mine = whole[MARGIN:MARGIN + size].view(t.dtype).view(t.shape)
        mine.copy_(t)
        self.all.append((whole, size))
        return mine

    def check(self, what):
        torch.cuda.synchronize()
        for i, (whole, size) in enumerate(self.all):
            assert bool((whole[:MARGIN] == 0xA5).all()) and bool((whole[MARGIN + size:] == 0xA5).all()), f"{what}: buffer {i}"


# one launch; pieces of runs; ranges; divided between short sequences and long ones; packed rows alone
SHAPES = [([(3, 50), (2, 30), (1, 80)], 9), ([(3, 50), (2, 30), (1, 80)], 300), ([(3, 50), (2, 30), (1, 80)], 90000),
          ([(3, 50), (20, 30), (1, 80)], 9), ([(3, 50), (20, 30), (1, 80)], 300), ([(30, 50), (40, 30), (10, 80)], 9),
          ([(30, 50), (40, 30), (10, 80)], 300)]


def contexts():
    return [-5, 1 << 30, 80], [(1 << 31) - 1, 0, -(1 << 31)], [50, 30, 80]


def bounds(T):
    return [0, 3, T - 1, T], [0, T, 5, T], [-9, 7, 7, 1 << 30], [T] * 4, [9, 6, 3, 0], [0, 1 << 30, -3, T]


def set_to(t, values):
    t.copy_(torch.tensor(values, dtype=torch.int64).int())


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("lens,wide", SHAPES)
def test_attention(cuda_device, weigh, lens, wide):
    M = A if weigh else W
    s = A.make(lens, 8, 2, 64, seed=4, wide=wide) if weigh else W.make(lens, 8, 2, 64, 20, 4, seed=4, wide=wide)
    s["kv"] = torch.nan_to_num(s["kv"], nan=0.5)
    g = Guarded()
    for name in ("out", "kv") + (("weights",) if weigh else ()):
        s[name] = g.like(s[name])
    ws = g.like(M.workspace(s))
    pool = s["kv"].clone()
    for ctx in contexts():
        for off in bounds(s["T"]):
            set_to(s["ctx"], ctx)
            set_to(s["off"], off)
            M.call(s, ws)
            g.check(f"{ctx} {off}")
    # table entries of any value
    set_to(s["ctx"], [c for _, c in lens])
    set_to(s["off"], [0, lens[0][0], lens[0][0] + lens[1][0], s["T"]])
    s["tables"].copy_(torch.randint(-(1 << 31), (1 << 31) - 1, s["tables"].shape, device=DEV))
    M.call(s, ws)
    g.check("tables")
    assert torch.equal(pool, s["kv"])


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lens", [[(9, 4), (2, 30), (7, 3)], [(900, 4), (700, 30), (800, 3)]])
def test_write(cuda_device, half, lens):
    s = N.make(lens, 8, 2, 64, half, seed=8)
    g = Guarded()
    s["q"], s["kv"] = g.like(s["q"]), g.like(s["kv"])
    for ctx in contexts():
        for off in bounds(s["T"]):
            set_to(s["ctx"], ctx)
            set_to(s["off"], off)
            N.call(s)
            g.check(f"{ctx} {off}")
    set_to(s["ctx"], [4, 30, 3])
    set_to(s["off"], [0, lens[0][0], lens[0][0] + lens[1][0], s["T"]])
    set_to(s["pos"], torch.randint(-(1 << 31), (1 << 31) - 1, s["pos"].shape).tolist())
    s["tables"].copy_(torch.randint(-(1 << 31), (1 << 31) - 1, s["tables"].shape, device=DEV))
    N.call(s)
    g.check("tables and positions")


@pytest.mark.parametrize("n", [1, 4, 9])
def test_eviction(cuda_device, n):
    """Requests in order, and with one out of order: nothing but what the call names is written."""
    lens = [100, 250, -1, 90, 300, 31, 17, 220, 64, 280]
    for wrong in (None, "id", "length", "blocks", "entry"):
        st = E.State(lens, 20, 8, seed=n, shared=[(1, 0, 4)])
        reqs = [1, 0, 4, 3, 5, 6, 7, 8, 9][:n]
        if wrong == "id":
            reqs[-1] = (1 << 31) - 1
        elif wrong == "length":
            st.lens[reqs[-1]] = (1 << 31) - 1
        elif wrong == "blocks":
            st.nblk[reqs[-1]] = (1 << 31) - 1
        elif wrong == "entry":
            st.t[reqs[-1]][0] = -(1 << 31)
        st.gpu()
        g = Guarded()
        for name in ("t", "nblk", "lens", "ref", "w", "pool", "status"):
            st.d[name] = g.like(st.d[name])
        kept = g.like(torch.full((n, 60), -5, dtype=torch.int32, device=DEV))
        ws = g.like(st.workspace(n, 60))
        torch.cuda.synchronize()
        st.call(reqs, 60, 4, 8, want_kept=kept, ws=ws)
        status, want = E.plain_evict(st.t, st.nblk, st.lens, st.ref, st.w, st.pool, reqs, 60, 4, 8)
        assert status == (S.OK if wrong is None else S.EINVAL)
        st.same(status, want, kept if wrong is None else None)
        g.check(str(wrong))
