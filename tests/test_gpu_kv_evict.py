"""specdec_kv_evict_pages and specdec_kv_evict: tables, counts, weights, lists
and every bit of the pool against a plain statement."""
import ctypes as C
import random

import numpy as np
import pytest
import torch

import specdec as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 16


def plain_evict(t, nblk, lens, ref, weights, pool, reqs, keep, first, last):
    """On lists / float arrays, in place; returns (status, kept).  Nothing is changed unless the status is OK."""
    n, wide, pages = len(reqs), len(t[0]), len(ref)
    kept, new_rows, moves, was = [], {}, [], list(ref)
    ref2 = list(ref)
    free = [p for p in range(pages) if was[p] == 0]
    for i, a in enumerate(reqs):
        if not 0 <= a < len(t) or reqs.count(a) > 1 or not 0 <= nblk[a] <= wide or not 0 <= lens[a] <= nblk[a] * PAGE or lens[a] > weights.shape[2]:
            return S.EINVAL, None
        if any(not 0 <= p < pages for p in t[a][:nblk[a]]):
            return S.EINVAL, None
    short = False
    for a in reqs:
        L = lens[a]
        if L <= keep:
            kept.append(list(range(L)) + [-1] * (keep - L))
            continue
        score = weights[a].astype(np.float64).sum(0).astype(np.float32)
        rank = lambda j: (-np.inf if np.isnan(score[j]) else -score[j], 0 if np.isnan(score[j]) else 1, j)  # noqa: E731
        must = set(range(first)) | set(range(L - last, L))
        rest = sorted((j for j in range(L) if j not in must), key=rank)
        stay = sorted(must | set(rest[:keep - len(must)]))
        kept.append(stay)
        hole = next((j for j, k in enumerate(stay) if j != k), keep)
        row = t[a][:nblk[a]]
        new = row[:-(-keep // PAGE)]
        start = hole
        if hole < keep:
            for d in range(hole // PAGE, len(new)):
                if was[row[d]] > 1:
                    if not free:
                        short = True
                        continue
                    new[d] = free.pop(0)
                    ref2[row[d]] -= 1
                    ref2[new[d]] += 1
                    if d == hole // PAGE:
                        start = d * PAGE
        for d in range(len(new), nblk[a]):
            ref2[row[d]] -= 1
        new_rows[a] = new + [-1] * (wide - nblk[a] + nblk[a] - len(new))
        moves.append((a, row, new, stay, start))
    if short:
        return S.ENOMEM, kept
    for a, row, new, stay, start in moves:
        if pool is not None and start < keep:
            at, to = torch.tensor(stay[start:]), torch.arange(start, keep)
            row_t, new_t = torch.tensor(row), torch.tensor(new)
            pool[:, new_t[to // PAGE], :, :, to % PAGE] = pool[:, row_t[at // PAGE], :, :, at % PAGE]
        w = weights[a][:, stay].copy()
        weights[a] = 0
        weights[a][:, :keep] = w
        t[a] = t[a][:0] + new_rows[a]
        nblk[a], lens[a] = len(new), keep
    ref[:] = ref2
    return S.OK, kept


class State:
    def __init__(self, lens, wide, spare, heads=2, layers=2, Hkv=2, hd=64, shared=(), ldw=None, seed=0, extra_pages=0):
        """lens: tokens of each request, -1 without a table; shared: (request, source, pages) whose first pages are the source's."""
        g = torch.Generator().manual_seed(seed)
        need = [-(-max(n, 0) // PAGE) + (extra_pages if n >= 0 else 0) for n in lens]
        common = {a: (src, k) for a, src, k in shared}  # (sources come before)
        self.pages = sum(need) - sum(k for _, k in common.values()) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        self.t, self.ref = [], [0] * self.pages
        for a, k in enumerate(need):
            src, c = common.get(a, (0, 0))
            self.t.append((self.t[src][:c] if c else []) + order[:k - c] + [-1] * (wide - k))
            order = order[k - c:]
        self.nblk = [k if n >= 0 else -1 for n, k in zip(lens, need)]
        self.lens = [max(n, 0) for n in lens]
        for row, k in zip(self.t, self.nblk):
            for p in row[:max(k, 0)]:
                self.ref[p] += 1
        self.ldw = ldw or wide * PAGE
        self.w = (torch.randn((len(lens), heads, self.ldw), generator=g) * 2).exp().numpy().astype(np.float32)
        self.pool = torch.randn((layers, self.pages, 2, Hkv, PAGE, hd), generator=g).half() if layers else None
        self.layers, self.Hkv, self.hd, self.wide = layers, Hkv, hd, wide

    def gpu(self):
        i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        self.d = dict(t=i(self.t), nblk=i(self.nblk), lens=i(self.lens), ref=i(self.ref), w=torch.tensor(self.w, device=DEV),
                      pool=None if self.pool is None else self.pool.to(DEV), status=i([-1]))
        return self

    def workspace(self, n, keep):
        size = S.lib().specdec_kv_evict_pages_workspace_bytes(self.pages, len(self.t), self.wide, n, keep)
        return torch.full((size,), 0xFF, dtype=torch.uint8, device=DEV)

    def call(self, reqs, keep, first, last, want_kept=True, ws=None, stream=None, **over):
        d = dict(self.d, **over)
        r = reqs if isinstance(reqs, torch.Tensor) else torch.tensor(reqs, dtype=torch.int32, device=DEV)
        ws = self.workspace(r.numel(), keep) if ws is None else ws
        kept = torch.full((max(1, r.numel()), keep), -5, dtype=torch.int32, device=DEV) if want_kept is True else want_kept
        p = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        st = (stream or torch.cuda.current_stream()).cuda_stream
        S.check(S.lib().specdec_kv_evict_pages(
            p(d["t"]), p(d["nblk"]), p(d["lens"]), p(d["ref"]), self.pages, len(self.t), self.wide, p(r), r.numel(), keep,
            first, last, p(d["w"]), self.w.shape[1], self.ldw, p(d["pool"]), self.layers,
            d["pool"].stride(0) if self.layers else 0, self.Hkv, self.hd, p(kept), p(d["status"]), p(ws), ws.numel(), st))
        self.hold = (r, ws, kept)
        return kept

    def same(self, status, kept=None, got=None):
        torch.cuda.synchronize()
        d = self.d
        assert int(d["status"]) == status
        assert d["t"].tolist() == self.t and d["nblk"].tolist() == self.nblk and d["lens"].tolist() == self.lens
        assert d["ref"].tolist() == self.ref
        assert np.array_equal(d["w"].cpu().numpy(), self.w, equal_nan=True)
        if self.layers:
            assert torch.equal(d["pool"].cpu().view(torch.int16), self.pool.view(torch.int16))
        if kept is not None and got is not None:
            assert got.tolist() == kept

    def check(self, reqs, keep, first, last):
        self.gpu()
        got = self.call(reqs, keep, first, last)
        status, kept = plain_evict(self.t, self.nblk, self.lens, self.ref, self.w, self.pool, list(reqs), keep, first, last)
        self.same(status, kept if status == S.OK else None, got)
        return status


CASES = [
    (dict(lens=[100], wide=8, spare=2), [0], 40, 4, 8),
    (dict(lens=[100], wide=8, spare=0), [0], 1, 0, 0),
    (dict(lens=[100], wide=8, spare=0), [0], 99, 0, 0),
    (dict(lens=[100], wide=8, spare=0), [0], 100, 4, 8),
    (dict(lens=[100], wide=8, spare=0), [0], 5000, 4, 8),
    (dict(lens=[100], wide=8, spare=0), [0], 40, 40, 0),      # the first ones alone: nothing moves
    (dict(lens=[100], wide=8, spare=0), [0], 40, 0, 40),      # the last ones alone: all move
    (dict(lens=[100], wide=8, spare=0), [0], 40, 16, 24),     # first and last alone
    (dict(lens=[17, 0, 1, 33, 64, 65], wide=7, spare=1), [3, 0, 2, 1, 5, 4], 16, 1, 3),
    (dict(lens=[200, 50, -1, 300], wide=20, spare=3), [3, 0], 64, 4, 16),
    (dict(lens=[200, 50, -1, 300], wide=22, spare=3, extra_pages=2), [1, 3], 40, 4, 16),
    (dict(lens=[200, 180, 300], wide=20, spare=13, shared=[(1, 0, 5), (2, 0, 3)]), [0, 1, 2], 70, 4, 16),
    (dict(lens=[200, 180, 300], wide=20, spare=6, shared=[(1, 0, 5), (2, 0, 3)]), [2], 70, 20, 16),
    (dict(lens=[200, 180, 300], wide=20, spare=1, shared=[(1, 0, 5), (2, 0, 3)]), [2, 1], 70, 4, 16),  # no room
    (dict(lens=[3000], wide=200, spare=0, heads=8, hd=128, layers=3), [0], 1024, 16, 256),
    (dict(lens=[5000, 4097, 9000], wide=600, spare=0, heads=1, layers=1, Hkv=1), [2, 0], 4096, 0, 0),
    (dict(lens=[2500], wide=160, spare=0, heads=40, layers=0), [0], 700, 3, 5),
    (dict(lens=[130], wide=10, spare=0, layers=2, Hkv=3, hd=24), [0], 50, 1, 1),
    (dict(lens=[130], wide=10, spare=0, layers=1, Hkv=1, hd=1024), [0], 50, 1, 1),
]


@pytest.mark.parametrize("state,reqs,keep,first,last", CASES)
def test_against_the_definition(cuda_device, state, reqs, keep, first, last):
    st = State(**state)
    status = st.check(reqs, keep, first, last)
    assert status == (S.ENOMEM if state["spare"] == 1 and "shared" in state else S.OK)


@pytest.mark.parametrize("n", [8, 9, 40])
def test_many_requests(cuda_device, n):
    """Up to 8 requests are selected and given their tables in one launch, more in two."""
    r = random.Random(n)
    lens = [r.randrange(1, 300) for _ in range(n + 3)]
    shared = [(i, i - 1, min(lens[i], lens[i - 1]) // 16) for i in range(1, n + 3, 5)]
    st = State(lens, 20, 10 * n, seed=n, shared=shared, layers=1)
    reqs = list(range(n + 3))
    r.shuffle(reqs)
    assert st.check(reqs[:n], 60, 3, 7) == S.OK
    st.lens[reqs[0]] += 16 * 30  # one request out of order among the others
    assert st.check(reqs[:n], 20, 3, 7) == S.EINVAL


@pytest.mark.parametrize("slots", [2047, 2048, 2049, 4096, 4100, 8192, 8193])
def test_sizes_at_which_the_selection_changes(cuda_device, slots):
    """Threads by the table's width, keys in registers by the request's length; weights that are not aligned to 16 bytes."""
    wide = (slots + 15) // 16
    for ldw in (wide * 16, wide * 16 + 5):
        st = State([slots], wide, 0, heads=2, layers=1, Hkv=1, ldw=ldw, seed=slots)
        assert st.check([0], slots - 700, 11, 200) == S.OK
        assert st.check([0], 77, 0, 0) == S.OK


@pytest.mark.parametrize("seed", range(8))
def test_random_rounds(cuda_device, seed):
    """Rounds of growth and eviction on the same tables."""
    r = random.Random(seed)
    lens = [r.randrange(1, 400) for _ in range(6)]
    st = State(lens, 40, 150, seed=seed, shared=[(1, 0, min(lens[0], lens[1]) // 16)], heads=r.choice((1, 2, 8)))
    for _ in range(4):
        reqs = r.sample(range(6), r.randrange(1, 7))
        keep = r.randrange(1, 300)
        first = r.randrange(0, keep + 1)
        st.check(reqs, keep, first, r.randrange(0, keep - first + 1))
        for a in range(6):  # more tokens, in new pages
            grow = min(r.randrange(0, 200), 40 * PAGE - st.lens[a])
            st.lens[a] += grow
            while st.nblk[a] * PAGE < st.lens[a]:
                p = next(i for i, x in enumerate(st.ref) if x == 0)
                st.t[a][st.nblk[a]] = p
                st.ref[p] = 1
                st.nblk[a] += 1
            st.w[a, :, st.lens[a] - grow:st.lens[a]] = np.random.RandomState(seed).rand(st.w.shape[1], grow)


def test_equal_weights_zeros_and_nan(cuda_device):
    """Of equal weights the lower slots stay, -0 is 0, NaN is above infinity."""
    st = State([300], 20, 0, heads=3)
    st.w[:] = 1.0
    st.check([0], 100, 10, 10)
    st = State([300], 20, 0, heads=1)
    st.w[:] = 0.0
    st.w[0, 0, ::2] = -0.0
    st.w[0, 0, 50:60] = 2.0
    st.check([0], 100, 10, 10)
    st = State([300], 20, 0, heads=2)
    st.w[0, 0, 100:140] = np.inf
    st.w[0, 1, 130:200] = np.nan
    st.w[0, :, 250] = -np.inf
    st.w[0, 0, 20:60] *= -1
    st.check([0], 95, 2, 3)
    # weights that differ in the last of 32 bits
    st = State([3000], 200, 0, heads=1, layers=1)
    st.w[0, 0, :3000] = np.float32(1.0) + np.random.RandomState(1).randint(0, 50, 3000).astype(np.float32) * 2.0 ** -23
    st.check([0], 1500, 7, 9)


@pytest.mark.parametrize("what", ["id", "negative", "twice", "no table", "entry", "entry below", "length", "blocks", "ldw"])
def test_all_or_nothing(cuda_device, what):
    """One request out of order: nothing of the call happens."""
    st = State([100, 200, -1, 120], 14, 4)
    reqs = [3, 0, 1]
    if what == "id":
        reqs[1] = 4
    elif what == "negative":
        reqs[1] = -1
    elif what == "twice":
        reqs[1] = 3
    elif what == "no table":
        reqs[1] = 2
    elif what == "entry":
        st.t[0][2] = st.pages
    elif what == "entry below":
        st.t[0][6] = -1
    elif what == "length":
        st.lens[0] = 8 * 16
    elif what == "blocks":
        st.nblk[0] = 15
    elif what == "ldw":
        st = State([100, 200, -1, 120], 14, 4, ldw=150)
    assert st.check(reqs, 60, 4, 4) == S.EINVAL


def test_captured_tables_only_and_without_a_list(cuda_device):
    st = State([100, 250, 90], 20, 8, shared=[(1, 0, 4)]).gpu()
    reqs = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    ws = st.workspace(2, 60)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        st.call(reqs, 60, 4, 8, want_kept=None, ws=ws, stream=side)
    graph.replay()
    assert plain_evict(st.t, st.nblk, st.lens, st.ref, st.w, st.pool, [1, 0], 60, 4, 8)[0] == S.OK
    st.same(S.OK)
    graph.replay()  # nothing is left to evict
    st.same(S.OK)
    # other requests and lengths in the same memory
    reqs.copy_(torch.tensor([2, 0], dtype=torch.int32))
    graph.replay()
    assert plain_evict(st.t, st.nblk, st.lens, st.ref, st.w, st.pool, [2, 0], 60, 4, 8)[0] == S.OK
    st.same(S.OK)


def test_two_calls_at_once(cuda_device):
    """Two caches on two streams, with workspaces of their own."""
    a, b = State([900, 850], 60, 4, seed=1).gpu(), State([700, 900, 640], 60, 4, seed=2).gpu()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    ka = a.call([0, 1], 300, 4, 64, stream=one)
    kb = b.call([2, 0, 1], 200, 4, 64, stream=two)
    for st, reqs, keep, got in ((a, [0, 1], 300, ka), (b, [2, 0, 1], 200, kb)):
        status, kept = plain_evict(st.t, st.nblk, st.lens, st.ref, st.w, st.pool, reqs, keep, 4, 64)
        st.same(status, kept, got)


def test_no_requests(cuda_device):
    st = State([100], 8, 0).gpu()
    st.call(torch.zeros(0, dtype=torch.int32, device=DEV), 20, 0, 0, want_kept=None, ws=torch.empty(4096, dtype=torch.uint8, device=DEV))
    st.same(S.OK)


def test_pools_past_32_bits(cuda_device):
    """Pages whose offsets in the pool are past 2^32 elements."""
    pages = 66000  # 66000 * 2 * 16 * 16 * 128 halves
    pool = torch.empty((1, pages, 2, 16, PAGE, 128), dtype=torch.float16, device=DEV)
    st = State([100], 8, 0, layers=0, Hkv=16, hd=128, heads=2)
    st.pages, st.layers = pages, 1
    st.t[0][:7] = [65999, 3, 65000, 64998, 17, 65998, 64000]
    st.ref = [0] * pages
    for p in st.t[0][:7]:
        st.ref[p] = 1
    st.gpu()
    for p in st.t[0][:7]:
        pool[:, p] = torch.randn(pool[:, p].shape, device=DEV).half()
    was = {p: pool[:, p].cpu() for p in st.t[0][:7]}
    st.d["pool"] = pool
    row = list(st.t[0])
    st.call([0], 50, 2, 20)
    status, kept = plain_evict(st.t, st.nblk, st.lens, st.ref, st.w, None, [0], 50, 2, 20)
    torch.cuda.synchronize()
    assert int(st.d["status"]) == S.OK and st.d["t"].tolist() == st.t
    for j, k in enumerate(kept[0]):
        assert torch.equal(pool[:, row[j // 16], :, :, j % 16].cpu(), was[row[k // 16]][:, :, :, k % 16])


def test_manager(cuda_device):
    kv = S.PagedKVCache(40, PAGE, max_requests=4, max_blocks_per_request=12)
    kv.append_batch([0, 1, 2], [150, 40, 90])
    kv.fork([0], [3])
    ldw = 12 * PAGE
    w = torch.rand((4, 2, ldw), device=DEV)
    tabs, lens, refs = kv.read()
    t, nblk = tabs.tolist(), [int((row >= 0).sum()) for row in tabs]
    lens, refs, wp = lens.tolist(), refs.tolist(), w.cpu().numpy().copy()
    kept = torch.full((3, 64), -5, dtype=torch.int32, device=DEV)
    kv.evict_by_weight([3, 1, 0], 64, 4, 16, w.data_ptr(), 2, ldw, kept.data_ptr())
    status, want = plain_evict(t, nblk, lens, refs, wp, None, [3, 1, 0], 64, 4, 16)
    assert status == S.OK and kept.tolist() == want
    got_t, got_l, got_r = kv.read()
    assert got_t.tolist() == t and got_l.tolist() == lens and got_r.tolist() == refs
    assert np.array_equal(w.cpu().numpy(), wp)
    # the manager goes on with these tables
    kv.append_batch([3], [20])
    assert int(kv.read()[1][3]) == 84
    with pytest.raises(S.SpecdecError) as e:
        kv.evict_by_weight([0, 0], 10, 1, 1, w.data_ptr(), 2, ldw)
    assert e.value.code == S.EINVAL and "twice" in str(e.value)
    with pytest.raises(S.SpecdecError, match="not memory of the current device"):
        kv.evict_by_weight([0], 10, 1, 1, wp.ctypes.data, 2, ldw)
    kv.evict_by_weight([0], 5000, 1, 1, w.data_ptr(), 2, ldw)  # a larger keep than before
    small = S.PagedKVCache(9, PAGE, max_requests=2, max_blocks_per_request=8)
    small.append_batch([0], [120])
    small.fork([0], [1])
    before = [x.tolist() for x in small.read()]
    with pytest.raises(S.SpecdecError) as e:  # all of its pages have another holder, none is free
        small.evict_by_weight([0], 100, 0, 0, w.data_ptr(), 2, 128)
    assert e.value.code == S.ENOMEM and [x.tolist() for x in small.read()] == before


def test_host_memory_is_refused(cuda_device):
    st = State([100, 80], 8, 2).gpu()
    for name in ("t", "nblk", "lens", "ref", "w", "pool", "status"):
        with pytest.raises(S.SpecdecError, match="not memory of the current device"):
            st.call([0], 20, 1, 1, **{name: st.d[name].cpu()})
    with pytest.raises(S.SpecdecError, match="not memory of the current device"):
        st.call([0], 20, 1, 1, want_kept=torch.zeros((1, 20), dtype=torch.int32))
    with pytest.raises(S.SpecdecError, match="not memory of the current device"):
        st.call(torch.tensor([0], dtype=torch.int32), 20, 1, 1)
    torch.cuda.synchronize()
    st.d["status"].zero_()
    st.same(0)
    assert C.sizeof(C.c_int32) == 4
