"""Forks of the paged cache: specdec_kv_fork_pages and specdec_kv_fork against
a plain restatement, the engine's fork, and the attention over what forks
make."""
import numpy as np
import pytest
import torch

import oracle as O
import specdec as S
from attn_plain import close, rows_plain
from helpers import steps_match_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TINY = S.MODEL_SHAPES["tiny"]
CFG = dict(TINY, block_size=16, rms_eps=1e-5, rope_theta=10000.0)


def plain_fork(tables, nblk, lens, ref, src, dst, pool):
    """The definition; returns the status and changes its arguments on OK only."""
    R, nb = tables.shape[0], ref.size
    if any(not (0 <= x < R) for x in list(src) + list(dst)) or len(set(dst)) < len(dst) or set(src) & set(dst):
        return S.EINVAL
    for s in src:
        use = -(-int(lens[s]) // 16)
        if nblk[s] < 0 or lens[s] < 0 or use > nblk[s] or any(not (0 <= p < nb) for p in tables[s, :use]):
            return S.EINVAL
    r = ref.copy()
    for d in dst:
        for p in tables[d, :max(0, nblk[d])]:
            if 0 <= p < nb:
                r[p] -= 1
    free = [p for p in range(nb) if r[p] == 0]
    if len(free) < sum(int(lens[s]) % 16 > 0 for s in src):
        return S.ENOMEM
    for s, d in zip(src, dst):
        row = [int(p) for p in tables[s, :lens[s] // 16]]
        for p in row:
            r[p] += 1
        part = int(lens[s]) % 16
        if part:
            p = free.pop(0)
            r[p] = 1
            pool[:, p, :, :, :part] = pool[:, tables[s, len(row)], :, :, :part]
            row.append(p)
        tables[d] = row + [-1] * (tables.shape[1] - len(row))
        nblk[d], lens[d] = len(row), lens[s]
    ref[:] = r
    return S.OK


def make(lens, slots, num_blocks, max_blocks, layers=3, Hkv=2, hd=64, seed=0):
    """lens: tokens of the slots that have a table, by slot."""
    rng = np.random.default_rng(seed)
    order = list(rng.permutation(num_blocks))
    tables = np.full((slots, max_blocks), -1, np.int32)
    nblk, ln, ref = np.full(slots, -1, np.int32), np.zeros(slots, np.int32), np.zeros(num_blocks, np.int32)
    for s, n in lens.items():
        need = -(-n // 16)
        tables[s, :need] = [order.pop() for _ in range(need)]
        ref[tables[s, :need]] = 1
        nblk[s], ln[s] = need, n
    pool = rng.standard_normal((layers, num_blocks, 2, Hkv, 16, hd)).astype(np.float16)
    return tables, nblk, ln, ref, pool


class OnGpu:
    def __init__(self, tables, nblk, lens, ref, pool, extra_stride=0):
        self.t = [torch.from_numpy(x.copy()).to(DEV) for x in (tables, nblk, lens, ref)]
        L = pool.shape[0]
        per = pool[0].size
        self.buf = torch.full((L, per + extra_stride), 3.0, dtype=torch.float16, device=DEV)
        self.buf[:, :per] = torch.from_numpy(pool.reshape(L, -1)).to(DEV)
        self.per, self.shape = per, pool.shape
        self.status = torch.full((1,), 99, dtype=torch.int32, device=DEV)

    def fork(self, src, dst, ws=None, pool=True):
        t, L = self.t, S.lib()
        n = len(src)
        self.ids = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (list(src) or [0], list(dst) or [0])]
        need = L.specdec_kv_fork_pages_workspace_bytes(t[3].numel(), t[0].shape[0], n)
        self.ws = torch.full((need,), 0xEE, dtype=torch.uint8, device=DEV) if ws is None else ws
        S.check(L.specdec_kv_fork_pages(
            t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), t[3].data_ptr(), t[3].numel(), t[0].shape[0],
            t[0].shape[1], self.ids[0].data_ptr(), self.ids[1].data_ptr(), n, self.buf.data_ptr() if pool else None,
            self.shape[0] if pool else 0, self.buf.stride(0), self.shape[3], self.shape[5], self.status.data_ptr(),
            self.ws.data_ptr(), self.ws.numel(), torch.cuda.current_stream().cuda_stream))

    def same(self, tables, nblk, lens, ref, pool, status):
        torch.cuda.synchronize()
        assert int(self.status) == status
        for got, ref_ in zip(self.t, (tables, nblk, lens, ref)):
            assert (got.cpu().numpy() == ref_).all()
        got = self.buf[:, :self.per].cpu().numpy().reshape(self.shape)
        assert (got.view(np.uint16) == pool.view(np.uint16)).all()
        assert bool((self.buf[:, self.per:] == 3.0).all())


CASES = [
    (dict(lens={0: 5}, slots=2, num_blocks=2, max_blocks=1), [0], [1]),
    (dict(lens={0: 16}, slots=3, num_blocks=1, max_blocks=2), [0, 0], [1, 2]),
    (dict(lens={0: 0, 1: 1}, slots=4, num_blocks=3, max_blocks=2), [0, 1], [2, 3]),
    (dict(lens={2: 205, 0: 33, 5: 48}, slots=8, num_blocks=40, max_blocks=13), [2, 2, 0, 5], [7, 1, 5 + 1, 3]),
    # targets that hold blocks (released first, and handed out again: none are free otherwise)
    (dict(lens={0: 31, 1: 40, 2: 7, 3: 100}, slots=4, num_blocks=2 + 3 + 1 + 7, max_blocks=7), [0, 0], [1, 3]),
    (dict(lens={0: 17, 1: 16}, slots=3, num_blocks=3, max_blocks=4), [0], [1]),
    # not enough blocks; a source without a table; ids out of range; a target twice; a target that is a source
    (dict(lens={0: 17}, slots=4, num_blocks=3, max_blocks=4), [0, 0], [1, 2]),
    (dict(lens={0: 17}, slots=4, num_blocks=8, max_blocks=4), [0, 3], [1, 2]),
    (dict(lens={0: 17}, slots=4, num_blocks=8, max_blocks=4), [0, 4], [1, 2]),
    (dict(lens={0: 17}, slots=4, num_blocks=8, max_blocks=4), [0, 0], [1, -1]),
    (dict(lens={0: 17}, slots=4, num_blocks=8, max_blocks=4), [0, 0], [1, 1]),
    (dict(lens={0: 17, 1: 3}, slots=4, num_blocks=8, max_blocks=4), [0, 1], [1, 2]),
]


@pytest.mark.parametrize("state,src,dst", CASES)
def test_against_the_definition(cuda_device, state, src, dst):
    st = make(**state)
    g = OnGpu(*st, extra_stride=64)
    status = plain_fork(*st[:4], src, dst, st[4])
    g.fork(src, dst)
    g.same(*st, status)


@pytest.mark.parametrize("seed", range(6))
def test_random_rounds(cuda_device, seed):
    """Forks upon forks, shared blocks and refusals among them."""
    rng = np.random.default_rng(seed)
    slots = int(rng.integers(3, 90))
    lens = {i: int(rng.integers(0, 700)) for i in range(max(1, slots // 3))}
    need = sum(-(-n // 16) for n in lens.values())
    st = make(lens, slots, need + int(rng.integers(0, 2 * slots)), 44, hd=64 * int(rng.integers(1, 3)), seed=seed)
    g = OnGpu(*st)
    for _ in range(5):
        ids = rng.permutation(slots)
        have = [i for i in ids if st[1][i] >= 0]
        src = have[:max(1, len(have) // 2)]
        dst = [int(i) for i in ids if i not in src][:int(rng.integers(1, slots))]
        src = [int(rng.choice(src)) for _ in dst]
        status = plain_fork(*st[:4], src, dst, st[4])
        g.fork(src, dst)
        g.same(*st, status)


def test_many_blocks_and_copies(cuda_device):
    st = make({0: 4000, 1: 3333, 2: 15}, 600, 9000, 300, layers=2, seed=1)
    src, dst = [i % 3 for i in range(590)], list(range(599, 9, -1))
    g = OnGpu(*st)
    assert plain_fork(*st[:4], src, dst, st[4]) == S.OK
    g.fork(src, dst)
    g.same(*st, S.OK)


def test_captured_and_tables_only(cuda_device):
    st = make({0: 100, 1: 64}, 6, 30, 8)
    g = OnGpu(*st)
    g.fork([0, 1], [2, 3])
    assert plain_fork(*st[:4], [0, 1], [2, 3], st[4]) == S.OK
    g.same(*st, S.OK)
    graph = torch.cuda.CUDAGraph()
    ids = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 0], [4, 5])]
    ws = g.ws
    with torch.cuda.graph(graph):
        t = g.t
        S.check(S.lib().specdec_kv_fork_pages(
            t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), t[3].data_ptr(), 30, 6, 8, ids[0].data_ptr(),
            ids[1].data_ptr(), 2, g.buf.data_ptr(), 3, g.buf.stride(0), 2, 64, g.status.data_ptr(), ws.data_ptr(),
            ws.numel(), torch.cuda.current_stream().cuda_stream))
    for src, dst in (([0, 0], [4, 5]), ([2, 1], [4, 0]), ([1, 1], [5, 5])):
        ids[0].copy_(torch.tensor(src))
        ids[1].copy_(torch.tensor(dst))
        status = plain_fork(*st[:4], src, dst, st[4])
        graph.replay()
        g.same(*st, status)
    # without a pool the tables change alone; no copies at all is fine
    keep = st[4].copy()
    plain_fork(*st[:4], [1], [0], st[4])
    g.fork([1], [0], pool=False)
    g.same(*st[:4], keep, S.OK)
    g.fork([], [])
    g.same(*st[:4], keep, S.OK)


def test_manager(cuda_device):
    kv = S.PagedKVCache(20, 16, max_requests=6, max_blocks_per_request=8)
    kv.append_batch([0, 1, 4], [40, 16, 70])
    tabs, lens, refs = kv.read()
    kv.fork([0, 0, 1], [2, 4, 3])  # request 4 held five blocks
    t2, l2, r2 = kv.read()
    assert l2.tolist() == [40, 16, 40, 16, 40, 0]
    assert t2[2, :2].tolist() == t2[4, :2].tolist() == tabs[0, :2].tolist() and t2[3, :1].tolist() == tabs[1, :1].tolist()
    own = {int(t2[0, 2]), int(t2[2, 2]), int(t2[4, 2])}
    assert len(own) == 3 and all(int(r2[p]) == 1 for p in own)
    assert [int(r2[p]) for p in tabs[0, :2]] == [3, 3] and int(r2[tabs[1, 0]]) == 2
    # the manager goes on: a copy grows into its own block, then frees
    kv.append_batch([2], [9])
    assert kv.read()[1].tolist() == [40, 16, 49, 16, 40, 0]
    for r in (0, 1, 2, 3, 4):
        kv.free_request(r)
    assert int(kv.read()[2].sum()) == 0
    # refusals change nothing
    kv.append_batch([0], [100])
    before = kv.read()
    for src, new in (([0, 0], [1, 1]), ([0], [0]), ([5], [1]), ([0], [6]), ([-1], [1]), ([0, 1], [1, 2])):
        with pytest.raises(S.SpecdecError) as e:
            kv.fork(src, new)
        assert e.value.code == S.EINVAL
    kv.append_batch([1, 4], [8 * 16, 5 * 16])  # 7 + 8 + 5 blocks: none is free
    before = kv.read()
    with pytest.raises(S.SpecdecError) as e:
        kv.fork([0, 0], [2, 3])
    assert e.value.code == S.ENOMEM and "nothing was changed" in str(e.value)
    assert all((a == b).all() for a, b in zip(before, kv.read()))
    kv.close()


def test_forked_requests_attend_as_their_source(cuda_device):
    """One prompt by prompt attention, forked; the copies' rows by shared-prefix
    attention and by prompt attention, over the same pool."""
    Hq, Hkv, hd, n, copies = 8, 2, 64, 333, 5
    st = make({0: n}, copies + 1, 64, 24, layers=2, Hkv=Hkv, hd=hd, seed=3)
    g = OnGpu(*st)
    g.fork([0] * copies, list(range(1, copies + 1)))
    L = S.lib()
    tables, layer = g.t[0], 1
    kv = g.buf[layer].view(64, 2, Hkv, 16, hd)
    st_ = torch.cuda.current_stream().cuda_stream
    # each copy's next token goes into its own block: slot n
    q = (torch.randn((copies + 1, 1, Hq, hd), device=DEV) * 1.5).half()
    for b in range(copies + 1):
        kv[int(tables[b, n // 16]), :, :, n % 16] = torch.randn((2, Hkv, hd), device=DEV).half()
    B = copies + 1
    ctx = torch.full((B,), n, dtype=torch.int32, device=DEV)
    mask = torch.ones(1, dtype=torch.int64, device=DEV)
    goff = torch.tensor([0, B], dtype=torch.int32, device=DEV)
    pages = torch.tensor([n // 16], dtype=torch.int32, device=DEV)
    out = torch.empty((2, B, Hq, hd), dtype=torch.float16, device=DEV)
    wa = torch.empty(L.specdec_attention_shared_prefix_workspace_bytes(B, 1, 1, Hq, Hkv, hd, 24), dtype=torch.uint8,
                     device=DEV)
    wb = torch.empty(L.specdec_attention_prompt_workspace_bytes(B, B, Hq, Hkv, hd, 24), dtype=torch.uint8, device=DEV)
    S.check(L.specdec_attention_shared_prefix(q.data_ptr(), kv.data_ptr(), 64, Hkv, hd, tables.data_ptr(), 24,
                                              ctx.data_ptr(), mask.data_ptr(), goff.data_ptr(), pages.data_ptr(), 1, B,
                                              1, Hq, out[0].data_ptr(), wa.data_ptr(), wa.numel(), st_))
    off = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    S.check(L.specdec_attention_prompt(q.data_ptr(), Hq * hd, kv.data_ptr(), 64, Hkv, hd, tables.data_ptr(), 24,
                                       ctx.data_ptr(), off.data_ptr(), B, B, Hq, out[1].data_ptr(), Hq * hd,
                                       wb.data_ptr(), wb.numel(), st_))
    torch.cuda.synchronize()
    assert int(g.status) == S.OK
    seen = torch.ones((1, n + 1), dtype=torch.bool, device=DEV)
    for b in range(B):
        o, tol = rows_plain(q[b], kv, tables[b], seen)
        close(out[0, b:b + 1], o, tol, f"shared {b}")
        close(out[1, b:b + 1], o, tol, f"prompt {b}")


@pytest.mark.parametrize("T", [0.0, 1.0])
def test_engine_fork(cuda_device, T):
    """One admitted prompt forked into the other slots: same state, blocks
    shared but the one in use, steps in parity with the oracle, and greedy
    generation equal in all slots."""
    B, k, seed = 4, 3, 7
    V, H = TINY["vocab"], TINY["hidden"]
    rng = np.random.default_rng(5)
    eng = S.Engine(TINY, batch=B, draft_len=k, max_ctx=256, temperature=T, seed=seed)
    eng.init_weights(0)
    cache = S.RadixKVCache()
    prompt = rng.integers(0, V, 74).astype(np.int32)
    for b in range(B):  # the other slots hold requests of their own first
        eng.admit(b, 10 + b, prompt if b == 0 else rng.integers(0, V, 30 + b).astype(np.int32), cache)
    nodes = cache.stats()
    eng.fork(0, [3, 1, 2], [20, 21, 22], cache)
    assert cache.stats()[1] < nodes[1]  # their prefix references are gone
    mb, nb = eng.info("max_blocks"), eng.info("num_blocks")
    tab, lens = eng.read("tables", np.int32, (B, mb)), eng.read("lens", np.int32, (B,))
    assert lens.tolist() == [73] * B
    assert all(tab[b, :4].tolist() == tab[0, :4].tolist() for b in range(B)) and len(set(tab[:, 4].tolist())) == B
    refs = eng.read("refcounts", np.int32, (nb,))
    assert [int(refs[p]) for p in tab[0, :5]] == [4] * 4 + [1] and int((refs > 0).sum()) == 4 + B
    h0, pend = eng.read("h0", np.float32, (B, H)), eng.read("pending", np.int32, (B,))
    assert (h0 == h0[0]).all() and (pend == pend[0]).all()
    if T:
        model = O.OracleModel(CFG, seed=0, rope_max_pos=256 + 80)
        steps_match_oracle(eng, model, TINY, B, k, T, seed, steps=2)
        model.close()
    else:
        for _ in range(6):
            acc, out = eng.step_host()
            assert all(acc[b] == acc[0] and out[b].tolist() == out[0].tolist() for b in range(B))
    # refusals, and a slot without a request as the source
    for bad in ([0], [1, 1], [4], [-1]):
        with pytest.raises(S.SpecdecError):
            eng.fork(0, bad)
    eng.retire(2, cache)
    with pytest.raises(S.SpecdecError) as e:
        eng.fork(2, [1])
    assert e.value.code == S.EINVAL
    assert eng.read("lens", np.int32, (B,))[1] > 0  # slot 1 kept its request
    eng.close()
    cache.close()


def test_host_pointers_are_refused(cuda_device):
    g = OnGpu(*make({0: 20}, 3, 8, 4))
    g.fork([0], [1])
    g.buf, keep = g.buf.cpu(), g.buf
    with pytest.raises(S.SpecdecError) as e:
        g.fork([0], [2])
    assert e.value.code == S.EINVAL
    g.buf = keep
    g.fork([0], [2])
    torch.cuda.synchronize()
    assert int(g.status) == S.OK


def test_host_tables_are_refused(cuda_device):
    g = OnGpu(*make({0: 20}, 3, 8, 4))
    for i in range(4):
        g.t[i], keep = g.t[i].cpu(), g.t[i]
        with pytest.raises(S.SpecdecError) as e:
            g.fork([0], [1])
        assert e.value.code == S.EINVAL and "device" in str(e.value)
        g.t[i] = keep
    need = S.lib().specdec_kv_fork_pages_workspace_bytes(8, 3, 1)
    with pytest.raises(S.SpecdecError) as e:
        g.fork([0], [1], ws=torch.zeros(need, dtype=torch.uint8))
    assert e.value.code == S.EINVAL and "device" in str(e.value)
    g.fork([0], [2])
    torch.cuda.synchronize()
    assert int(g.status) == S.OK and int(g.t[2][2]) == 20


@pytest.mark.parametrize("state,src,dst", CASES)
def test_wide_tables(cuda_device, state, src, dst):
    """The same calls on tables that one CTA does not work on alone."""
    st = make(**dict(state, max_blocks=2500))
    g = OnGpu(*st)
    status = plain_fork(*st[:4], src, dst, st[4])
    g.fork(src, dst)
    g.same(*st, status)
