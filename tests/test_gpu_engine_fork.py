"""Engine.fork beyond a fresh admission: request ids and prefix references,
branches of a running generation, of a prompt that is not complete, and of a
tree engine."""
import numpy as np
import pytest

import oracle as O
import specdec as S
from helpers import steps_match_oracle

pytestmark = pytest.mark.gpu
TINY = S.MODEL_SHAPES["tiny"]
V, H = TINY["vocab"], TINY["hidden"]


def engine(B=4, **kw):
    kw = dict(dict(draft_len=3, max_ctx=256, temperature=0.0, seed=7), **kw)
    eng = S.Engine(TINY, batch=B, **kw)
    eng.init_weights(0)
    return eng


def slots(eng):
    """Tables, lengths, reference counts, pending tokens and draft states."""
    B, mb, nb = eng.batch, eng.info("max_blocks"), eng.info("num_blocks")
    return [eng.read("tables", np.int32, (B, mb)).copy(), eng.read("lens", np.int32, (B,)).copy(),
            eng.read("refcounts", np.int32, (nb,)).copy(), eng.read("pending", np.int32, (B,)).copy(),
            eng.read("h0", np.float32, (B, H)).copy()]


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


def test_request_ids_are_one_request_each(cuda_device):
    """An id that the source, another slot or another copy has is refused and
    changes nothing; the source's prefix references outlive the copies'."""
    rng = np.random.default_rng(1)
    eng, cache = engine(), S.RadixKVCache()
    prompts = [rng.integers(0, V, 70 + b).astype(np.int32) for b in range(4)]
    for b, p in enumerate(prompts):
        eng.admit(b, 10 + b, p, cache)
    before, index = slots(eng), cache.stats()
    for new, ids in (([1], [10]), ([1, 2], [20, 20]), ([1, 2], [20, 13]), ([1], [12])):
        with pytest.raises(S.SpecdecError) as err:
            eng.fork(0, new, ids, cache)
        assert err.value.code == S.EINVAL and "request id" in str(err.value)
        assert same(before, slots(eng)) and cache.stats() == index
    eng.fork(0, [1, 2], [20, -1], cache)
    eng.fork(0, [2, 3], [12, 11], cache)  # ids that no other slot holds any more
    for b in (1, 2, 3):
        eng.retire(b, cache)
    assert cache.match_prefix(prompts[0][:69])[0] == 69  # still the source's
    eng.admit(2, 30, prompts[0], cache)
    tab = eng.read("tables", np.int32, (4, eng.info("max_blocks")))
    assert tab[2, :4].tolist() == tab[0, :4].tolist()
    eng.close()
    cache.close()


def kv_rows(eng, b, n):
    """K/V of the first n tokens of slot b, raw bits."""
    shape = (TINY["layers"], eng.info("num_blocks"), 2, TINY["n_kv_heads"], 16, TINY["head_dim"])
    pool = eng.read("kv", np.uint16, shape)
    tab = eng.read("tables", np.int32, (eng.batch, eng.info("max_blocks")))[b]
    t = np.arange(n)
    return pool[:, tab[t // 16], :, :, t % 16, :]


def fork(eng, src, copies):
    """Forks; the copies have the same tokens, states and K/V, whole blocks are
    shared and the one in use is not."""
    held = slots(eng)[2]
    eng.fork(src, copies)
    tab, lens, refs, pend, h0 = slots(eng)
    n = int(lens[src])
    rows = kv_rows(eng, src, n)
    for b in copies:
        assert lens[b] == n and pend[b] == pend[src] and np.array_equal(h0[b], h0[src])
        assert np.array_equal(kv_rows(eng, b, n), rows)
        assert tab[b, :n // 16].tolist() == tab[src, :n // 16].tolist()
        assert n % 16 == 0 or tab[b, n // 16] != tab[src, n // 16]
    assert all(refs[p] == held[p] + len(copies) for p in tab[src, :n // 16])


def test_a_running_generation_branches(cuda_device):
    """After some steps, with copies of copies; the next steps against the oracle."""
    B, k, T, seed = 4, 3, 1.0, 11
    cfg = dict(TINY, block_size=16, rms_eps=1e-5, rope_theta=10000.0)
    rng = np.random.default_rng(2)
    eng = engine(B, temperature=T, seed=seed)
    for b in range(B):
        eng.admit(b, b, rng.integers(0, V, 40 + 17 * b).astype(np.int32))
    for _ in range(3):
        eng.step_host()
    fork(eng, 2, [0, 3])
    model = O.OracleModel(cfg, seed=0, rope_max_pos=256 + 80)
    steps_match_oracle(eng, model, TINY, B, k, T, seed, steps=2)
    fork(eng, 3, [1])  # a copy, which has gone its own way
    steps_match_oracle(eng, model, TINY, B, k, T, seed, steps=2)
    model.close()
    eng.close()


def test_a_prompt_branches_before_it_is_complete(cuda_device):
    """The copies of a slot in the middle of its prompt take their own rest, and
    end as slots that were given the whole prompts."""
    rng = np.random.default_rng(3)
    head = rng.integers(0, V, 128)
    prompts = [np.concatenate([head, rng.integers(0, V, n)]).astype(np.int32) for n in (9, 40, 70)]
    ref, eng = engine(3, use_graph=True), engine(3, use_graph=True)
    for b, p in enumerate(prompts):
        ref.admit(b, b, p)
    eng.set_active([0, 0, 0])
    for c in (head[:64], head[64:]):
        eng.prefill_chunk(0, c.astype(np.int32), final=False, request_id=0)
    eng.fork(0, [1, 2], [1, 2])
    for b in (2, 0, 1):
        rest = prompts[b][128:]
        if rest.size > 64:
            eng.prefill_chunk(b, rest[:64], final=False, request_id=b)
            rest = rest[64:]
        eng.prefill_chunk(b, rest, final=True, request_id=b)
    eng.set_active([1, 1, 1])
    for _ in range(3):
        for b, p in enumerate(prompts):
            n = int(ref.read("lens", np.int32, (3,))[b])
            assert np.array_equal(kv_rows(eng, b, n), kv_rows(ref, b, n))
        assert all(np.array_equal(x, y) for x, y in zip(slots(eng)[3:] + slots(eng)[1:2], slots(ref)[3:] + slots(ref)[1:2]))
        (acc, out), (acc_r, out_r) = eng.step_host(), ref.step_host()
        assert acc.tolist() == acc_r.tolist() and out.tolist() == out_r.tolist()
    eng.close()
    ref.close()


def test_a_tree_engine_branches(cuda_device):
    eng = engine(3, draft_len=0, tree_branching=[4, 4, 2, 2], tree_nodes=64, max_ctx=512)
    eng.seed_state(np.array([120, 77, 31], np.int32), 5)
    eng.step_host()
    fork(eng, 1, [2, 0])
    for _ in range(4):
        acc, out = eng.step_host()
        assert acc[0] == acc[1] == acc[2] and out[0].tolist() == out[1].tolist() == out[2].tolist()
    assert same([x[0] for x in slots(eng)[1:2] + slots(eng)[3:]], [x[2] for x in slots(eng)[1:2] + slots(eng)[3:]])
    eng.close()
