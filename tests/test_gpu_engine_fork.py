"""Engine.fork beyond a fresh admission: request ids and prefix references."""
import numpy as np
import pytest

import specdec as S

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
