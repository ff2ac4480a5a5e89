"""specdec_kv_evict and PagedKVCache.evict_by_weight with the K/V that the tables
name: every bit of the pool against the plain statement, and the moves that are
left to a caller without a pool."""
import pytest
import torch

import specdec as S
from test_gpu_kv_evict import PAGE, plain_evict

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LAYERS, HKV, HD, WIDE, BLOCKS = 3, 2, 64, 20, 70


def make(seed):
    """A manager with four requests, the last a fork of the first; pool and weights; the same as lists."""
    kv = S.PagedKVCache(BLOCKS, PAGE, max_requests=5, max_blocks_per_request=WIDE)
    kv.append_batch([0, 1, 2], [250, 40, 180])
    kv.fork([0], [3])
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    # layers further apart than their blocks
    whole = torch.randn((LAYERS, BLOCKS + 1, 2, HKV, PAGE, HD), generator=g, device=DEV).half()
    w = torch.rand((5, HKV, WIDE * PAGE), generator=g, device=DEV)
    tabs, lens, refs = kv.read()
    plain = [tabs.tolist(), [int((r >= 0).sum()) for r in tabs], lens.tolist(), refs.tolist(), w.cpu().numpy().copy(),
             whole.cpu()[:, :BLOCKS]]
    torch.cuda.synchronize()
    return kv, whole, w, plain


def same(kv, w, plain):
    tabs, lens, refs = kv.read()
    assert tabs.tolist() == plain[0] and lens.tolist() == plain[2] and refs.tolist() == plain[3]
    assert (w.cpu().numpy() == plain[4]).all()


@pytest.mark.parametrize("reqs,keep,first,last", [([3, 2], 64, 4, 16), ([0], 100, 20, 5), ([1, 0, 2, 3], 70, 0, 0), ([2], 33, 16, 17)])
@pytest.mark.parametrize("side", [False, True])
def test_the_pool_moves_with_the_tables(cuda_device, reqs, keep, first, last, side):
    kv, whole, w, plain = make(keep)
    behind = whole[:, BLOCKS].clone()
    kept = torch.full((len(reqs), keep), -5, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if side else None
    kv.evict_by_weight(reqs, keep, first, last, w.data_ptr(), HKV, w.shape[2], kept.data_ptr(), pool=whole.data_ptr(),
                       layers=LAYERS, layer_stride=whole.stride(0), n_kv_heads=HKV, head_dim=HD,
                       stream=stream.cuda_stream if side else None)
    status, want = plain_evict(*plain, reqs, keep, first, last)
    assert status == S.OK and kept.tolist() == want
    same(kv, w, plain)
    assert torch.equal(whole[:, :BLOCKS].cpu().view(torch.int16), plain[5].view(torch.int16))
    assert torch.equal(whole[:, BLOCKS], behind)


def test_moves_by_the_list_and_the_former_tables(cuda_device):
    """Without a pool: what the list and a copy of the tables say is what the call with a pool does."""
    kv, whole, w, plain = make(9)
    reqs, keep = [3, 2, 0], 64
    before = kv.read()[0]
    kept = torch.full((len(reqs), keep), -5, dtype=torch.int32, device=DEV)
    kv.evict_by_weight(reqs, keep, 4, 16, w.data_ptr(), HKV, w.shape[2], kept.data_ptr())
    status, _ = plain_evict(*plain, reqs, keep, 4, 16)
    assert status == S.OK
    same(kv, w, plain)
    after = kv.read()[0]
    was = whole.clone()
    for i, a in enumerate(reqs):
        for j, k in enumerate(kept[i].tolist()):
            whole[:, int(after[a][j // PAGE]), :, :, j % PAGE] = was[:, int(before[a][k // PAGE]), :, :, k % PAGE]
    for a in reqs:  # the tokens of every request (of replaced pages the rest is nobody's)
        for j in range(keep):
            assert torch.equal(whole[:, int(after[a][j // PAGE]), :, :, j % PAGE].cpu(),
                               plain[5][:, plain[0][a][j // PAGE], :, :, j % PAGE])


def test_a_pool_that_does_not_fit_is_refused(cuda_device):
    kv, whole, w, plain = make(3)
    before = whole.clone()
    good = dict(pool=whole.data_ptr(), layers=LAYERS, layer_stride=whole.stride(0), n_kv_heads=HKV, head_dim=HD)
    host = whole.cpu()
    for bad, what in ((dict(pool=None), "kv_evict"), (dict(layers=-1), "kv_evict"), (dict(layer_stride=8), "kv_evict"),
                      (dict(n_kv_heads=0), "kv_evict"), (dict(head_dim=60), "kv_evict"),
                      (dict(pool=host.data_ptr()), "not memory of the current device")):
        with pytest.raises(S.SpecdecError, match=what) as e:
            kv.evict_by_weight([0, 2], 64, 4, 16, w.data_ptr(), HKV, w.shape[2], **dict(good, **bad))
        assert e.value.code == S.EINVAL
    same(kv, w, plain)
    other = S.PagedKVCache(8, 32, max_requests=2, max_blocks_per_request=4)  # blocks of another size
    other.append_batch([0], [100])
    with pytest.raises(S.SpecdecError, match="16 tokens"):
        other.evict_by_weight([0], 20, 1, 1, w.data_ptr(), HKV, w.shape[2], **good)
    torch.cuda.synchronize()
    assert torch.equal(whole, before)


def test_what_the_manager_did_before_is_seen_on_another_stream(cuda_device):
    """free_request does not wait: the blocks that it gives back are the only ones that the eviction can take."""
    for _ in range(20):
        kv = S.PagedKVCache(33, PAGE, max_requests=4, max_blocks_per_request=16)
        kv.append_batch([0, 1], [250, 256])
        kv.fork([0], [3])
        w = torch.rand((4, HKV, 256), device=DEV)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with pytest.raises(S.SpecdecError) as e:
            kv.evict_by_weight([3], 64, 4, 16, w.data_ptr(), HKV, 256, stream=stream.cuda_stream)
        assert e.value.code == S.ENOMEM
        torch.cuda._sleep(2_000_000)  # keeps the default stream busy for a millisecond
        kv.free_request(1)
        kv.evict_by_weight([3], 64, 4, 16, w.data_ptr(), HKV, 256, stream=stream.cuda_stream)
        assert int(kv.read()[1][3]) == 64
