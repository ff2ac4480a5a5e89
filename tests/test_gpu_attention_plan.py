"""How the prompt and shared-prefix attention cut their key ranges, read from the
workspace: 256 bytes, then six int32 a sequence (pieces of the shared prefix,
first row, stride; pieces of the own range, first row, stride)."""
import pytest
import torch

import test_gpu_prompt_attention as P
import test_gpu_shared_prefix as X

pytestmark = pytest.mark.gpu


def pieces(ws, sequences):
    torch.cuda.synchronize()
    return ws[256:256 + 24 * sequences].view(torch.int32).view(sequences, 6)[:, [0, 3]].tolist()


@pytest.mark.parametrize("prompt", [2800, 2900])
def test_a_long_range_is_cut_beside_many_short_ones(cuda_device, prompt):
    """A token on 100,000 slots beside 250 sequences of 5 rows, in calls of less
    and of more than 4096 rows: one CTA would walk 782 key tiles for it."""
    lens = [(5, 600)] * 250 + [(prompt, 0), (1, 100000)]
    s = P.make(lens, 32, 8, 128, seed=2)
    ws = P.call(s)
    got = pieces(ws, len(lens))
    assert got[251][1] >= 16
    off = s["off"].tolist()
    for b in (0, 1, 249, 250, 251):
        P.close(s["out"][off[b]:off[b + 1]], *P.want(s, b), f"sequence {b}")
    del ws


@pytest.mark.parametrize("groups,R,own,alone", [
    ([(200, 30)], 21, 90, ()), ([(40, 12), (0, 3), (60, 5)], 64, 33, (70, 5)),  # more rows than there is room for duals
    ([(3, 4)], 5, 40, (90,)), ([], 5, 0, (3, 40, 0, 200)), ([], 64, 0, (150,) * 60), ([], 3, 0, (900, 5000) * 30)])
def test_shared_prefixes_in_the_room_there_is(cuda_device, groups, R, own, alone):
    """Calls of many rows, of short tables (16 pages at most) and of no groups."""
    n = sum(g for g, _ in groups)
    s = X.make(groups, [(own * b) % (own + 1) for b in range(n)], R, 8, 2, 64, seed=R + n, alone=alone)
    ws = X.call(s)
    X.verify(s)
    del ws


class Guarded:
    """A tensor with a pattern in front of it and behind."""
    N = 1 << 16

    def __init__(self, like):
        size = like.numel() * like.element_size()
        self.buf = torch.full((size + 2 * self.N,), 0x5A, dtype=torch.uint8, device=like.device)
        self.at = self.buf[self.N:self.N + size].view(like.dtype).view(like.shape)

    def check(self):
        end = self.buf.numel() - self.N
        assert bool((self.buf[:self.N] == 0x5A).all()) and bool((self.buf[end:] == 0x5A).all())


def timed(f):
    """Far below the two seconds after which a kernel's wait gives up."""
    e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    e[0].record()
    f()
    e[1].record()
    torch.cuda.synchronize()
    assert e[0].elapsed_time(e[1]) < 200.0


def test_group_bounds_that_no_caller_should_give(cuda_device):
    """The call ends in time and writes in its output and its workspace alone."""
    s = X.make([(2, 20), (3, 14)], [30, 5, 9, 700, 41], 2, 8, 2, 64, seed=7, alone=(333,))
    out, ws = Guarded(s["out"]), Guarded(X.workspace(s))
    s["out"] = out.at
    X.call(s, ws.at)
    for off in ([0, 6, 0], [3, 1, 4], [-5, 9, 2], [6, 6, 6], [0, 1 << 30, -1], [-(1 << 31), (1 << 31) - 1, 0], [5, 0, 6]):
        for pages in ([20, 14], [1 << 30, -1], [-(1 << 31), (1 << 31) - 1]):
            s["goff"].copy_(torch.tensor(off))
            s["pages"].copy_(torch.tensor(pages))
            timed(lambda: X.call(s, ws.at))
            out.check()
            ws.check()
    s["goff"].copy_(torch.tensor([0, 2, 5]))
    s["pages"].copy_(torch.tensor([20, 14]))
    X.call(s, ws.at)
    X.verify(s)


@pytest.mark.parametrize("spare", [0, 40])
def test_row_bounds_and_lengths_that_no_caller_should_give(cuda_device, spare):
    s = P.make([(3, 2000), (130, 7), (0, 0), (1, 300)], 8, 2, 64, seed=8, tail_rows=spare)
    good = s["off"].clone(), s["ctx"].clone()
    out, ws = Guarded(s["out"]), Guarded(P.workspace(s))
    s["out"] = out.at
    P.call(s, ws.at)
    big = (1 << 31) - 1
    for off in ([0, 134, 0, 134, 0], [134, 3, 2, 1, 0], [-5, 1 << 30, -1, 7, big], [-big - 1] * 5, [big] * 5,
                [0, big, -big, big, 134]):
        for ctx in ([2000, 7, 0, 300], [big, -1, -big - 1, 1 << 30], [1 << 30] * 4):
            s["off"].copy_(torch.tensor(off))
            s["ctx"].copy_(torch.tensor(ctx))
            timed(lambda: P.call(s, ws.at))
            out.check()
            ws.check()
    s["off"].copy_(good[0])
    s["ctx"].copy_(good[1])
    s["out"].fill_(7.0)
    P.call(s, ws.at)
    P.verify(s)
