"""The operators of a bounded cache together, as a serving loop uses them: prompts
written (normed, rotated) and attended to, their weights added up, tokens evicted,
and decoding steps whose positions go on while their slots do not; against lists
of tokens in 64 bits."""
import math

import pytest
import torch

import specdec as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE, EPS = 16, 1e-6


class Loop:
    def __init__(self, Hq, Hkv, hd, B, wide, seed=0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.g, self.Hq, self.Hkv, self.hd, self.B, self.wide = g, Hq, Hkv, hd, B, wide
        self.pages = B * wide
        i32 = lambda *a: torch.zeros(a, dtype=torch.int32, device=DEV)  # noqa: E731
        self.tables = torch.randperm(self.pages, generator=g, device=DEV).int().reshape(B, wide)
        self.nblk, self.lens, self.ref = i32(B) + wide, i32(B), i32(self.pages) + 1
        self.kv = torch.full((self.pages, 2, Hkv, PAGE, hd), float("nan"), dtype=torch.float16, device=DEV)
        self.w = torch.zeros((B, Hkv, wide * PAGE), device=DEV)
        self.qn, self.kn = (1 + 0.2 * torch.randn(hd, generator=g, device=DEV) for _ in range(2))
        angle = torch.arange(4096, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
            -2.0 * torch.arange(hd // 2, device=DEV, dtype=torch.float64) / hd)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.pos = [0] * B                        # next position of each sequence
        self.tokens = [[] for _ in range(B)]      # (k, v, weight [Hkv]) of the tokens held, in order

    def forward(self, rows, window=None):
        """rows[b] new tokens of each sequence; returns the outputs, and what they should be with bounds."""
        L, Hq, Hkv, hd, B = S.lib(), self.Hq, self.Hkv, self.hd, self.B
        off = [0]
        for n in rows:
            off.append(off[-1] + n)
        T, st = off[-1], torch.cuda.current_stream().cuda_stream
        x = torch.randn((T, (Hq + 2 * Hkv) * hd), generator=self.g, device=DEV)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        o, pos = i32(off), i32([self.pos[b] + i for b in range(B) for i in range(rows[b])])
        q, out = (torch.zeros((T, Hq, hd), dtype=torch.float16, device=DEV) for _ in range(2))
        p = lambda t: t.data_ptr()  # noqa: E731
        S.check(L.specdec_qk_norm_rope_kv(p(x), 0, x.shape[1], p(self.qn), p(self.kn), EPS, p(self.cos), p(self.sin), 4096,
                                          hd, p(pos), p(self.kv), self.pages, Hkv, hd, p(self.tables), self.wide,
                                          p(self.lens), p(o), B, T, Hq, p(q), Hq * hd, st))
        head = (p(q), Hq * hd, p(self.kv), self.pages, Hkv, hd, p(self.tables), self.wide, p(self.lens), p(o), B, T, Hq)
        if window:
            n = L.specdec_attention_window_workspace_bytes(B, T, Hq, Hkv, hd, self.wide)
            ws = torch.empty(n, dtype=torch.uint8, device=DEV)
            S.check(L.specdec_attention_window(*head, *window, p(out), Hq * hd, p(ws), n, st))
        else:
            n = L.specdec_attention_accumulate_workspace_bytes(B, T, Hq, Hkv, hd, self.wide)
            ws = torch.empty(n, dtype=torch.uint8, device=DEV)
            S.check(L.specdec_attention_accumulate(*head, p(self.w), self.wide * PAGE, p(out), Hq * hd, p(ws), n, st))
        torch.cuda.synchronize()
        want = torch.zeros((T, Hq, hd), dtype=torch.float64, device=DEV)
        for b in range(B):
            for i in range(rows[b]):
                r = off[b] + i
                h = x[r].double().reshape(-1, hd)
                at = self.pos[b] + i
                co, si = self.cos[at].double(), self.sin[at].double()

                def turn(y, w):
                    y = y / torch.sqrt((y ** 2).mean(1, keepdim=True) + EPS) * w.double()
                    a, d = y[:, :hd // 2], y[:, hd // 2:]
                    return torch.cat([a * co - d * si, d * co + a * si], 1)
                self.tokens[b].append([turn(h[Hq:Hq + Hkv], self.kn), h[Hq + Hkv:], torch.zeros(Hkv, dtype=torch.float64, device=DEV)])
                slot = len(self.tokens[b]) - 1
                see = [j for j in range(slot + 1) if not window or j < window[1] or j > slot - window[0]]
                k = torch.stack([self.tokens[b][j][0] for j in see])
                v = torch.stack([self.tokens[b][j][1] for j in see])
                s = torch.einsum("hgd,khd->hgk", turn(h[:Hq], self.qn).reshape(Hkv, -1, hd), k) / math.sqrt(hd)
                w = torch.softmax(s, -1)
                want[r] = torch.einsum("hgk,khd->hgd", w, v).reshape(Hq, hd)
                if not window:
                    for n_, j in enumerate(see):
                        self.tokens[b][j][2] += w[:, :, n_].sum(1)
            self.pos[b] += rows[b]
        self.lens += i32(rows)
        # q, k and v are rounded to fp16: scores of rows of length sqrt(hd) (norms 1.8 at most) are off by less than 2^-10 of
        # |q| |k| / sqrt(hd) < 2^-10 * 3.3 sqrt(hd), a weight by 2^-10 * 3.3 * 11.4 < 2^-4.7 of itself; v and the output by 2^-11
        assert bool(((out.double() - want).abs() <= 2 * 2.0 ** -4.7 * 4.5).all())
        # and most of these errors are far smaller
        assert float((out.double() - want).square().mean().sqrt()) <= 2.0 ** -9
        return out

    def weights_agree(self):
        for b in range(self.B):
            n = len(self.tokens[b])
            w = torch.stack([t[2] for t in self.tokens[b]], 1)
            got = self.w[b, :, :n].double()
            assert bool(((got - w).abs() <= 2.0 ** -4.6 * w + 1e-6).all()), "a weight"
            assert bool((self.w[b, :, n:] == 0).all())

    def evict(self, reqs, keep, first, last):
        L, st = S.lib(), torch.cuda.current_stream().cuda_stream
        r = torch.tensor(reqs, dtype=torch.int32, device=DEV)
        kept = torch.zeros((len(reqs), keep), dtype=torch.int32, device=DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV) - 1
        n = L.specdec_kv_evict_pages_workspace_bytes(self.pages, self.B, self.wide, len(reqs), keep)
        ws = torch.empty(n, dtype=torch.uint8, device=DEV)
        p = lambda t: t.data_ptr()  # noqa: E731
        S.check(L.specdec_kv_evict_pages(p(self.tables), p(self.nblk), p(self.lens), p(self.ref), self.pages, self.B, self.wide,
                                         p(r), len(reqs), keep, first, last, p(self.w), self.Hkv, self.wide * PAGE,
                                         p(self.kv), 1, self.kv.numel(), self.Hkv, self.hd, p(kept), p(status), p(ws), n, st))
        torch.cuda.synchronize()
        assert int(status) == S.OK
        for b, row in zip(reqs, kept.tolist()):
            held = len(self.tokens[b])
            stay = [j for j in row if j >= 0]
            assert len(stay) == min(held, keep)
            if held > keep:
                assert stay[:first] == list(range(first)) and stay[keep - last:] == list(range(held - last, held))
                score = torch.stack([t[2].sum() for t in self.tokens[b]])
                gone = sorted(set(range(held)) - set(stay))
                others = [j for j in stay if first <= j < held - last]
                if others:  # by the weights in 64 bits, up to what fp16 inputs change of them
                    assert float(score[others].min()) >= float(score[gone].max()) * (1 - 2.0 ** -3.5)
            self.tokens[b] = [self.tokens[b][j] for j in stay]
        # pages were given back: the scheduler takes free ones again
        tables, ref = self.tables.tolist(), self.ref.tolist()
        for b in range(self.B):
            for d in range(self.wide):
                if tables[b][d] < 0:
                    tables[b][d] = ref.index(0)
                    ref[tables[b][d]] = 1
        self.tables.copy_(torch.tensor(tables, dtype=torch.int32))
        self.ref.copy_(torch.tensor(ref, dtype=torch.int32))
        self.nblk.fill_(self.wide)
        assert self.lens.tolist() == [len(t) for t in self.tokens]


@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 2, 64), (4, 1, 128)])
def test_prompts_eviction_and_steps(cuda_device, Hq, Hkv, hd):
    loop = Loop(Hq, Hkv, hd, 3, 12, seed=hd)
    loop.forward([70, 33, 5])                     # prompts
    loop.weights_agree()
    loop.evict([2, 0], 40, 4, 8)                  # the third holds fewer
    loop.forward([1, 1, 1])                       # positions go on, slots do not
    loop.forward([3, 2, 40])                      # verify rows, a prompt's next chunk
    loop.evict([0, 1, 2], 24, 2, 6)
    loop.weights_agree()
    for _ in range(3):
        loop.forward([1, 1, 1])
    loop.weights_agree()
    loop.forward([5, 1, 20], window=(16, 3))      # a layer that sees a window of the slots
    loop.forward([1, 0, 1], window=(10, 0))
