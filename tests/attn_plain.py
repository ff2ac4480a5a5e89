"""64-bit attention over a paged pool, row by row from the definition, with a
bound on what fp16 kernels may be off (torch holds the tensors only).

Bound, element by element, with p the weights, A = sum p |v| / sum p:
  2^-11 |o|   the output's rounding to fp16;
  2^-11 A     each weight's rounding to fp16;
  2^-13 A     scores and exponents in fp32: a score of hd products with
              sum |q k| below 2^10 is off by less than hd 2^-24 2^10 / 8, the
              base-2 exponent's factor log2(e) / sqrt(hd) makes that less than
              2^-13 of a weight when the sums round at random (2^-16 at most
              measured products), and exp2 itself is off by 2^-22;
  2^-25 sum |v| over the visible slots: weights below 2^-14 are subnormal in
              fp16 (the row's largest weight is at least 1);
  2^-25       the output's own subnormal step.
"""
import math

import torch


def rows_plain(q, kv, table, seen):
    """q [n, Hq, hd], kv pool [nb, 2, Hkv, 16, hd], table: page of every 16 slots,
    seen [n, slots] bool -> (o, bound) [n, Hq, hd] float64.  Slots that a row
    does not see take no part, whatever they hold."""
    n, Hq, hd = q.shape
    Hkv = kv.shape[2]
    G = Hq // Hkv
    slots = seen.shape[1]
    o = torch.zeros((n, Hq, hd), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    if slots == 0 or n == 0:
        return o, tol + 2.0 ** -25
    pages = table[:(slots + 15) // 16].long()
    for h in range(Hkv):
        kp = kv[pages, :, h].double()
        k, v = kp[:, 0].reshape(-1, hd)[:slots], kp[:, 1].reshape(-1, hd)[:slots]
        for g in range(G):
            x = (q[:, h * G + g].double()[:, None, :] * k[None]).sum(-1) if n * slots * hd < 1 << 24 else \
                q[:, h * G + g].double() @ torch.where(seen.any(0)[:, None], k, 0.0).T
            x = torch.where(seen, x / math.sqrt(hd), -math.inf)
            top = x.amax(1, keepdim=True)
            p = torch.where(seen, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
            l = p.sum(1, keepdim=True)
            l = torch.where(l == 0, 1.0, l)
            fin = torch.isfinite(v)
            vz = torch.where(fin, v, 0.0)
            oo = p @ vz / l
            if not bool(fin.all()):  # infinities and NaN of the visible slots only
                for d in range(hd):
                    bad = ~fin[:, d]
                    if bool(bad.any()):
                        add = torch.where(seen[:, bad], v[bad, d][None], 0.0).sum(1)
                        oo[:, d] += add
            o[:, h * G + g] = oo
            A = p @ vz.abs() / l
            S = seen.double() @ vz.abs()
            tol[:, h * G + g] = 2.0 ** -11 * oo.abs().nan_to_num(posinf=0.0) + (2.0 ** -11 + 2.0 ** -13) * A + 2.0 ** -25 * S + 2.0 ** -25
    return o, tol


def close(got, o, tol, what=""):
    got = got.double()
    fin = torch.isfinite(o)
    assert bool((torch.isnan(got) == torch.isnan(o)).all()), f"{what}: NaN elsewhere"
    inf = ~fin & ~torch.isnan(o)
    assert bool((got[inf] == o[inf]).all()), f"{what}: infinities differ"
    over = ((got - o).abs() / tol)[fin]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst} of the bound"
