"""Cases, plain forms and calls of three operators that serve a paged fp16 K/V cache:

  prompt   causal attention over packed sequences of different lengths, whose keys and values are in pages
  shared   attention of verify rows whose sequences begin with the same pages
  fork     requests that become copies of others: shared whole pages, a copy of the page in use, the old pages freed

`own = False` computes them with elementary torch operations in 32 bits; `own = True` calls the library.
A page holds 16 tokens of one layer as [K|V][kv head][16][head_dim]; a pool is [pages] of them.
"""
import math
import random

import torch

own = False

PAGE = 16
DEV = "cuda"


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one pending token of one short request: latency alone
        dict(name="prompt one token", op="prompt", heads=8, kv_heads=2, head_dim=64, batch=1, rows=1, cached=40, spread=0),
        # short questions of the small model, packed for one forward
        dict(name="prompt short, 4 packed", op="prompt", heads=8, kv_heads=2, head_dim=64, batch=4, rows=333, cached=0, spread=3),
        # one token a request, long ragged caches: the decode form
        dict(name="prompt 1 row x 64, cached 8k", op="prompt", heads=32, kv_heads=8, head_dim=128, batch=64, rows=1, cached=8192, spread=5),
        # the next chunk of prompts whose beginning is in the cache (40 query heads: 5 for each kv head)
        dict(name="prompt chunks 512 on 4k", op="prompt", heads=40, kv_heads=8, head_dim=128, batch=4, rows=512, cached=4096, spread=0),
        # packed prompts of very different lengths
        dict(name="prompt ragged, 8 packed", op="prompt", heads=32, kv_heads=8, head_dim=128, batch=8, rows=4001, cached=0, spread=11),
        # one long prompt from its first token: bound by the tensor cores
        dict(name="prompt 8192", op="prompt", heads=32, kv_heads=8, head_dim=128, batch=1, rows=8192, cached=0, spread=0),
        # single tokens of a few requests under one short system prompt
        dict(name="shared 4 x 1, 512", op="shared", heads=8, kv_heads=2, head_dim=64, batch=4, rows=1, groups=1, prefix=512, suffix=75, spread=2, tree=False),
        # chain verify rows of a batch under one system prompt
        dict(name="shared 32 x 5, 4k", op="shared", heads=32, kv_heads=8, head_dim=128, batch=32, rows=5, groups=1, prefix=4096, suffix=600, spread=4, tree=False),
        # draft trees, two system prompts
        dict(name="shared 16 x 21 tree, 2 of 2k", op="shared", heads=40, kv_heads=8, head_dim=128, batch=16, rows=21, groups=2, prefix=2048, suffix=999, spread=6, tree=True),
        # a large batch of chain verify rows under a long document
        dict(name="shared 128 x 5, 8k", op="shared", heads=32, kv_heads=8, head_dim=128, batch=128, rows=5, groups=1, prefix=8192, suffix=1024, spread=8, tree=False),
        # one prompt sampled four times, small model
        dict(name="fork 1 to 4", op="fork", layers=4, kv_heads=2, head_dim=64, slots=8, sources=1, copies=4, tokens=205, pages=256, spread=0),
        # a beam step: 16 survivors continue as 48 requests in all 32 layers
        dict(name="fork 16 to 48, 32 layers", op="fork", layers=32, kv_heads=8, head_dim=128, slots=64, sources=16, copies=3, tokens=1500, pages=1800, spread=9),
    ]


HEADS = ((8, 2, 64), (32, 8, 128), (40, 8, 128))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "shared", "shared", "fork"))
    heads, kv_heads, hd = rng.choice(HEADS)
    if op == "prompt":
        rows = _log(rng, 1, 6000)
        cached = rng.choice((0, _log(rng, 1, 8192)))
        # the padded plain form stays below the largest listed case
        most = max(1, min(64, int(32 * 8192 * 8192 / (heads * rows * (rows + cached))), 16384 // rows + 1))
        return dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=hd, batch=_log(rng, 1, most), rows=rows, cached=cached, spread=rng.randrange(1, 1000))
    if op == "shared":
        batch, rows = _log(rng, 1, 128), rng.choice((1, 4, 5, 8, 13, 21, 64))
        batch = min(batch, max(1, 640 // rows))
        return dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=hd, batch=batch, rows=rows, groups=min(batch, rng.choice((1, 1, 2, 3))), prefix=PAGE * _log(rng, 1, 512), suffix=_log(rng, 1, 1024), spread=rng.randrange(1, 1000), tree=rng.random() < 0.4)
    sources, copies = _log(rng, 1, 16), _log(rng, 1, 3)
    tokens = _log(rng, 5, 1500)
    slots = sources * (1 + copies) + rng.randrange(4)
    return dict(op=op, layers=rng.choice((2, 4, 32)), kv_heads=kv_heads, head_dim=hd, slots=slots, sources=sources, copies=copies, tokens=tokens, pages=slots * 2 + sources * (tokens // PAGE + 1) + 8, spread=rng.randrange(1, 1000))


def _ragged(r, most, spread):
    """A length up to `most`, spread over its logarithm."""
    return most if not spread else _log(r, max(1, most // 64), most)


def _prompt_lens(case):
    """(new rows, cached tokens) of each sequence; the first has the case's own."""
    r = random.Random(case["spread"])
    got = [(case["rows"], case["cached"])]
    for _ in range(case["batch"] - 1):
        got.append((_ragged(r, case["rows"], case["spread"]), _ragged(r, case["cached"], case["spread"]) if case["cached"] else 0))
    return got


def _shared_plan(case):
    """Group bounds over the batch, shared pages of each group, own tokens of each sequence."""
    r = random.Random(case["spread"])
    off = [case["batch"] * g // case["groups"] for g in range(case["groups"] + 1)]
    pages = [case["prefix"] // PAGE if g == 0 else max(1, case["prefix"] // PAGE - 3 * g) for g in range(case["groups"])]
    return off, pages, [_ragged(r, case["suffix"], case["spread"]) for _ in range(case["batch"])]


def _fork_plan(case):
    """Tokens of each slot (-1: no table), sources and targets."""
    r = random.Random(case["spread"])
    n, k = case["sources"], case["copies"]
    lens = [_ragged(r, case["tokens"], case["spread"]) for _ in range(n)]
    dst = list(range(n, n + n * k))
    # a target holds a short finished request, or nothing
    lens += [r.randrange(1, 17) if r.random() < 0.7 else -1 for _ in dst]
    lens += [-1] * (case["slots"] - len(lens))
    return lens, [i for i in range(n) for _ in range(k)], dst


def _visible(case):
    """Sum over the query rows of a call of the keys that each sees."""
    if case["op"] == "prompt":
        return sum(n * c + n * (n + 1) // 2 for n, c in _prompt_lens(case))
    off, pages, tail = _shared_plan(case)
    R = case["rows"]
    fresh = sum(bin(m).count("1") for m in _masks(case))
    return sum(R * (PAGE * pages[g] + tail[b]) + fresh for g in range(len(pages)) for b in range(off[g], off[g + 1]))


def work(case):
    if case["op"] == "fork":
        lens, src, dst = _fork_plan(case)
        token = case["layers"] * 2 * case["kv_heads"] * case["head_dim"] * 2
        # each used row of a page in use is read once for its source and written for each copy; the tables' entries
        pages = sum(-(-lens[s] // PAGE) for s in src)
        return {"bytes": sum(lens[s] % PAGE for s in set(src)) * token + sum(lens[s] % PAGE for s in src) * token + 4 * 4 * pages, "flops": 0}
    Hq, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "prompt":
        lens = _prompt_lens(case)
        rows, keys = sum(n for n, _ in lens), sum(n + c for n, c in lens)
    else:
        off, pages, tail = _shared_plan(case)
        rows, keys = case["batch"] * case["rows"], PAGE * sum(pages) + sum(tail) + case["batch"] * case["rows"]
    return {"bytes": 2 * 2 * rows * Hq * hd + 2 * 2 * keys * Hkv * hd, "flops": 4 * hd * Hq * _visible(case)}


def _masks(case):
    """Row r's visible new rows as bits: a chain, or a tree in breadth-first order with up to three children a node."""
    if not case["tree"]:
        return [(2 << r) - 1 for r in range(case["rows"])]
    bits = [1]
    for r in range(1, case["rows"]):
        bits.append(bits[(r - 1) // 3] | 1 << r)
    return bits


def _i64(bits):
    return [b - (1 << 64) if b >> 63 else b for b in bits]


# ----------------------------------------------------------------------------- inputs
def _pool(g, shape):
    """fp16 values as a cache holds them: unit variance, a few wide channels."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)
    x[..., 3::29] *= 4
    return x


def _tables(g, need, blocks):
    """A table for each request from shuffled pages: need[i] pages, -1 behind."""
    order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32).tolist()
    wide, rows = max(1, max(need)), []
    for n in need:
        rows.append(order[:n] + [-1] * (wide - n))
        order = order[n:]
    return rows, order


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "fork":
        lens, src, dst = _fork_plan(case)
        rows, free = _tables(g, [-(-max(n, 0) // PAGE) for n in lens], case["pages"])
        ref = [1] * case["pages"]
        for p in free:
            ref[p] = 0
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        s["tables"], s["lens"], s["ref"] = i32(rows), i32([max(n, 0) for n in lens]), i32(ref)
        s["n_blocks"] = i32([-1 if n < 0 else -(-n // PAGE) for n in lens])
        s["src"], s["dst"], s["status"] = i32(src), i32(dst), i32([0])
        s["pool"] = _pool(g, (case["layers"], case["pages"], 2, case["kv_heads"], PAGE, case["head_dim"]))
        return s
    Hq, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "prompt":
        lens = _prompt_lens(case)
        off = [0]
        for n, _ in lens:
            off.append(off[-1] + n)
        rows, _ = _tables(g, [-(-(n + c) // PAGE) for n, c in lens], sum(-(-(n + c) // PAGE) for n, c in lens) + 3)
        s["blocks"], T = sum(-(-(n + c) // PAGE) for n, c in lens) + 3, off[-1]
        s["ctx"] = torch.tensor([c for _, c in lens], dtype=torch.int32, device=DEV)
        s["off"] = torch.tensor(off, dtype=torch.int32, device=DEV)
        s["most"] = max(n for n, _ in lens)
        # queries lie in the fused projection's rows: [q | k | v]
        s["fused"] = torch.randn((T, (Hq + 2 * Hkv) * hd), generator=g, device=DEV, dtype=torch.float16) * 1.5
        s["out"] = torch.empty((T, Hq, hd), dtype=torch.float16, device=DEV)
    else:
        goff, pages, tail = _shared_plan(case)
        R, of = case["rows"], [g_ for g_ in range(case["groups"]) for _ in range(goff[g_], goff[g_ + 1])]
        mine = [-(-(t + R) // PAGE) for t in tail]
        s["blocks"] = sum(pages) + sum(mine) + 3
        got, _ = _tables(g, pages + mine, s["blocks"])
        rows = [got[of[b]][:pages[of[b]]] + got[len(pages) + b][:mine[b]] for b in range(case["batch"])]
        wide = max(map(len, rows))
        rows = [r + [-1] * (wide - len(r)) for r in rows]
        s["ctx"] = torch.tensor([PAGE * pages[of[b]] + tail[b] for b in range(case["batch"])], dtype=torch.int32, device=DEV)
        s["mask"] = torch.tensor(_i64(_masks(case)), dtype=torch.int64, device=DEV)
        s["goff"] = torch.tensor(goff, dtype=torch.int32, device=DEV)
        s["pages"] = torch.tensor(pages, dtype=torch.int32, device=DEV)
        s["q"] = torch.randn((case["batch"], R, Hq, hd), generator=g, device=DEV, dtype=torch.float16) * 1.5
        s["out"] = torch.empty((case["batch"], R, Hq, hd), dtype=torch.float16, device=DEV)
    s["tables"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
    s["kv"] = _pool(g, (s["blocks"], 2, Hkv, PAGE, hd))
    return s


# ----------------------------------------------------------------------------- plain forms
def _keys(s, wide):
    """Keys and values [B, Hkv, slots, hd] in 32 bits from the pages of each table."""
    x = s["kv"][s["tables"][:, :wide].clamp(min=0).long()]  # [B, pages, 2, Hkv, 16, hd]
    B, n, _, H, P, hd = x.shape
    x = x.permute(2, 0, 3, 1, 4, 5).reshape(2, B, H, n * P, hd).float()
    return x[0], x[1]


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(hd)) v over the keys where `seen`; a row that sees none gives zeros."""
    x = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(q.shape[-1])).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    return (x @ v) / torch.where(total == 0, 1.0, total)


def _plain_prompt(s):
    Hq, Hkv, hd, most = s["heads"], s["kv_heads"], s["head_dim"], s["most"]
    T, B = s["fused"].shape[0], s["batch"]
    q = s["fused"][:, :Hq * hd].reshape(T, Hq, hd)
    k, v = _keys(s, s["tables"].shape[1])
    j = torch.arange(most, device=DEV)
    at = (s["off"][:-1, None] + j).clamp(max=T - 1).long()  # [B, most]
    q = q[at].float().reshape(B, most, Hkv, Hq // Hkv, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, hd)
    slot = torch.arange(k.shape[2], device=DEV)
    seen = slot <= (s["ctx"][:, None] + j)[:, :, None]  # [B, most, slots]
    seen = seen[:, None, None].expand(B, 1, Hq // Hkv, most, slot.numel()).reshape(B, 1, -1, slot.numel())
    o = _attend(q, k, v, seen).reshape(B, Hkv, Hq // Hkv, most, hd).permute(0, 3, 1, 2, 4).reshape(B, most, Hq, hd)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(s["off"][1:].long(), t, right=True)
    return o[b, t - s["off"][b]].half()


def _plain_shared(s):
    Hq, Hkv, hd, B, R = s["heads"], s["kv_heads"], s["head_dim"], s["batch"], s["rows"]
    k, v = _keys(s, s["tables"].shape[1])
    q = s["q"].float().reshape(B, R, Hkv, Hq // Hkv, hd).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, hd)
    slot = torch.arange(k.shape[2], device=DEV)
    new = slot - s["ctx"][:, None]  # [B, slots]
    bit = (s["mask"][None, :, None] >> new.clamp(0, 63)[:, None, :]) & 1  # [B, R, slots]
    seen = (new < 0)[:, None, :] | ((new >= 0) & (new < R))[:, None, :] & (bit == 1)
    seen = seen[:, None, :, None].expand(B, 1, R, Hq // Hkv, slot.numel()).reshape(B, 1, -1, slot.numel())
    o = _attend(q, k, v, seen).reshape(B, Hkv, R, Hq // Hkv, hd)
    return o.permute(0, 2, 1, 3, 4).reshape(B, R, Hq, hd).half()


def _plain_fork(s):
    tables, ref, src, dst = s["tables"], s["ref"], s["src"].long(), s["dst"].long()
    col = torch.arange(tables.shape[1], device=DEV)
    count = torch.zeros(s["pages"] + 1, dtype=torch.int32, device=DEV)  # the last entry takes what is no page
    one = lambda rows, keep, w: count.index_add_(0, torch.where(keep, rows, s["pages"]).reshape(-1).long(), torch.full((rows.numel(),), w, dtype=torch.int32, device=DEV))  # noqa: E731
    one(tables[dst], col < s["n_blocks"][dst][:, None], -1)
    length = s["lens"][src]
    whole, part = length // PAGE, length % PAGE
    keep = col < whole[:, None]
    new = torch.where(keep, tables[src], -1)
    one(new, keep, 1)
    ref += count[:-1]
    free = torch.argsort((ref != 0).int(), stable=True)
    page = torch.where(part > 0, free[(part > 0).cumsum(0) - 1].int(), -1)
    new = torch.where((col == whole[:, None]) & (part > 0)[:, None], page[:, None], new)
    count.zero_()
    one(page, part > 0, 1)
    ref += count[:-1]
    old = tables[src].gather(1, ((length - 1) // PAGE)[:, None].long())[:, 0].long()  # the page in use, or a whole one that stays
    to = torch.where(part > 0, page.long(), old)
    used = (torch.arange(PAGE, device=DEV) < part[:, None])[None, :, None, None, :, None]
    s["pool"][:, to] = torch.where(used, s["pool"][:, old], s["pool"][:, to])
    tables[dst] = new
    s["lens"][dst] = length
    s["n_blocks"][dst] = (length + PAGE - 1) // PAGE
    s["status"].zero_()
    return [tables, s["n_blocks"], s["lens"], ref, s["status"], s["pool"]]


# ----------------------------------------------------------------------------- the library's calls
def _lib():
    import os
    import sys

    place = os.path.join(os.getcwd(), "sme-llm-edge_b200")
    if place not in sys.path:
        sys.path.insert(0, place)
    import specdec

    return specdec


def _work_space(s, size):
    """The call's workspace: its size asked for once, kept with the buffers as a serving loop does."""
    if "ws" not in s:
        s["ws"] = torch.empty(size(), dtype=torch.uint8, device=DEV)
    return s["ws"]


def _own_prompt(s):
    S = _lib()
    L, T = S.lib(), s["fused"].shape[0]
    Hq, Hkv, hd, B, wide = s["heads"], s["kv_heads"], s["head_dim"], s["batch"], s["tables"].shape[1]
    ws = _work_space(s, lambda: L.specdec_attention_prompt_workspace_bytes(B, T, Hq, Hkv, hd, wide))
    S.check(L.specdec_attention_prompt(s["fused"].data_ptr(), s["fused"].shape[1], s["kv"].data_ptr(), s["blocks"], Hkv, hd, s["tables"].data_ptr(), wide, s["ctx"].data_ptr(), s["off"].data_ptr(), B, T, Hq, s["out"].data_ptr(), Hq * hd, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return s["out"]


def _own_shared(s):
    S = _lib()
    L = S.lib()
    Hq, Hkv, hd, B, R, wide = s["heads"], s["kv_heads"], s["head_dim"], s["batch"], s["rows"], s["tables"].shape[1]
    ws = _work_space(s, lambda: L.specdec_attention_shared_prefix_workspace_bytes(B, R, s["groups"], Hq, Hkv, hd, wide))
    S.check(L.specdec_attention_shared_prefix(s["q"].data_ptr(), s["kv"].data_ptr(), s["blocks"], Hkv, hd, s["tables"].data_ptr(), wide, s["ctx"].data_ptr(), s["mask"].data_ptr(), s["goff"].data_ptr(), s["pages"].data_ptr(), s["groups"], B, R, Hq, s["out"].data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return s["out"]


def _own_fork(s):
    S = _lib()
    L, pool, n = S.lib(), s["pool"], s["src"].numel()
    ws = _work_space(s, lambda: L.specdec_kv_fork_pages_workspace_bytes(s["pages"], s["slots"], n))
    S.check(L.specdec_kv_fork_pages(s["tables"].data_ptr(), s["n_blocks"].data_ptr(), s["lens"].data_ptr(), s["ref"].data_ptr(), s["pages"], s["slots"], s["tables"].shape[1], s["src"].data_ptr(), s["dst"].data_ptr(), n, pool.data_ptr(), s["layers"], pool.stride(0), s["kv_heads"], s["head_dim"], s["status"].data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return [s["tables"], s["n_blocks"], s["lens"], s["ref"], s["status"], pool]


def run(state):
    if own:
        return {"prompt": _own_prompt, "shared": _own_shared, "fork": _own_fork}[state["op"]](state)
    return {"prompt": _plain_prompt, "shared": _plain_shared, "fork": _plain_fork}[state["op"]](state)


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fork":
        lens, src, dst = _fork_plan(case)
        tables, ref = s["tables"].tolist(), s["ref"].tolist()
        n_blocks = s["n_blocks"].tolist()
        for d in dst:  # the targets' old pages
            for p in tables[d][:max(0, n_blocks[d])]:
                ref[p] -= 1
        for a in src:
            for p in tables[a][:lens[a] // PAGE]:
                ref[p] += 1
        free = [p for p in range(case["pages"]) if ref[p] == 0]
        pool = s["pool"].double()
        for a, d in zip(src, dst):
            row = tables[a][:lens[a] // PAGE]
            if lens[a] % PAGE:
                p = free.pop(0)
                ref[p] = 1
                pool[:, p, :, :, :lens[a] % PAGE] = pool[:, tables[a][len(row)], :, :, :lens[a] % PAGE]
                row = row + [p]
            tables[d], n_blocks[d] = row + [-1] * (len(tables[d]) - len(row)), len(row)
        full = [max(0, n) for n in lens]
        for a, d in zip(src, dst):
            full[d] = lens[a]
        return [torch.tensor(tables), torch.tensor(n_blocks), torch.tensor(full), torch.tensor(ref), torch.tensor([0]), pool]
    Hq, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    G = Hq // Hkv
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    ctx = s["ctx"].tolist()
    for b in range(case["batch"]):
        if case["op"] == "prompt":
            lo, hi = s["off"][b].item(), s["off"][b + 1].item()
            q, n = s["fused"][lo:hi, :Hq * hd].reshape(hi - lo, Hq, hd), hi - lo
            see = torch.ones((n, ctx[b] + n), dtype=torch.bool, device=DEV).tril(ctx[b])
        else:
            q, n = s["q"][b], case["rows"]
            see = torch.ones((n, ctx[b] + n), dtype=torch.bool, device=DEV)
            see[:, ctx[b]:] = torch.tensor([[m >> i & 1 for i in range(n)] for m in _masks(case)], device=DEV) == 1
        pages = s["tables"][b, :-(-(ctx[b] + n) // PAGE)].long()
        for h in range(Hkv):
            kv = s["kv"][pages, :, h].double()  # [pages, 2, 16, hd]
            k, v = (kv[:, i].reshape(-1, hd)[:ctx[b] + n] for i in (0, 1))
            for i in range(h * G, h * G + G):
                x = torch.einsum("nd,kd->nk", q[:, i].double(), k) / hd ** 0.5
                p = torch.softmax(x.masked_fill(~see, -math.inf), 1)
                if case["op"] == "prompt":
                    out[lo:hi, i] = p @ v
                else:
                    out[b, :, i] = p @ v
    return out
