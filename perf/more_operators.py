"""Cases, plain forms and calls of the operators of a cache of bounded length, over the paged fp16 K/V pool:

  write       queries and keys of new tokens normed per head and rotated, keys and values put into their pages
  window      causal attention of packed rows that see a window of slots and a few first ones
  accumulate  causal attention of packed rows that also adds up the weight that each slot received
  evict       requests that keep their first, their last and their heaviest tokens; the others' room is given back

`own = False` computes them with elementary torch operations in 32 bits; `own = True` calls the library.
A page holds 16 tokens of one layer as [K|V][kv head][16][head_dim]; a pool is [pages] of them.
"""
import math
import random

import torch

own = False

PAGE = 16
DEV = "cuda"
EPS = 1e-5
THETA = 10000.0


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # the pending token of one short request of the small model: latency alone
        dict(name="write 1 row", op="write", heads=8, kv_heads=2, head_dim=64, batch=1, rows=1, cached=40, spread=0, half=False),
        # chain verify rows of a batch, from the projection's 32-bit rows
        dict(name="write 32 x 5 rows", op="write", heads=32, kv_heads=8, head_dim=128, batch=32, rows=5, cached=2048, spread=3, half=False),
        # packed prompts of different lengths, from a projection that gives 16 bits
        dict(name="write 8 prompts", op="write", heads=40, kv_heads=8, head_dim=128, batch=8, rows=2501, cached=0, spread=7, half=True),
        # one pending token, window longer than the context
        dict(name="window 1 x 1 on 200", op="window", heads=8, kv_heads=2, head_dim=64, batch=1, rows=1, cached=200, spread=0, window=512, sinks=4),
        # single tokens of a batch with long ragged contexts: the decode form
        dict(name="window 64 x 1, 4096 of 8k", op="window", heads=32, kv_heads=8, head_dim=128, batch=64, rows=1, cached=8192, spread=5, window=4096, sinks=4),
        # the next chunk of prompts whose beginning is in the cache
        dict(name="window chunks 512, 2000 of 4k", op="window", heads=40, kv_heads=8, head_dim=128, batch=4, rows=512, cached=4099, spread=0, window=2000, sinks=20),
        # one long prompt from its first token
        dict(name="window prompt 8192, 1024", op="window", heads=32, kv_heads=8, head_dim=128, batch=1, rows=8192, cached=0, spread=0, window=1024, sinks=4),
        # one pending token of the small model
        dict(name="accumulate 1 x 1 on 200", op="accumulate", heads=8, kv_heads=2, head_dim=64, batch=1, rows=1, cached=200, spread=0),
        # single tokens of a batch, every decoding step
        dict(name="accumulate 64 x 1 on 4k", op="accumulate", heads=32, kv_heads=8, head_dim=128, batch=64, rows=1, cached=4096, spread=5),
        # the last rows of prompts, whose weights say what of each prompt is kept
        dict(name="accumulate 4 x 16 on 8k", op="accumulate", heads=32, kv_heads=8, head_dim=128, batch=4, rows=16, cached=8176, spread=2),
        # one request of the small model that has outgrown its room
        dict(name="evict 1, 300 to 200", op="evict", layers=4, kv_heads=2, head_dim=64, requests=1, others=2, tokens=300, keep=200, first=4, last=32, shared=0, spread=0),
        # long requests, half of them under one system prompt, in all 32 layers
        dict(name="evict 8, 3000 to 1024", op="evict", layers=32, kv_heads=8, head_dim=128, requests=8, others=2, tokens=3000, keep=1024, first=16, last=256, shared=20, spread=4),
    ]


HEADS = ((8, 2, 64), (32, 8, 128), (40, 8, 128))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "window", "window", "accumulate", "accumulate", "evict"))
    heads, kv_heads, hd = rng.choice(HEADS)
    if op == "write":
        rows, cached = _log(rng, 1, 6000), rng.choice((0, _log(rng, 1, 4096)))
        batch = _log(rng, 1, max(1, min(64, 16384 // rows)))
        return dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=hd, batch=batch, rows=rows, cached=cached, spread=rng.randrange(1, 1000), half=rng.random() < 0.5)
    if op == "window":
        rows, cached = rng.choice((1, 1, _log(rng, 1, 6000))), rng.choice((0, _log(rng, 1, 8192)))
        # the padded plain form stays below the largest listed case
        most = max(1, min(64, int(32 * 8192 * 8192 / (heads * rows * (rows + cached))), 16384 // rows + 1))
        return dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=hd, batch=_log(rng, 1, most), rows=rows, cached=cached, spread=rng.randrange(1, 1000), window=_log(rng, 1, 8192), sinks=rng.choice((0, 1, 4, 16, _log(rng, 1, 256))))
    if op == "accumulate":
        rows, cached = rng.choice((1, 1, 5, _log(rng, 1, 32))), _log(rng, 1, 8192)
        most = max(1, min(64, 64 * 4096 // (cached * max(1, rows // 4))))
        return dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=hd, batch=_log(rng, 1, most), rows=rows, cached=cached, spread=rng.randrange(1, 1000))
    requests, tokens = _log(rng, 1, 8), _log(rng, 40, 3000)
    keep = _log(rng, 20, max(21, tokens - 1))
    first, last = rng.randrange(0, 1 + min(64, keep // 3)), rng.randrange(0, 1 + keep // 3)
    return dict(op=op, layers=rng.choice((2, 4, 32)), kv_heads=kv_heads, head_dim=hd, requests=requests, others=rng.randrange(4), tokens=tokens, keep=keep, first=first, last=last, shared=rng.choice((0, rng.randrange(1 + tokens // 64))), spread=rng.randrange(1, 1000))


def _ragged(r, most, spread, least=64):
    """A length up to `most`, spread over its logarithm."""
    return most if not spread else _log(r, max(1, most // least), most)


def _lens(case):
    """(new rows, cached tokens) of each sequence; the first has the case's own."""
    r = random.Random(case["spread"])
    got = [(case["rows"], case["cached"])]
    for _ in range(case["batch"] - 1):
        n = case["rows"] if case["rows"] <= 32 else _ragged(r, case["rows"], case["spread"])
        got.append((n, _ragged(r, case["cached"], case["spread"]) if case["cached"] else 0))
    return got


def _evict_plan(case):
    """Tokens of each request (the last `others` are not evicted), shared pages of its beginning, and the requests named."""
    r = random.Random(case["spread"])
    n = case["requests"] + case["others"]
    lens = [case["tokens"] if not i or not case["spread"] else max(1, int(case["tokens"] * r.uniform(0.4, 1.0))) for i in range(n)]
    shared = [case["shared"] if i % 2 == 0 and PAGE * case["shared"] <= lens[i] and case["requests"] > 1 else 0 for i in range(n)]
    reqs = list(range(case["requests"]))
    r.shuffle(reqs)
    return lens, shared, reqs


def _seen_by(n, c, window, sinks):
    """Slots that the rows of a sequence see: how many in all, and how many of them any row sees."""
    total = sum(min(c + i + 1, window) + min(sinks, max(0, c + i + 1 - window)) for i in range(n))
    return total, min(n + c, window + n - 1) + min(sinks, max(0, c + 1 - window))


def work(case):
    Hkv, hd = case["kv_heads"], case["head_dim"]
    if case["op"] == "evict":
        lens, _, reqs = _evict_plan(case)
        token = case["layers"] * 2 * Hkv * hd * 2
        gone = [a for a in reqs if lens[a] > case["keep"]]
        # what stays behind the first tokens moves up; the weights are read, and written for those that stay
        moved = len(gone) * (case["keep"] - case["first"])
        return {"bytes": 2 * moved * token + sum(4 * Hkv * 2 * lens[a] + 4 * lens[a] // PAGE for a in gone), "flops": sum(Hkv * lens[a] for a in gone)}
    Hq, lens = case["heads"], _lens(case)
    rows = sum(n for n, _ in lens)
    if case["op"] == "write":
        one = (Hq + 2 * Hkv) * hd
        # each row's values once in and once out, its angles, its position and slot
        return {"bytes": rows * one * ((2 if case["half"] else 4) + 2) + rows * (4 * hd + 8), "flops": rows * 7 * (Hq + Hkv) * hd}
    window, sinks = (case["window"], case["sinks"]) if case["op"] == "window" else (1 << 30, 0)
    pairs, keys = map(sum, zip(*(_seen_by(n, c, window, sinks) for n, c in lens)))
    more = 2 * 4 * Hkv * keys if case["op"] == "accumulate" else 0
    return {"bytes": 2 * 2 * rows * Hq * hd + 2 * 2 * keys * Hkv * hd + more, "flops": 4 * hd * Hq * pairs}


# ----------------------------------------------------------------------------- inputs
def _pool(g, shape):
    """fp16 values as a cache holds them: unit variance, a few wide channels."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)
    x[..., 3::29] *= 4
    return x


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _prepare_evict(case, g, s):
    lens, shared, reqs = _evict_plan(case)
    n, need = len(lens), [-(-x // PAGE) for x in lens]
    pages = case["shared"] + sum(need) + case["requests"] * -(-case["keep"] // PAGE) + 5
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    common, order, wide = order[:case["shared"]], order[case["shared"]:], max(need) + 2
    rows, ref = [], [0] * pages
    for i in range(n):
        own_pages = need[i] - shared[i]
        row, order = common[:shared[i]] + order[:own_pages], order[own_pages:]
        for p in row:
            ref[p] += 1
        rows += row + [-1] * (wide - len(row))
    s["slots"], s["wide"], s["pages"], s["ldw"] = n, wide, pages, wide * PAGE
    w = torch.randn((n, case["kv_heads"], s["ldw"]), generator=g, device=DEV).mul_(2).exp_()
    for i in range(n):
        w[i, :, lens[i]:] = 0
    # tables, their lengths in pages and tokens, reference counts and weights, side by side
    s["grown"] = torch.cat([_i32(rows + need + lens + ref), w.reshape(-1).view(torch.int32)])
    s["live"] = s["grown"].clone()
    parts = s["live"].split([n * wide, n, n, pages, w.numel()])
    s["tables"], s["n_blocks"], s["lens"], s["ref"] = parts[0].view(n, wide), parts[1], parts[2], parts[3]
    s["weights"] = parts[4].view(torch.float32).view(n, case["kv_heads"], s["ldw"])
    s["reqs"], s["status"] = _i32(reqs), _i32([0])
    s["kept"] = torch.full((len(reqs), case["keep"]), -1, dtype=torch.int32, device=DEV)
    s["pool"] = _pool(g, (case["layers"], pages, 2, case["kv_heads"], PAGE, case["head_dim"]))
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "evict":
        return _prepare_evict(case, g, s)
    Hq, Hkv, hd, lens = case["heads"], case["kv_heads"], case["head_dim"], _lens(case)
    off = [0]
    for n, _ in lens:
        off.append(off[-1] + n)
    need, T = [-(-(n + c) // PAGE) for n, c in lens], off[-1]
    s["blocks"], wide, rows = sum(need) + 3, max(need), []
    order = torch.randperm(s["blocks"], generator=g, device=DEV).tolist()
    for k in need:
        rows.append(order[:k] + [-1] * (wide - k))
        order = order[k:]
    s["tables"], s["off"], s["ctx"] = _i32(rows), _i32(off), _i32([c for _, c in lens])
    s["most"], s["T"] = max(n for n, _ in lens), T
    if case["op"] == "write":
        # a projection's rows: [q | k | v]
        x = torch.randn((T, (Hq + 2 * Hkv) * hd), generator=g, device=DEV)
        x[:, 5::37] *= 6
        s["qkv"] = x.half() if case["half"] else x
        s["q_norm"], s["k_norm"] = (1 + 0.2 * torch.randn(hd, generator=g, device=DEV) for _ in range(2))
        far = max(n + c for n, c in lens)
        angle = torch.arange(far, device=DEV, dtype=torch.float64)[:, None] * THETA ** (-2.0 * torch.arange(hd // 2, device=DEV, dtype=torch.float64) / hd)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["pos"] = torch.cat([torch.arange(c, c + n, dtype=torch.int32, device=DEV) for n, c in lens])
        s["q"] = torch.empty((T, Hq, hd), dtype=torch.float16, device=DEV)
    else:
        s["q"] = torch.randn((T, Hq, hd), generator=g, device=DEV, dtype=torch.float16) * 1.5
        s["out"] = torch.empty((T, Hq, hd), dtype=torch.float16, device=DEV)
        if case["op"] == "accumulate":
            # what earlier steps have added up
            s["ldw"] = wide * PAGE
            s["weights"] = torch.rand((case["batch"], Hkv, s["ldw"]), generator=g, device=DEV) * 0.01
    s["kv"] = _pool(g, (s["blocks"], 2, Hkv, PAGE, hd))
    return s


# ----------------------------------------------------------------------------- plain forms
def _places(s):
    """Sequence, slot and page of each packed row."""
    t = torch.arange(s["T"], device=DEV)
    b = torch.searchsorted(s["off"][1:].long(), t, right=True)
    slot = s["ctx"][b] + t - s["off"][b]
    return b, slot, s["tables"][b, slot // PAGE].long()


def _plain_write(s):
    Hq, Hkv, hd, T = s["heads"], s["kv_heads"], s["head_dim"], s["T"]
    x = s["qkv"].float().reshape(T, Hq + 2 * Hkv, hd)
    w = torch.cat([s["q_norm"].expand(Hq, hd), s["k_norm"].expand(Hkv, hd)])
    y = x[:, :Hq + Hkv]
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    c, n = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    y = torch.cat([a * c - b * n, b * c + a * n], -1).half()
    _, slot, page = _places(s)
    s["q"].copy_(y[:, :Hq])
    s["kv"][page, 0, :, slot % PAGE] = y[:, Hq:]
    s["kv"][page, 1, :, slot % PAGE] = x[:, Hq + Hkv:].half()
    return [s["q"], s["kv"]]


def _plain_attend(s):
    Hq, Hkv, hd, most, T, B = s["heads"], s["kv_heads"], s["head_dim"], s["most"], s["T"], s["batch"]
    x = s["kv"][s["tables"].clamp(min=0).long()].permute(2, 0, 3, 1, 4, 5).reshape(2, B, Hkv, -1, hd).float()
    k, v = x[0], x[1]
    j = torch.arange(most, device=DEV)
    at = (s["off"][:-1, None] + j).clamp(max=T - 1).long()  # [B, most]
    q = s["q"][at].float().reshape(B, most, Hkv, Hq // Hkv, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, hd)
    slot = torch.arange(k.shape[2], device=DEV)
    row = (s["ctx"][:, None] + j)[:, :, None]
    seen = (slot <= row) & (j < (s["off"][1:] - s["off"][:-1])[:, None])[:, :, None]  # [B, most, slots]
    if s["op"] == "window":
        seen &= (slot < s["sinks"]) | (slot > row - s["window"])
    seen = seen[:, None, None].expand(B, 1, Hq // Hkv, most, slot.numel()).reshape(B, 1, -1, slot.numel())
    x = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(hd)).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    x /= torch.where(total == 0, 1.0, total)
    o = (x @ v).reshape(B, Hkv, Hq // Hkv, most, hd).permute(0, 3, 1, 2, 4).reshape(B, most, Hq, hd)
    b, at, _ = _places(s)
    s["out"].copy_(o[b, at - s["ctx"][b]])
    if s["op"] == "window":
        return s["out"]
    s["weights"][..., :slot.numel()] += x.sum(2)
    return [s["out"], s["weights"]]


def _plain_evict(s):
    keep, first, last, n = s["keep"], s["first"], s["last"], s["reqs"].numel()
    tables, ref, lens, n_blocks, weights = s["tables"], s["ref"], s["lens"], s["n_blocks"], s["weights"]
    r, wide = s["reqs"].long(), s["wide"]
    length = lens[r].long()
    gone = length > keep  # [n]: the others stay as they are
    slot = torch.arange(s["ldw"], device=DEV)
    # first and last tokens before all, slots behind the length after all; of equal weights the lower slot
    rank = weights[r].double().sum(1).float().double()
    rank = torch.where((slot < first) | (slot >= (length - last)[:, None]), math.inf, rank)
    rank = torch.where(slot < length[:, None], rank, -math.inf)
    best = torch.sort(rank, dim=1, descending=True, stable=True)[1][:, :keep]
    best = torch.cat([best, best.new_full((n, keep - best.shape[1]), s["ldw"])], 1) if best.shape[1] < keep else best
    place = torch.arange(keep, device=DEV)
    kept = torch.where(gone[:, None], torch.sort(best, dim=1)[0], torch.where(place < length[:, None], place, -1))
    moved = (kept != place) & gone[:, None]
    hole = torch.where(moved.any(1), moved.int().argmax(1), keep)  # the first token that moves
    # pages that are written: shared ones are replaced
    page = torch.arange(wide, device=DEV)
    pages = -(-keep // PAGE)
    old = tables[r].long()
    held = (page < n_blocks[r][:, None]) & gone[:, None]
    written = held & (page >= (hole // PAGE)[:, None]) & (page < pages) & (hole < keep)[:, None]
    swap = written & (ref[old.clamp(min=0)] > 1)
    free = torch.argsort((ref != 0).int(), stable=True)
    fresh = free[(swap.reshape(-1).cumsum(0) - 1).clamp(min=0)].reshape(n, wide)
    new = torch.where(swap, fresh, torch.where(held & (page >= pages), -1, old))
    # tokens: from the first that moves on, and what stands before it on a page that is replaced
    start = torch.where(swap.gather(1, (hole // PAGE).clamp(max=wide - 1)[:, None])[:, 0], hole // PAGE * PAGE, hole)
    i, j = torch.nonzero((place >= start[:, None]) & gone[:, None] & (hole < keep)[:, None], as_tuple=True)
    a = kept[i, j]
    x = s["pool"][:, old[i, a // PAGE], :, :, a % PAGE]
    s["pool"][:, new[i, j // PAGE], :, :, j % PAGE] = x
    w = weights[r].gather(2, kept.clamp(min=0)[:, None].expand(-1, weights.shape[1], -1))
    full = torch.zeros_like(weights[r])
    full[..., :keep] = w[..., :s["ldw"]]
    weights[r] = torch.where(gone[:, None, None], full, weights[r])
    drop = swap | (held & (page >= pages))
    ref.index_add_(0, old.clamp(min=0).reshape(-1), -drop.reshape(-1).int())
    ref.index_add_(0, fresh.reshape(-1), swap.reshape(-1).int())
    tables[r] = new.int()
    n_blocks[r] = torch.where(gone, pages, n_blocks[r].long()).int()
    lens[r] = torch.where(gone, keep, length).int()
    s["kept"].copy_(kept)
    s["status"].zero_()
    return [tables, n_blocks, lens, ref, s["kept"], s["status"], weights, s["pool"]]


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


def _own_write(s):
    S = _lib()
    Hq, Hkv, hd = s["heads"], s["kv_heads"], s["head_dim"]
    S.check(S.lib().specdec_qk_norm_rope_kv(s["qkv"].data_ptr(), int(s["half"]), s["qkv"].shape[1], s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), EPS, s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], hd, s["pos"].data_ptr(), s["kv"].data_ptr(), s["blocks"], Hkv, hd, s["tables"].data_ptr(), s["tables"].shape[1], s["ctx"].data_ptr(), s["off"].data_ptr(), s["batch"], s["T"], Hq, s["q"].data_ptr(), Hq * hd, torch.cuda.current_stream().cuda_stream))
    return [s["q"], s["kv"]]


def _own_window(s):
    S = _lib()
    L, T, B = S.lib(), s["T"], s["batch"]
    Hq, Hkv, hd, wide = s["heads"], s["kv_heads"], s["head_dim"], s["tables"].shape[1]
    ws = _work_space(s, lambda: L.specdec_attention_window_workspace_bytes(B, T, Hq, Hkv, hd, wide))
    S.check(L.specdec_attention_window(s["q"].data_ptr(), Hq * hd, s["kv"].data_ptr(), s["blocks"], Hkv, hd, s["tables"].data_ptr(), wide, s["ctx"].data_ptr(), s["off"].data_ptr(), B, T, Hq, s["window"], s["sinks"], s["out"].data_ptr(), Hq * hd, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return s["out"]


def _own_accumulate(s):
    S = _lib()
    L, T, B = S.lib(), s["T"], s["batch"]
    Hq, Hkv, hd, wide = s["heads"], s["kv_heads"], s["head_dim"], s["tables"].shape[1]
    ws = _work_space(s, lambda: L.specdec_attention_accumulate_workspace_bytes(B, T, Hq, Hkv, hd, wide))
    S.check(L.specdec_attention_accumulate(s["q"].data_ptr(), Hq * hd, s["kv"].data_ptr(), s["blocks"], Hkv, hd, s["tables"].data_ptr(), wide, s["ctx"].data_ptr(), s["off"].data_ptr(), B, T, Hq, s["weights"].data_ptr(), s["ldw"], s["out"].data_ptr(), Hq * hd, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return [s["out"], s["weights"]]


def _own_evict(s):
    S = _lib()
    L, pool, n = S.lib(), s["pool"], s["reqs"].numel()
    ws = _work_space(s, lambda: L.specdec_kv_evict_pages_workspace_bytes(s["pages"], s["slots"], s["wide"], n, s["keep"]))
    S.check(L.specdec_kv_evict_pages(s["tables"].data_ptr(), s["n_blocks"].data_ptr(), s["lens"].data_ptr(), s["ref"].data_ptr(), s["pages"], s["slots"], s["wide"], s["reqs"].data_ptr(), n, s["keep"], s["first"], s["last"], s["weights"].data_ptr(), s["kv_heads"], s["ldw"], pool.data_ptr(), s["layers"], pool.stride(0), s["kv_heads"], s["head_dim"], s["kept"].data_ptr(), s["status"].data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return [s["tables"], s["n_blocks"], s["lens"], s["ref"], s["kept"], s["status"], s["weights"], pool]


def run(state):
    if state["op"] == "evict":
        state["live"].copy_(state["grown"])  # the requests have grown again, in the scheduler's tables
    if own:
        return {"write": _own_write, "window": _own_window, "accumulate": _own_accumulate, "evict": _own_evict}[state["op"]](state)
    return {"write": _plain_write, "window": _plain_attend, "accumulate": _plain_attend, "evict": _plain_evict}[state["op"]](state)


# ----------------------------------------------------------------------------- 64 bits
def _exact_write(s):
    Hq, Hkv, hd = s["heads"], s["kv_heads"], s["head_dim"]
    x = s["qkv"].double()
    q = torch.zeros((s["T"], Hq, hd), dtype=torch.float64, device=DEV)
    kv = s["kv"].double()
    b, slot, page = _places(s)
    angle = s["pos"].double()[:, None] * THETA ** (-2.0 * torch.arange(hd // 2, device=DEV, dtype=torch.float64) / hd)
    turn = torch.complex(angle.cos(), angle.sin())
    for h in range(Hq + 2 * Hkv):
        y = x[:, h * hd:(h + 1) * hd]
        if h < Hq + Hkv:
            w = (s["q_norm"] if h < Hq else s["k_norm"]).double()
            y = y / (y.square().sum(1, keepdim=True) / hd + EPS).sqrt() * w
            z = torch.complex(y[:, :hd // 2], y[:, hd // 2:]) * turn
            y = torch.cat([z.real, z.imag], 1)
        if h < Hq:
            q[:, h] = y
        else:
            kv[page, int(h >= Hq + Hkv), (h - Hq) % Hkv, slot % PAGE] = y
    return [q, kv]


def _exact_attend(s):
    Hq, Hkv, hd = s["heads"], s["kv_heads"], s["head_dim"]
    G = Hq // Hkv
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    weights = s["weights"].double() if s["op"] == "accumulate" else None
    ctx, off = s["ctx"].tolist(), s["off"].tolist()
    for b in range(s["batch"]):
        lo, hi = off[b], off[b + 1]
        n, L = hi - lo, ctx[b] + hi - lo
        see = torch.ones((n, L), dtype=torch.bool, device=DEV).tril(ctx[b])
        if s["op"] == "window":
            see &= ~torch.ones_like(see).tril(ctx[b] - s["window"]) | (torch.arange(L, device=DEV) < s["sinks"])
        pages = s["tables"][b, :-(-L // PAGE)].long()
        for h in range(Hkv):
            kv = s["kv"][pages, :, h].double()  # [pages, 2, 16, hd]
            k, v = (kv[:, i].reshape(-1, hd)[:L] for i in (0, 1))
            for i in range(h * G, h * G + G):
                x = torch.einsum("nd,kd->nk", s["q"][lo:hi, i].double(), k) / hd ** 0.5
                p = torch.softmax(x.masked_fill(~see, -math.inf), 1)
                out[lo:hi, i] = p @ v
                if weights is not None:
                    weights[b, h, :L] += p.sum(0)
    return out if weights is None else [out, weights]


def _exact_evict(s):
    keep = s["keep"]
    tables, n_blocks, lens, ref = (s[k].tolist() for k in ("tables", "n_blocks", "lens", "ref"))
    weights, pool, was = s["weights"].double(), s["pool"].double(), list(ref)
    free = [p for p, r in enumerate(ref) if r == 0]
    kept = []
    for a in s["reqs"].tolist():
        L = lens[a]
        if L <= keep:
            kept.append(list(range(L)) + [-1] * (keep - L))
            continue
        score = weights[a].sum(0).float().tolist()
        must = set(range(s["first"])) | set(range(L - s["last"], L))
        rest = sorted((j for j in range(L) if j not in must), key=lambda j: (-score[j], j))
        stay = sorted(must | set(rest[:keep - len(must)]))
        kept.append(stay)
        hole = next((j for j, k in enumerate(stay) if j != k), keep)
        row = tables[a]
        new = row[:-(-keep // PAGE)]
        start = hole
        for d in range(hole // PAGE, len(new)) if hole < keep else ():
            if was[row[d]] > 1:
                new[d] = free.pop(0)
                ref[row[d]] -= 1
                ref[new[d]] += 1
                start = min(start, max(d * PAGE, hole // PAGE * PAGE))
        for d in range(len(new), n_blocks[a]):
            ref[row[d]] -= 1
        if start < keep:
            at = torch.tensor(stay[start:], device=DEV)
            to = torch.arange(start, keep, device=DEV)
            old_pages, new_pages = torch.tensor(row, device=DEV), torch.tensor(new, device=DEV)
            pool[:, new_pages[to // PAGE], :, :, to % PAGE] = pool[:, old_pages[at // PAGE], :, :, at % PAGE]
        w = weights[a][:, torch.tensor(stay, device=DEV)]
        weights[a] = 0
        weights[a][:, :keep] = w
        tables[a] = new + [-1] * (len(row) - len(new))
        n_blocks[a], lens[a] = len(new), keep
    return [torch.tensor(tables), torch.tensor(n_blocks), torch.tensor(lens), torch.tensor(ref), torch.tensor(kept), torch.tensor([0]), weights, pool]


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "window": _exact_attend, "accumulate": _exact_attend, "evict": _exact_evict}[case["op"]](s)
