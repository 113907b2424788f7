"""Measured cases of the paged K/V cache operators: append (RoPE and page write), attend (a chunk of new
tokens, or one token, over paged histories) and the page operators (reserve, fork, free, compact).

A pool holds pages of 64 positions, laid out as the engine's: [layer][kv head][K | V][head_dim / 64][64
positions][64 dims], the eight 16-byte blocks of a position's 64 dims stored at block ^ (position & 7).  `table`
maps (slot, page number) to a page of the pool (-1: none), `refs` counts the slots that share a page, `lengths`
holds each slot's positions.  Batch entry b is slot slots[b] with rows q_start[b] .. q_start[b + 1]; its row i of
n stands at position lengths[slot] - n + i.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

PAGE = 64
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hawkpoint-npu-llm_b200")


# ---- cases -------------------------------------------------------------------------
def attend(seqs, rows, ctx, heads, dtype="bfloat16", window=0, mix=1, **more):
    """seqs sequences, (least, most) new rows, (least, most) positions with them, (q heads, kv heads, head_dim)"""
    return dict(op="attend", seqs=seqs, rows_min=rows[0], rows_max=rows[1], ctx_min=ctx[0], ctx_max=ctx[1],
                q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2], dtype=dtype, window=window, mix=mix, **more)


def append(seqs, rows, ctx, heads, dtype="bfloat16", mix=1, **more):
    return dict(attend(seqs, rows, ctx, heads, dtype, 0, mix, **more), op="append")


def listed():
    qwen, smol, wide = (14, 2, 64), (9, 3, 64), (32, 8, 128)
    return [
        # one stream of the 4096-position context decodes a token: latency
        attend(1, (1, 1), (4032, 4032), qwen, name="attend: decode, 1 stream"),
        # a serving step of 128 ragged streams, a token each
        attend(128, (1, 1), (200, 4096), qwen, mix=2, name="attend: decode, 128 streams"),
        # the same far beyond the engine's context, heads of 128, FP16: the most bytes
        attend(48, (1, 1), (4000, 16000), wide, "float16", mix=3, name="attend: decode, long, heads of 128"),
        # a 256-row step: most streams decode, a few take a 32-position prefill chunk
        attend(96, (1, 32), (33, 3000), smol, mix=4, name="attend: mixed step"),
        # chunks of 200 to 512 prompt positions late in long prompts, a sliding window
        attend(4, (200, 512), (1000, 8000), wide, window=1024, mix=5, name="attend: chunks, window"),
        # whole prompts: the most arithmetic
        attend(4, (3000, 4096), (3000, 4096), qwen, mix=6, name="attend: whole prompts"),
        # one decoded token of one stream: the smallest call
        append(1, (1, 1), (900, 900), qwen, mix=7, name="append: 1 row"),
        # 24 prompts in one step
        append(24, (300, 2000), (300, 4000), qwen, mix=8, name="append: 24 prompts"),
        # a beam forks a stream once
        dict(op="fork", slots=8, count=1, ctx_min=700, ctx_max=700, layers=30, kv_heads=3, head_dim=64, mix=9,
             name="fork: 1 stream"),
        # 64 requests start from kept prefixes of the 24-layer model
        dict(op="fork", slots=96, count=64, ctx_min=100, ctx_max=2000, layers=24, kv_heads=2, head_dim=64, mix=10,
             name="fork: 64 requests"),
        # a long-running server's pool closes its gaps
        dict(op="compact", slots=96, pages=3000, ctx_min=100, ctx_max=2000, layers=24, kv_heads=2, head_dim=64,
             mix=11, name="compact: a server's pool"),
        # between two steps: 32 requests end, 32 start with their prompts' pages
        dict(op="turnover", slots=256, pages=8192, count=32, ctx_min=8, ctx_max=2000, mix=12,
             name="free and reserve: 32 requests"),
    ]


def spread(rng, lo, hi):
    """an integer of [lo, hi], even over its logarithm"""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    mix = rng.randrange(1 << 20)
    op = rng.choice(["attend", "attend", "attend", "append", "fork", "compact", "turnover"])
    heads = rng.choice([(14, 2, 64), (9, 3, 64), (4, 4, 64), (32, 8, 128), (16, 1, 128), (3, 1, 64)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if op == "attend":
        kind = rng.choice(["decode", "mixed", "chunk", "whole"])
        window = rng.choice([0, 0, 0, spread(rng, 16, 2000)])
        if kind == "decode":
            top = spread(rng, 1, 12000)
            seqs = spread(rng, 1, max(1, min(200, 200000 // top)))
            rows = (1, rng.choice([1, 1, 2, 5]))
            return attend(seqs, rows, (max(rows[1], top // 16), max(rows[1], top)), heads, dtype, window, mix)
        if kind == "mixed":
            top = spread(rng, 64, 4000)
            return attend(spread(rng, 2, 64), (1, spread(rng, 2, 48)), (49, max(49, top)), heads, dtype, window, mix)
        if kind == "chunk":
            rows = spread(rng, 17, 600)
            return attend(spread(rng, 1, 4), (max(1, rows // 3), rows), (rows, rows + spread(rng, 1, 6000)), heads,
                          dtype, window, mix)
        top = spread(rng, 100, 2000)
        return attend(spread(rng, 1, 4), (top // 2, top), (top // 2, top), heads, dtype, window, mix)
    if op == "append":
        top = spread(rng, 1, 1500)
        return append(spread(rng, 1, 24), (max(1, top // 8), top), (top, top + spread(rng, 1, 2000)), heads, dtype, mix)
    layers, (_, kv_heads, head_dim) = spread(rng, 1, 24), heads
    layers = min(layers, max(1, 8192 // (kv_heads * head_dim * 2)))
    if op == "fork":
        count = spread(rng, 1, 64)
        return dict(op=op, slots=count + spread(rng, 1, 40), count=count, ctx_min=1, ctx_max=spread(rng, 1, 2000),
                    layers=layers, kv_heads=kv_heads, head_dim=head_dim, mix=mix)
    if op == "compact":
        slots = spread(rng, 1, 96)
        return dict(op=op, slots=slots, pages=slots * 16 + spread(rng, 1, 1400), ctx_min=1, ctx_max=1000,
                    layers=layers, kv_heads=kv_heads, head_dim=head_dim, mix=mix)
    slots, top = spread(rng, 2, 256), spread(rng, 1, 2000)
    return dict(op=op, slots=slots, pages=2 * slots * (top // PAGE + 1) + 8, count=spread(rng, 1, slots), ctx_min=1,
                ctx_max=top, mix=mix)


# ---- what a case fixes: lengths, rows and page tables (host) ------------------------
def plan(case):
    """The case's slots, rows, lengths and page table as NumPy arrays: the same for every seed."""
    r = np.random.default_rng(case["mix"])
    op = case["op"]
    if op in ("attend", "append"):
        n = case["seqs"]
        rows = r.integers(case["rows_min"], case["rows_max"] + 1, n)
        if case["rows_max"] > case["rows_min"]:  # a mixed step: most streams decode
            few = r.permutation(n)[: max(1, n // 8)]
            if case["rows_min"] == 1 and n > 8:
                rows = np.ones(n, np.int64)
                rows[few] = r.integers(1, case["rows_max"] + 1, len(few))
            rows[few[0]] = case["rows_max"]
        top = r.integers(case["ctx_min"], case["ctx_max"] + 1, n)
        top[r.integers(0, n)] = case["ctx_max"]
        lengths = np.maximum(top, rows)
        slots = r.permutation(n)
        by_slot = np.empty(n, np.int64)
        by_slot[slots] = lengths
        held = by_slot
        pages = int((-(-held // PAGE)).sum()) + 3
        refs_groups = 0
    else:
        n = case["slots"]
        rows = slots = None
        held = r.integers(case["ctx_min"], case["ctx_max"] + 1, n)
        if op == "fork":
            held[n - case["count"]:] = 0  # the slots forked into are empty
            pages = int((-(-held // PAGE)).sum()) + 2 * case["count"] + 5
        else:
            pages = case["pages"]
        refs_groups = n // 4 if op == "compact" else 0
        by_slot = held
    width = -(-int(max(held.max(), case["ctx_max"])) // PAGE) + 1
    need = -(-held // PAGE)
    order = r.permutation(pages)
    table = np.full((n, width), -1, np.int64)
    at = 0
    for s in range(n):
        k = int(need[s])
        table[s, :k] = order[at: at + k]
        at += k
    for g in range(refs_groups):  # kept prefixes: a slot shares the first pages of another
        a, b = 2 * g, 2 * g + 1
        k = int(min(need[a], need[b])) // 2
        table[b, :k] = table[a, :k]
    refs = np.zeros(pages, np.int64)
    np.add.at(refs, table[table >= 0], 1)
    p = dict(pages=pages, width=width, table=table, refs=refs, lengths=by_slot, rows=rows, slots=slots)
    if op == "fork":
        parents = n - case["count"]
        p["src"] = r.integers(0, parents, case["count"])
        p["dst"] = parents + r.permutation(case["count"])
        p["counts"] = np.maximum(1, (held[p["src"]] * r.uniform(0.5, 1.0, case["count"])).astype(np.int64))
    if op == "turnover":
        p["slots"] = r.permutation(n)[: case["count"]]
        p["counts"] = r.integers(case["ctx_min"], case["ctx_max"] + 1, case["count"])
    return p


def visible(case, p):
    """positions that every row sees, summed over the rows; positions that any row of an entry sees, summed"""
    pairs = held = 0
    w = case["window"]
    for n, length in zip(p["rows"], p["lengths"][p["slots"]]):
        first, last = int(length - n), int(length - 1)
        if not w:
            pairs += (first + 1 + last + 1) * int(n) // 2
            held += last + 1
        else:
            cut = min(max(w - 1, first), last + 1)  # rows below see all before them
            pairs += (first + 1 + cut) * (cut - first) // 2 + (last + 1 - cut) * w
            held += last - max(0, first - w + 1) + 1
    return pairs, held


def work(case):
    p = plan(case)
    op = case["op"]
    if op == "attend":
        pairs, held = visible(case, p)
        rows, d = int(p["rows"].sum()), case["head_dim"]
        return {"bytes": 2 * rows * case["q_heads"] * d * 2 + rows * case["q_heads"] * 4
                + held * case["kv_heads"] * d * 2 * 2, "flops": 4 * d * case["q_heads"] * pairs}
    if op == "append":
        rows, d = int(p["rows"].sum()), case["head_dim"]
        return {"bytes": 2 * rows * (case["q_heads"] + 2 * case["kv_heads"]) * d * 2 + rows * d * 4,
                "flops": 3 * rows * (case["q_heads"] + case["kv_heads"]) * d}
    if op == "turnover":
        k, w = case["count"], p["width"]
        return {"bytes": 4 * (4 * k * w + p["pages"] + 4 * k), "flops": 0}
    page = case["layers"] * case["kv_heads"] * 2 * PAGE * case["head_dim"] * 2
    if op == "fork":
        return {"bytes": 2 * int((p["counts"] % PAGE).sum()) * (page // PAGE) + 8 * case["count"] * p["width"]
                + 4 * p["pages"], "flops": 0}
    live = int((p["refs"] > 0).sum())
    return {"bytes": 2 * int((p["refs"][live:] > 0).sum()) * page + 8 * p["table"].size + 12 * p["pages"], "flops": 0}


# ---- what a program holds before the call -------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    p = plan(case)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    op = case["op"]
    ints = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    dtype = getattr(torch, case.get("dtype", "bfloat16"))
    # attention and append work on one layer of several; the pages of a turnover are not touched
    layers, kv_heads, d = case.get("layers", 2), case.get("kv_heads", 1), case.get("head_dim", 64)
    layers = 1 if op == "turnover" else layers
    pool = torch.empty((p["pages"], layers, kv_heads, 2, d // 64, PAGE, 64), dtype=dtype, device=dev)
    pool.normal_(generator=g)
    s = dict(op=op, pool=pool, table=ints(p["table"]), refs=ints(p["refs"]), lengths=ints(p["lengths"]),
             width=p["width"])
    if op in ("attend", "append"):
        start = np.concatenate([[0], np.cumsum(p["rows"])])
        rows, qh = int(start[-1]), case["q_heads"]
        s.update(slots=ints(p["slots"]), q_start=ints(start), max_rows=int(p["rows"].max()), layer=1,
                 window=case["window"], q_heads=qh)
        if op == "attend":
            s["q"] = (1.5 * torch.randn((rows, qh, d), device=dev, generator=g)).to(dtype)
        else:
            s["qkv"] = torch.randn((rows, (qh + 2 * kv_heads) * d), device=dev, generator=g).to(dtype)
            inv = 1.0 / 1e6 ** (torch.arange(d // 2, device=dev, dtype=torch.float32) / (d // 2))
            angle = torch.arange(p["width"] * PAGE, device=dev, dtype=torch.float32)[:, None] * inv
            s.update(cos=torch.cos(angle), sin=torch.sin(angle))
    elif op == "fork":
        s.update(src=ints(p["src"]), dst=ints(p["dst"]), counts=ints(p["counts"]))
    elif op == "compact":
        s.update(table0=s["table"].clone(), refs0=s["refs"].clone())
    else:
        s.update(slots=ints(p["slots"]))
        # other prompts for other seeds, in the same pages
        k = np.random.default_rng(seed).integers(0, PAGE, case["count"])
        s["counts"] = ints(np.minimum(p["counts"] // PAGE * PAGE + 1 + k, p["width"] * PAGE))
    if own:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        from runtime.paged_kv import PagedKVCache

        s["cache"] = PagedKVCache.wrap(pool, s["table"], s["refs"], s["lengths"])
    return s


# ---- one pass ------------------------------------------------------------------------
def run(s):
    op = s["op"]
    if not own:
        return PLAIN[op](s)
    cache = s["cache"]
    if op == "attend":
        out, lse = cache.attend(s["layer"], s["q"], s["slots"], s["q_start"], s["max_rows"], window=s["window"],
                                lse=True)
        return {"out": out, "lse": lse}
    if op == "append":
        q = cache.append(s["layer"], s["qkv"], s["slots"], s["q_start"], s["max_rows"], s["cos"], s["sin"])
        return {"q": q, "pool": s["pool"]}
    if op == "fork":
        cache.fork(s["src"], s["dst"], s["counts"])
        return {"pool": s["pool"], "table": s["table"], "refs": s["refs"], "lengths": s["lengths"]}
    if op == "compact":  # the gaps that the next hour's requests leave
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
        page_map = cache.compact()
        return {"pool": s["pool"], "table": s["table"], "refs": s["refs"], "map": page_map}
    cache.free(s["slots"])
    cache.reserve(s["slots"], s["counts"])
    return {"table": s["table"], "refs": s["refs"], "lengths": s["lengths"]}


# ---- the plain forms -------------------------------------------------------------------
def block_of(device):
    """[64, 8]: where a position's 16-byte blocks are stored"""
    return torch.arange(8, device=device)[None, :] ^ (torch.arange(PAGE, device=device)[:, None] & 7)


def plain_attend(s):
    q, pool, slots, start = s["q"], s["pool"], s["slots"].long(), s["q_start"].long()
    dev, (rows, qh, d) = q.device, q.shape
    b, width, most, kvh = slots.numel(), s["width"], s["max_rows"], pool.shape[2]
    n, length = start[1:] - start[:-1], s["lengths"].long()[slots]
    pages = s["table"].long()[slots]
    kv = pool[:, s["layer"]][pages.clamp(min=0)].view(b, width, kvh, 2, d // 64, PAGE, 8, 8)
    kv = kv[..., torch.arange(PAGE, device=dev)[:, None], block_of(dev), :]
    kv = kv.permute(3, 0, 2, 1, 5, 4, 6, 7).reshape(2, b, kvh, width * PAGE, d)
    i = torch.arange(most, device=dev)
    qp = q[(start[:-1, None] + i).clamp(max=rows - 1)].float()  # [b, most, qh, d]
    qp = qp.view(b, most, kvh, qh // kvh, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, d)
    scores = torch.matmul(qp, kv[0].float().transpose(2, 3)).view(b, kvh, qh // kvh, most, -1)
    scores *= 1.0 / math.sqrt(d)
    at, j = (length - n)[:, None] + i, torch.arange(width * PAGE, device=dev)
    see = (j <= at[..., None]) & (pages >= 0).repeat_interleave(PAGE, dim=1)[:, None, :]
    if s["window"]:
        see &= j > at[..., None] - s["window"]
    scores.masked_fill_(~see[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(b, kvh, -1, width * PAGE), kv[1].float()).view(b, kvh, qh // kvh, most, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total))[..., 0]
    row = torch.arange(rows, device=dev)
    entry = torch.searchsorted(start[1:], row, right=True)
    k = row - start[entry]
    return {"out": out[entry, :, :, k].reshape(rows, qh, d).to(q.dtype), "lse": lse[entry, :, :, k].reshape(rows, qh)}


def plain_append(s):
    qkv, pool, slots, start = s["qkv"], s["pool"], s["slots"].long(), s["q_start"].long()
    dev, rows = qkv.device, qkv.shape[0]
    layers, kvh, d, qh = pool.shape[1], pool.shape[2], pool.shape[4] * 64, s["q_heads"]
    row = torch.arange(rows, device=dev)
    entry = torch.searchsorted(start[1:], row, right=True)
    slot = slots[entry]
    pos = s["lengths"].long()[slot] - (start[entry + 1] - row)
    x = qkv.view(rows, qh + 2 * kvh, d)[:, : qh + kvh].float()
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    lo, hi = x[..., : d // 2], x[..., d // 2:]
    turned = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1).to(qkv.dtype)
    new = torch.stack([turned[:, qh:], qkv.view(rows, qh + 2 * kvh, d)[:, qh + kvh:]], 2)  # [rows, kvh, 2, d]
    page = s["table"].long()[slot, pos // PAGE]
    dim, at = torch.arange(d, device=dev), (pos % PAGE)[:, None]
    inner = (dim // 64 * PAGE + at) * 64 + (((dim % 64) // 8) ^ (at & 7)) * 8 + dim % 8  # [rows, d]
    head = torch.arange(kvh * 2, device=dev)
    base = (page * layers + s["layer"])[:, None] * (kvh * 2) + head
    index = base[..., None] * (PAGE * d) + inner[:, None]
    pool.view(-1)[index.view(rows, kvh, 2, d)] = new
    return {"q": turned[:, :qh], "pool": pool}


def lowest_free(refs, need):
    """[need]: the lowest pages that nobody holds"""
    free = refs == 0
    rank = torch.cumsum(free, 0) - 1
    out = torch.zeros(need + 1, dtype=torch.long, device=refs.device)
    out[torch.where(free & (rank < need), rank, need)] = torch.arange(refs.numel(), device=refs.device)
    return out[:need]


def count_refs(refs, pages, by):
    """refs[pages] += by, where pages >= 0"""
    pages = pages.reshape(-1)
    refs.index_add_(0, pages.clamp(min=0), torch.where(pages >= 0, by, 0).to(refs.dtype))


def plain_fork(s):
    pool, table, refs, lengths = s["pool"], s["table"], s["refs"], s["lengths"]
    src, dst, counts = s["src"].long(), s["dst"].long(), s["counts"].long()
    n, width, dev = src.numel(), table.shape[1], table.device
    whole, rest = counts // PAGE, counts % PAGE
    fresh = lowest_free(refs, n)[(torch.cumsum(rest > 0, 0) - 1).clamp(min=0)]
    w = torch.arange(width, device=dev)
    rows = table.long()[src]
    new = torch.where(w < whole[:, None], rows, -1)
    count_refs(refs, table.long()[dst], -1)
    count_refs(refs, new, 1)
    took = torch.where(rest > 0, fresh, -1)
    count_refs(refs, took, 1)
    new = torch.where((w == whole[:, None]) & (rest > 0)[:, None], took[:, None], new)
    table[dst] = new.int()
    lengths[dst] = counts.int()
    some = (rest > 0).nonzero()[:, 0]
    old = rows[some, whole[some]]
    keep = torch.arange(PAGE, device=dev)[:, None] < rest[some].view(-1, 1, 1, 1, 1, 1, 1)
    pool[took[some]] = torch.where(keep, pool[old], pool[took[some]])
    return {"pool": pool, "table": table, "refs": refs, "lengths": lengths}


def plain_compact(s):
    pool, table, refs = s["pool"], s["table"], s["refs"]
    table.copy_(s["table0"])
    refs.copy_(s["refs0"])
    pages, dev = refs.numel(), refs.device
    live = refs > 0
    index, total = torch.arange(pages, device=dev), live.sum()
    movers, holes = (live & (index >= total)).nonzero()[:, 0], (~live & (index < total)).nonzero()[:, 0]
    pool[holes] = pool[movers]
    page_map = torch.where(live, index, -1)
    page_map[movers] = holes
    refs[holes] = refs[movers]
    refs[movers] = 0
    table.copy_(torch.where(table >= 0, page_map[table.clamp(min=0).long()].int(), table))
    return {"pool": pool, "table": table, "refs": refs, "map": page_map.int()}


def plain_turnover(s):
    table, refs, lengths = s["table"], s["refs"], s["lengths"]
    slots, counts = s["slots"].long(), s["counts"].long()
    count_refs(refs, table.long()[slots], -1)
    need = -(-counts // PAGE)
    w = torch.arange(table.shape[1], device=table.device)
    took = w < need[:, None]
    fresh = lowest_free(refs, refs.numel())
    new = torch.where(took, fresh[((torch.cumsum(need, 0) - need)[:, None] + w).clamp(max=refs.numel() - 1)], -1)
    count_refs(refs, new, 1)
    table[slots] = new.int()
    lengths[slots] = counts.int()
    return {"table": table, "refs": refs, "lengths": lengths}


PLAIN = {"attend": plain_attend, "append": plain_append, "fork": plain_fork, "compact": plain_compact,
         "turnover": plain_turnover}


# ---- the definitions in 64 bits ---------------------------------------------------------
def positions(pool, pages, layer, kind):
    """[kv heads, positions, d] in 64 bits of the pages in order: whole pages a step at a time"""
    x = pool[pages, layer, :, kind].double()  # [pages, kvh, d / 64, 64, 64]
    out = torch.empty_like(x)
    for r in range(8):
        for c in range(8):
            out[..., r::8, c * 8: c * 8 + 8] = x[..., r::8, (c ^ r) * 8: (c ^ r) * 8 + 8]
    return out.permute(1, 0, 3, 2, 4).reshape(x.shape[1], -1, x.shape[2] * 64)


def exact_attend(case, p, s):
    q, d, qh = s["q"].double(), case["head_dim"], case["q_heads"]
    group, w = qh // case["kv_heads"], case["window"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    at = 0
    for n, slot in zip(p["rows"].tolist(), p["slots"].tolist()):
        length = int(p["lengths"][slot])
        pages = torch.from_numpy(p["table"][slot, : -(-length // PAGE)]).to(q.device)
        k = positions(s["pool"], pages, s["layer"], 0)[:, :length]
        v = positions(s["pool"], pages, s["layer"], 1)[:, :length]
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            pos = torch.arange(length - n + lo, length - n + hi, device=q.device)[:, None]
            j = torch.arange(length, device=q.device)[None]
            hidden = (j > pos) | ((j <= pos - w) if w else (j < 0))
            for head in range(qh):
                x = q[at + lo: at + hi, head] @ k[head // group].T / math.sqrt(d)
                x = x.masked_fill(hidden, -math.inf)
                lse[at + lo: at + hi, head] = torch.logsumexp(x, 1)
                out[at + lo: at + hi, head] = torch.softmax(x, 1) @ v[head // group]
        at += n
    return {"out": out, "lse": lse}


def exact_append(case, p, s):
    d, qh, kvh = case["head_dim"], case["q_heads"], case["kv_heads"]
    x = s["qkv"].double().view(-1, qh + 2 * kvh, d)
    start = np.concatenate([[0], np.cumsum(p["rows"])])
    pos = np.concatenate([np.arange(p["lengths"][t] - n, p["lengths"][t]) for n, t in zip(p["rows"], p["slots"])])
    page = np.concatenate([p["table"][t, np.arange(p["lengths"][t] - n, p["lengths"][t]) // PAGE]
                           for n, t in zip(p["rows"], p["slots"])])
    assert len(pos) == start[-1]
    pos, page = torch.from_numpy(pos).to(x.device), torch.from_numpy(page).to(x.device)
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]
    z = torch.complex(x[:, : qh + kvh, : d // 2], x[:, : qh + kvh, d // 2:]) * turn
    turned = torch.cat([z.real, z.imag], -1)
    pool = s["pool"].double()
    for kind, rows in ((0, turned[:, qh:]), (1, x[:, qh + kvh:])):
        for c in range(d // 8):
            block = (c % 8) ^ (pos % 8)
            for e in range(8):
                pool[page, s["layer"], :, kind, c // 8, pos % PAGE, block * 8 + e] = rows[:, :, c * 8 + e]
    return {"q": turned[:, :qh].contiguous(), "pool": pool}


def exact_fork(case, p, s):
    pool, refs = s["pool"], p["refs"].copy()
    free = [i for i in range(p["pages"]) if refs[i] == 0]
    for a, n in zip(p["src"].tolist(), p["counts"].tolist()):
        if n % PAGE:
            pool[free.pop(0), :, :, :, :, : n % PAGE] = pool[int(p["table"][a, n // PAGE]), :, :, :, :, : n % PAGE]
    return {"pool": pool, "table": None, "refs": None, "lengths": None}


def exact_compact(case, p, s):
    pool = s["pool"]
    live = int((p["refs"] > 0).sum())
    holes = [i for i in range(live) if p["refs"][i] == 0]
    for i in range(live, p["pages"]):
        if p["refs"][i] > 0:
            pool[holes.pop(0)] = pool[i]
    return {"pool": pool, "table": None, "refs": None, "map": None}


def exact(case, seed):
    form = {"attend": exact_attend, "append": exact_append, "fork": exact_fork, "compact": exact_compact}
    if case["op"] not in form:
        return None  # whole numbers alone
    return form[case["op"]](case, plan(case), prepare(case, seed))
