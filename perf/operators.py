"""Operators of a serving step over a paged cache of keys and values in 8 bits, with the inputs, the sizes and the
plain forms they are measured against.

tables     block tables and slot maps of a batch of requests, from their lengths
write      new keys and values into the cache: e4m3 codes, one power-of-two scale for each page and head
attention  queries against the cache through the block tables, causal, grouped heads, ragged batches
matvec     y = x W^T with W in 4 bits, a scale (and a zero point) for each group of columns

A cache page holds `page` consecutive tokens of one request: codes [pages, kv heads, page, head dim], scales
[pages, kv heads]; a value is code * scale.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls the framework's operators; False: their plain forms

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3_MAX = 448.0
MIN_EXPONENT = -64  # of a page's scale

# ------------------------------------------------------------------------------------------------ the cases


def listed():
    return [
        # One decoding step of a full server: every request adds a token, one in sixteen needs a page.
        dict(name="tables: a step of 256", op="tables", requests=256, cached=8192, added=1, page=16, short=False),
        # Prompts admitted together behind a shared prefix; ragged, thousands of new pages.
        dict(name="tables: 48 prompts", op="tables", requests=48, cached=2048, added=4096, page=64, short=False),
        # The same decoding step's keys and values: one token a request, into pages that are partly full.
        dict(name="write: a step of 256", op="write", requests=256, added=1, kv_heads=8, dim=128, page=16, type="bf16"),
        # Prompts' keys and values: whole pages, first and last ones partial.
        dict(name="write: 8 prompts", op="write", requests=8, added=4096, kv_heads=8, dim=64, page=64, type="f16"),
        # The smallest call: one user, a short context; latency.
        dict(name="attention: one request", op="attention", requests=1, length=700, queries=1, q_heads=32, kv_heads=8, dim=128, page=16, type="bf16"),
        # An ordinary batch of decoding requests, ragged.
        dict(name="attention: 64 requests", op="attention", requests=64, length=8192, queries=1, q_heads=32, kv_heads=8, dim=128, page=64, type="bf16"),
        # Few requests with very long contexts: the work has to be split along the keys.
        dict(name="attention: 3 long contexts", op="attention", requests=3, length=262144, queries=1, q_heads=64, kv_heads=8, dim=128, page=128, type="f16"),
        # Drafted tokens checked together, a head of keys for each head of queries, wide heads.
        dict(name="attention: 32 drafts", op="attention", requests=32, length=2500, queries=5, q_heads=16, kv_heads=16, dim=256, page=16, type="f16"),
        # Pieces of prompts against what the cache holds of them: bound by arithmetic.
        dict(name="attention: 6 prompt pieces", op="attention", requests=6, length=6000, queries=509, q_heads=16, kv_heads=4, dim=64, page=32, type="bf16"),
        # One token through a square projection: latency.
        dict(name="matvec: 1 x 4096 x 4096", op="matvec", rows=1, n=4096, k=4096, group=128, zeros=False, type="bf16"),
        # A small batch, an odd number of outputs, zero points.
        dict(name="matvec: 13 x 10001 x 8192", op="matvec", rows=13, n=10001, k=8192, group=64, zeros=True, type="f16"),
        # One token through a large feed-forward projection: the weights' 4 bits are all there is.
        dict(name="matvec: 1 x 28672 x 8192", op="matvec", rows=1, n=28672, k=8192, group=128, zeros=True, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of these ranges; the work of the largest listed one bounds it."""
    op = rng.choice(["tables", "write", "attention", "attention", "matvec"])
    if op == "tables":
        requests = _log(rng, 1, 2048)
        return dict(op=op, requests=requests, cached=_log(rng, 1, 32768), added=_log(rng, 1, max(1, min(16384, 262144 // requests))),
                    page=rng.choice([16, 32, 64, 128]), short=rng.random() < 0.25)
    if op == "write":
        requests = _log(rng, 1, 512)
        return dict(op=op, requests=requests, added=_log(rng, 1, max(1, min(8192, 16384 // requests))), kv_heads=rng.randint(1, 16),
                    dim=rng.choice([64, 128, 192, 256]), page=rng.choice([16, 32, 64, 128]), type=rng.choice(["bf16", "f16"]))
    if op == "attention":
        requests, kv_heads, dim = _log(rng, 1, 128), rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 128, 192, 256])
        group = rng.choice([1, 2, 3, 4, 6, 8, 16])
        # what the longest listed case holds bounds keys and values; the products bound the queries
        length = min(262144, max(64, 402_000_000 // (requests * kv_heads * dim)))
        length = _log(rng, 17, length)
        queries = 1 if rng.random() < 0.6 else _log(rng, 2, max(2, min(600, 28_000_000_000 // (requests * kv_heads * group * length * dim))))
        return dict(op=op, requests=requests, length=length, queries=min(queries, length), q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128]), type=rng.choice(["bf16", "f16"]))
    group = rng.choice([32, 64, 128])
    n = _log(rng, 65, 28672)
    k = group * _log(rng, 2, min(28672, 230_000_000 // n) // group)
    return dict(op=op, rows=_log(rng, 1, 64), n=n, k=k, group=group, zeros=rng.random() < 0.5, type=rng.choice(["bf16", "f16"]))


# ------------------------------------------------------------------------------------------------ inputs


class State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(1_000_003 * (seed + 1))
    return g


def _int32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)


def _normal(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * sigma).to(dtype)


def _ragged(rs, b, *ranges):
    """An array of b whole numbers for each range [lo, hi): the same tuples in every batch of a case, so that outputs keep their shapes, in an order of the seed's."""
    fixed, order = np.random.RandomState(5), rs.permutation(b)
    return [fixed.randint(lo, hi, b)[order] for lo, hi in ranges]


def _pages_of(tokens, page):
    return (tokens + page - 1) // page


def _tables_inputs(c, rs):
    b, page = c["requests"], c["page"]
    cached, added = _ragged(rs, b, (0, c["cached"] + 1), (1, c["added"] + 1))
    if b >= 8:
        added[added.argmin()] = 0  # a request that only fills the batch
    before, after = _pages_of(cached, page), _pages_of(cached + added, page)
    width = int(_pages_of(c["cached"] + c["added"], page))
    need = int((after - before).sum())
    held = int(before.sum())
    order = rs.permutation(held + need + 64)
    table = np.full((b, width), -1, dtype=np.int32)
    table[np.arange(width)[None, :] < before[:, None]] = order[:held]
    free = order[held:]
    count = need // 2 if c["short"] else len(free)
    tokens = int(added.sum()) + 17  # the slot map is longer than what is added, as in a captured step
    return State(op="tables", page=page, cached=_int32(cached), added=_int32(added), free=_int32(free), count=_int32([count]),
                 table=_int32(table), lengths=torch.zeros(b, dtype=torch.int32, device=DEVICE),
                 starts=torch.zeros(b + 1, dtype=torch.int32, device=DEVICE),
                 slots=torch.zeros(tokens, dtype=torch.int32, device=DEVICE), counts=torch.zeros(2, dtype=torch.int32, device=DEVICE))


def _codes(x, scales):
    """e4m3 codes of x [pages, heads, page, dim] under its pages' scales."""
    return (x / scales[:, :, None, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _scale_of(amax):
    """The smallest power of two that brings amax within the range of e4m3."""
    f, e = torch.frexp(amax.float())
    e = torch.where(f > 0.875, e - 8, e - 9).clamp_(min=MIN_EXPONENT)
    return torch.ldexp(torch.ones_like(f), torch.where(amax > 0, e, torch.full_like(e, MIN_EXPONENT)))


def _cache(g, pages, heads, page, dim, used):
    """Codes and scales of random keys or values; pages that no request holds are full of NaN."""
    codes = torch.full((pages, heads, page, dim), 0x7F, dtype=torch.uint8, device=DEVICE)
    scales = torch.full((pages, heads), float("inf"), device=DEVICE)
    for lo in range(0, len(used), 4096):  # in pieces: the fp32 values of a long cache are four times its size
        at = used[lo:lo + 4096]
        x = torch.randn((len(at), heads, page, dim), generator=g, device=DEVICE) * torch.exp(0.5 * torch.randn((len(at), heads, 1, 1), generator=g, device=DEVICE))
        s = _scale_of(x.abs().amax(dim=(2, 3)))
        codes[at], scales[at] = _codes(x, s).view(torch.uint8), s
    return codes.view(torch.float8_e4m3fn), scales


def _write_inputs(c, rs, g):
    b, page, heads, dim, dtype = c["requests"], c["page"], c["kv_heads"], c["dim"], TYPES[c["type"]]
    cached, added = _ragged(rs, b, (0, 4 * page), (1, c["added"] + 1))
    first, last = cached // page, _pages_of(cached + added, page)
    pages = int((last - first).sum()) + 64
    order, at, slots = rs.permutation(pages), 0, []
    for i in range(b):
        mine = order[at:at + last[i] - first[i]]
        at += len(mine)
        pos = np.arange(cached[i], cached[i] + added[i])
        slots.append(mine[pos // page - first[i]].astype(np.int64) * page + pos % page)
    slots = np.concatenate(slots + [np.full(5, -1)])
    tokens = len(slots)
    kv = _normal(g, (tokens, 2, heads, dim), dtype) * torch.exp(0.5 * torch.randn((tokens, 2, heads, 1), generator=g, device=DEVICE)).to(dtype)
    used = torch.arange(pages, device=DEVICE)
    kc, ks = _cache(g, pages, heads, page, dim, used)
    vc, vs = _cache(g, pages, heads, page, dim, used)
    return State(op="write", page=page, dim=dim, type=c["type"], k=kv[:, 0], v=kv[:, 1], slots=_int32(slots), k_cache=kc, v_cache=vc, k_scales=ks, v_scales=vs)


def _attention_inputs(c, rs, g):
    b, page, heads, dim, dtype = c["requests"], c["page"], c["kv_heads"], c["dim"], TYPES[c["type"]]
    lengths, queries = _ragged(rs, b, (max(1, c["length"] // 2), c["length"] + 1), (1, c["queries"] + 1))
    queries = np.minimum(queries, lengths)
    if b >= 8:
        lengths[queries.argmin()] = 0  # a request that only fills the batch: nothing to attend to
    width = int(_pages_of(c["length"], page)) + 1
    held = _pages_of(lengths, page)
    order = rs.permutation(int(held.sum()) + 16)
    table = np.full((b, width), -1, dtype=np.int32)
    table[np.arange(width)[None, :] < held[:, None]] = order[:int(held.sum())]
    used = torch.from_numpy(np.sort(order[:int(held.sum())])).to(DEVICE)
    kc, ks = _cache(g, len(order), heads, page, dim, used)
    vc, vs = _cache(g, len(order), heads, page, dim, used)
    starts = np.concatenate([[0], np.cumsum(queries)])
    tokens = int(starts[-1])
    qkv = _normal(g, (tokens, c["q_heads"] + 2 * heads, dim), dtype)  # queries stand in the fused projection's output
    return State(op="attention", page=page, dim=dim, type=c["type"], q=qkv[:, :c["q_heads"]], k_cache=kc, v_cache=vc, k_scales=ks, v_scales=vs,
                 table=_int32(table), lengths=_int32(lengths), starts=_int32(starts), scale=1.0 / math.sqrt(dim), queries=c["queries"], length=c["length"],
                 out=torch.zeros((tokens, c["q_heads"], dim), dtype=dtype, device=DEVICE))


def _matvec_inputs(c, rs, g):
    rows, n, k, group, dtype = c["rows"], c["n"], c["k"], c["group"], TYPES[c["type"]]
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEVICE, dtype=torch.uint8)
    scales = ((0.5 + torch.rand((k // group, n), generator=g, device=DEVICE)) * 0.01).to(dtype)
    zeros = torch.randint(5, 11, (k // group, n), generator=g, device=DEVICE, dtype=torch.uint8) if c["zeros"] else None
    return State(op="matvec", group=group, type=c["type"], x=_normal(g, (rows, k), dtype), codes=codes, scales=scales, zeros=zeros,
                 y=torch.zeros((rows, n), dtype=dtype, device=DEVICE))


def _inputs(c, seed):
    rs = np.random.RandomState((977 * seed + 11) % 2**32)
    if c["op"] == "tables":
        return _tables_inputs(c, rs)
    return {"write": _write_inputs, "attention": _attention_inputs, "matvec": _matvec_inputs}[c["op"]](c, rs, _generator(seed))


_handles = {}  # the pipelines of this program, by what they were created for


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import gern_amd

        make = {"tables": lambda: gern_amd.PageTable(page_size=s.page),
                "write": lambda: gern_amd.CacheWrite(head_dim=s.dim, page_size=s.page, dtype=s.type),
                "attention": lambda: gern_amd.CacheAttention(head_dim=s.dim, page_size=s.page, dtype=s.type),
                "matvec": lambda: gern_amd.Matvec4(group=s.group, dtype=s.type)}[s.op]
        key = (s.op,) + tuple(case.get(n) for n in ("dim", "page", "type", "group"))
        if key not in _handles:
            _handles[key] = make()
        s.handle = _handles[key]
        if s.op == "attention":
            s.workspace = torch.empty(s.handle.workspace_bytes(tokens=s.q.shape[0], requests=s.lengths.shape[0], q_heads=s.q.shape[1], kv_heads=s.k_cache.shape[1],
                                                               max_queries=s.queries, max_length=s.length), dtype=torch.uint8, device=DEVICE)
    return s


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    if s.op == "tables":
        if own:
            s.handle(s.cached, s.added, s.free, s.count, s.table, s.lengths, s.starts, s.slots, s.counts)
            return dict(table=s.table, lengths=s.lengths, starts=s.starts, slots=s.slots, counts=s.counts)
        return _plain_tables(s)
    if s.op == "write":
        if own:
            s.handle(s.k, s.v, s.slots, s.k_cache, s.v_cache, s.k_scales, s.v_scales)
        else:
            _plain_write(s.k, s.slots, s.k_cache, s.k_scales, s.page)
            _plain_write(s.v, s.slots, s.v_cache, s.v_scales, s.page)
        return dict(k_cache=s.k_cache, v_cache=s.v_cache, k_scales=s.k_scales, v_scales=s.v_scales)
    if s.op == "attention":
        if own:
            return s.handle(s.q, s.k_cache, s.v_cache, s.k_scales, s.v_scales, s.table, s.lengths, s.starts, s.out, s.scale, max_queries=s.queries,
                            max_length=s.length, workspace=s.workspace)
        return _plain_attention(s)
    if own:
        return s.handle(s.x, s.codes, s.scales, s.y, zeros=s.zeros)
    return _plain_matvec(s)


def _plain_tables(s):
    """New pages are taken from the end of the free list, request by request; a page that the list no longer has is -1, as are its tokens' slots."""
    page = s.page
    lengths = s.cached + s.added
    before, after = (s.cached + page - 1) // page, (lengths + page - 1) // page
    need = after - before
    first = torch.cumsum(need, 0) - need
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEVICE), torch.cumsum(s.added, 0)])
    j = torch.arange(s.table.shape[1], device=DEVICE)[None, :]
    at = s.count - 1 - (first[:, None] + j - before[:, None])
    fresh = torch.where(at >= 0, s.free[at.clamp(0, s.free.shape[0] - 1)], torch.full_like(at, -1).int())
    table = torch.where((j >= before[:, None]) & (j < after[:, None]), fresh, s.table)
    t = torch.arange(s.slots.shape[0], device=DEVICE)
    b = torch.searchsorted(starts[1:], t, right=True)
    there = b < lengths.shape[0]
    b = b.clamp(max=lengths.shape[0] - 1)
    pos = s.cached[b] + t - starts[b]
    held = table[b, (pos // page).clamp(0, table.shape[1] - 1)]
    slots = torch.where(there & (held >= 0), held * page + pos % page, torch.full_like(pos, -1))
    total = need.sum()
    counts = torch.stack([(s.count[0] - total).clamp(min=0), (total - s.count[0]).clamp(min=0)])
    return dict(table=table, lengths=lengths, starts=starts.int(), slots=slots.int(), counts=counts.int())


def _plain_write(x, slots, cache, scales, page):
    """A page's scale is the smallest power of two for what the page holds already and what is added; codes that are there move to the new scale."""
    x, slots = x.float(), slots.long()
    ok = slots >= 0
    at = torch.where(ok, slots // page, torch.full_like(slots, cache.shape[0]))  # what is not stored goes to a page behind the last
    amax = torch.zeros((cache.shape[0] + 1, cache.shape[1]), device=DEVICE)
    amax.index_reduce_(0, at, x.abs().amax(dim=2), "amax")
    low = torch.full((cache.shape[0] + 1,), page, dtype=torch.int64, device=DEVICE).index_reduce_(0, at, slots % page, "amin")[:-1]
    touched = low < page
    fresh = _scale_of(amax[:-1])
    new = torch.where((low > 0)[:, None], torch.maximum(scales, fresh), fresh)
    new = torch.where(touched[:, None], new, scales)
    old = torch.arange(page, device=DEVICE)[None, :] < low[:, None]
    pages = touched.nonzero()[:, 0]
    moved = (cache[pages].float() * (scales[pages] / new[pages])[:, :, None, None]).to(torch.float8_e4m3fn)
    keep = old[pages][:, None, :, None]
    raw = cache.view(torch.uint8)
    raw[pages] = torch.where(keep, moved.view(torch.uint8), raw[pages])
    scales.copy_(new)
    t = ok.nonzero()[:, 0]
    to = slots[t]
    raw[to // page, :, to % page] = (x[t] / new[to // page][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def _gathered(cache, scales, pages, there):
    """[requests, heads, tokens, dim] in fp32, zero where there is no token."""
    b, w = pages.shape
    _, heads, page, dim = cache.shape
    x = cache.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * scales[pages][:, :, :, None, None]
    x = x.permute(0, 2, 1, 3, 4).reshape(b, heads, w * page, dim)
    return torch.where(there[:, None, :, None], x, torch.zeros((), device=DEVICE))


def _plain_attention(s):
    tokens, q_heads, dim = s.q.shape
    b, kv_heads, page = s.lengths.shape[0], s.k_cache.shape[1], s.page
    group, w = q_heads // kv_heads, (s.length + page - 1) // page
    lengths, starts = s.lengths.long(), s.starts.long()
    key = torch.arange(w * page, device=DEVICE)
    there = key[None, :] < lengths[:, None]
    pages = s.table[:, :w].long().clamp(min=0)
    k, v = _gathered(s.k_cache, s.k_scales, pages, there), _gathered(s.v_cache, s.v_scales, pages, there)
    t = torch.arange(tokens, device=DEVICE)
    of = torch.searchsorted(starts[1:], t, right=True)
    at = t - starts[of]
    q = torch.zeros((b, s.queries, q_heads, dim), device=DEVICE)
    q[of, at] = s.q.float()
    q = q.reshape(b, s.queries, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(b, kv_heads, s.queries * group, dim)
    scores = torch.matmul(q, k.transpose(2, 3)) * s.scale
    # query i of n sees the keys up to length - n + i
    last = lengths[:, None] - (starts[1:] - starts[:-1])[:, None] + torch.arange(s.queries, device=DEVICE)[None, :]
    seen = there[:, None, :] & (key[None, None, :] <= last[:, :, None])
    seen = seen[:, None, :, None, :].expand(b, kv_heads, s.queries, group, w * page).reshape(b, kv_heads, s.queries * group, w * page)
    scores = scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(dim=3, keepdim=True)
    p = torch.exp_(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(dim=3, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.reshape(b, kv_heads, s.queries, group, dim).permute(0, 2, 1, 3, 4).reshape(b, s.queries, q_heads, dim)
    return out[of, at].to(s.q.dtype)


def _plain_matvec(s):
    n, half = s.codes.shape
    q = torch.stack([s.codes & 15, s.codes >> 4], dim=2).reshape(n, half * 2 // s.group, s.group).float()
    zero = 8.0 if s.zeros is None else s.zeros.t().float()[:, :, None]
    w = ((q - zero) * s.scales.t().float()[:, :, None]).reshape(n, half * 2)
    return torch.matmul(s.x.float(), w.t()).to(s.x.dtype)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "tables":
        # lengths in and out; half of the ragged additions on average
        b, tokens = c["requests"], c["requests"] * (c["added"] + 1) / 2
        return {"bytes": 4 * (4 * b + tokens + 3 * (tokens / c["page"])), "flops": 2 * b + 4 * tokens}
    if c["op"] == "write":
        tokens = c["requests"] * (c["added"] + 1) / 2 if c["added"] > 1 else c["requests"]
        return {"bytes": tokens * (2 * c["kv_heads"] * c["dim"] * 3 + 4) + 4 * 4 * c["kv_heads"] * (tokens / c["page"] + c["requests"]),
                "flops": 2 * tokens * c["kv_heads"] * c["dim"] * 2}
    if c["op"] == "attention":
        keys = 0.75 * c["length"] * c["requests"]
        q = c["requests"] * (c["queries"] + 1) / 2
        # the last query of a request sees every key, the first one all but the others' own
        seen = q * max(0.75 * c["length"] - c["queries"] / 4, 1)
        return {"bytes": 2 * keys * c["kv_heads"] * (c["dim"] + 4 / c["page"]) + 2 * q * c["q_heads"] * c["dim"] * 2, "flops": 4 * seen * c["q_heads"] * c["dim"]}
    groups = c["k"] // c["group"]
    return {"bytes": c["n"] * c["k"] / 2 + c["n"] * groups * (3 if c["zeros"] else 2) + 2 * c["rows"] * (c["n"] + c["k"]), "flops": 2 * c["rows"] * c["n"] * c["k"]}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    return {"tables": _exact_tables, "write": _exact_write, "attention": _exact_attention, "matvec": _exact_matvec}[s.op](s)


def _exact_tables(s):
    cached, added, free = s.cached.cpu().numpy(), s.added.cpu().numpy(), s.free.cpu().numpy()
    table, page, left = s.table.cpu().numpy().copy(), s.page, int(s.count.cpu()[0])
    missing, starts, slots = 0, [0], []
    for b in range(len(cached)):
        for pos in range(int(cached[b]), int(cached[b] + added[b])):
            if pos % page == 0:
                if left > 0:
                    left -= 1
                    table[b, pos // page] = free[left]
                else:
                    missing += 1
                    table[b, pos // page] = -1
            held = int(table[b, pos // page])
            slots.append(held * page + pos % page if held >= 0 else -1)
        starts.append(len(slots))
    slots += [-1] * (s.slots.shape[0] - len(slots))
    return dict(table=table, lengths=cached + added, starts=np.array(starts, dtype=np.int32), slots=np.array(slots, dtype=np.int32),
                counts=np.array([left, missing], dtype=np.int32))


def _round_e4m3(x):
    """The nearest value with 3 bits behind the leading one, ties to even, a step of 2^-9 at least, 448 at most."""
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 4, -9).astype(np.float64))
    return np.clip(np.rint(x / step) * step, -E4M3_MAX, E4M3_MAX)


def _exact_write_one(x, slots, codes, scales, page):
    codes, scales = codes.float().cpu().numpy().astype(np.float64), scales.double().cpu().numpy()
    x, slots = x.double().cpu().numpy(), slots.cpu().numpy()
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        p, low, n = slots[t] // page, slots[t] % page, 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and low + n < page:
            n += 1
        new = x[t:t + n].transpose(1, 0, 2)  # [heads, tokens, dim]
        exponent = np.ceil(np.log2(np.maximum(np.abs(new).max(axis=(1, 2)), 1e-300) / E4M3_MAX))
        need = np.exp2(np.maximum(exponent, MIN_EXPONENT))
        scale = np.maximum(scales[p], need) if low > 0 else need
        codes[p, :, :low] = _round_e4m3(codes[p, :, :low] * (scales[p] / scale)[:, None, None])
        codes[p, :, low:low + n] = _round_e4m3(new / scale[:, None, None])
        scales[p] = scale
        t += n
    return codes, scales


def _exact_write(s):
    kc, ks = _exact_write_one(s.k, s.slots, s.k_cache, s.k_scales, s.page)
    vc, vs = _exact_write_one(s.v, s.slots, s.v_cache, s.v_scales, s.page)
    return dict(k_cache=kc, v_cache=vc, k_scales=ks, v_scales=vs)


def _exact_attention(s):
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    lengths, starts, heads = s.lengths.tolist(), s.starts.tolist(), s.k_cache.shape[1]
    group, dim = s.q.shape[1] // heads, s.q.shape[2]
    for b, n in enumerate(lengths):
        m = starts[b + 1] - starts[b]
        if n == 0 or m == 0:
            continue
        pages = s.table[b, :_pages_of(n, s.page)].long()
        limit = n - m + torch.arange(m, device=DEVICE)
        hidden = (torch.arange(n, device=DEVICE)[None, :] > limit[:, None])[:, None, :]
        for h in range(heads):
            k = (s.k_cache.view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).double() * s.k_scales[pages, h].double()[:, None, None]).reshape(-1, dim)[:n]
            v = (s.v_cache.view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).double() * s.v_scales[pages, h].double()[:, None, None]).reshape(-1, dim)[:n]
            q = s.q[starts[b]:starts[b + 1], h * group:(h + 1) * group].double()
            z = (torch.mm(q.reshape(-1, dim), k.t()) * s.scale).reshape(m, group, n).masked_fill(hidden, float("-inf"))
            out[starts[b]:starts[b + 1], h * group:(h + 1) * group] = torch.mm(torch.softmax(z, dim=2).reshape(-1, n), v).reshape(m, group, dim)
    return out


def _exact_matvec(s):
    y = torch.zeros(s.y.shape, dtype=torch.float64, device=DEVICE)
    for j in range(s.scales.shape[0]):  # group by group: y += scale * (sum of x q - zero * sum of x)
        x = s.x[:, j * s.group:(j + 1) * s.group].double()
        packed = s.codes[:, j * s.group // 2:(j + 1) * s.group // 2]
        dots = torch.mm(x[:, 0::2], (packed % 16).double().t()) + torch.mm(x[:, 1::2], (packed // 16).double().t())
        zero = torch.full_like(s.scales[j], 8, dtype=torch.float64) if s.zeros is None else s.zeros[j].double()
        y += s.scales[j].double()[None, :] * (dots - zero[None, :] * x.sum(dim=1, keepdim=True))
    return y
