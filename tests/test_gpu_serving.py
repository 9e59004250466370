"""The operators of a serving step on the device, against tests/serving_oracle.py."""
import numpy as np
import pytest

import serving_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the gpu-marked tests must run on an MI355X box")
    return torch


@pytest.fixture(scope="module")
def gpu():
    """Pipelines of gern_amd, each made once."""
    import gern_amd
    made = {}

    def make(name, **kw):
        key = (name,) + tuple(sorted(kw.items()))
        if key not in made:
            made[key] = getattr(gern_amd, name)(**kw)
        return made[key]
    make.error = gern_amd.GernError
    return make


def i32(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


# ------------------------------------------------------------------------------------------------ block tables

def run_tables(torch, gpu, cached, added, page, width, count, tokens, seed=0, capacity=None):
    rs = np.random.RandomState(seed)
    cached, added = (np.asarray(a, dtype=np.int64) for a in (cached, added))
    n = len(cached)
    held = -(-np.maximum(cached, 0) // page)
    order = rs.permutation(int(held.sum()) + max(count, capacity or 0))
    table = np.full((n, width), -7, dtype=np.int32)
    at = 0
    for b in range(n):
        table[b, :held[b]] = order[at:at + held[b]][:width]
        at += held[b]
    free = order[at:]
    want = so.tables(cached, added, free, min(count, len(free)), table, page, tokens)
    t = dict(table=i32(torch, table), lengths=i32(torch, np.full(n, -9)), starts=i32(torch, np.full(n + 1, -9)), slots=i32(torch, np.full(tokens, -9)),
             counts=i32(torch, [-9, -9]))
    gpu("PageTable", page_size=page)(i32(torch, cached), i32(torch, added), i32(torch, free), i32(torch, [count]), **t)
    torch.cuda.synchronize()
    for name, w in want.items():
        assert np.array_equal(t[name].cpu().numpy(), w), name


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1023, 1024, 1025, 8192])
@pytest.mark.parametrize("page", [16, 128])
def test_tables(torch, gpu, n, page):
    rs = np.random.RandomState(n)
    most = 3 * page if n < 1000 else 5
    cached, added = rs.randint(0, 4 * page, n), rs.randint(0, most + 1, n)
    run_tables(torch, gpu, cached, added, page, width=8, count=8 * n + 3, tokens=int(added.sum()) + n % 3, seed=n)


@pytest.mark.parametrize("cached, added", [([], []), ([0], [0]), ([0], [1]), ([16], [1]), ([15], [1]), ([15], [2]), ([0, 0, 0], [0, 0, 0]), ([5, 0, 7], [0, 40, 0]),
                                           ([-3, 4], [2, -5]), ([1], [100_000])])
def test_tables_of_few_requests(torch, gpu, cached, added):
    cached, added = np.array(cached), np.array(added)
    run_tables(torch, gpu, cached, added, 16, width=7000, count=7000, tokens=int(np.maximum(added, 0).sum()) + 5)


def test_tables_pages_run_out(torch, gpu):
    cached, added = np.array([3, 0, 31, 16]), np.array([40, 33, 2, 1])
    for count in range(0, 9):
        run_tables(torch, gpu, cached, added, 16, width=6, count=count, tokens=80, capacity=9)
    # more free pages claimed than the list holds
    run_tables(torch, gpu, cached, added, 16, width=6, count=5, tokens=80)


def test_tables_narrow_table_and_short_slot_map(torch, gpu):
    cached, added = np.array([3, 30, 50]), np.array([60, 1, 20])
    run_tables(torch, gpu, cached, added, 16, width=3, count=20, tokens=200)
    run_tables(torch, gpu, cached, added, 16, width=3, count=20, tokens=37)
    run_tables(torch, gpu, cached, added, 16, width=9, count=20, tokens=0)


# ------------------------------------------------------------------------------------------------ writing the cache

E4M3 = so.e4m3_table()


def fresh_cache(torch, rs, pages, heads, page, dim, exponents=(-3, 3)):
    """(codes on the device, scales on the device, values of the codes, scales)."""
    codes = rs.randint(0, 256, (pages, heads, page, dim)).astype(np.uint8)
    codes[(codes & 127) == 127] = 8
    scales = np.exp2(rs.randint(*exponents, (pages, heads))).astype(np.float32)
    return torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), E4M3[codes], scales


def run_write(torch, gpu, x, y, slots, cache, dtype, page, dim, faults=0):
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    w = gpu("CacheWrite", head_dim=dim, page_size=page, dtype=dtype)
    kx, vx = (torch.from_numpy(a).to(t) for a in (x, y))
    (kc, ks, kv, kss), (vc, vs, vv, vss) = cache
    # a token's heads stand inside a wider row, as in the output of a fused projection
    n, heads, _ = x.shape
    rows = torch.zeros((n, 3, heads, dim), dtype=t, device="cuda")
    rows[:, 0], rows[:, 2] = kx.cuda(), vx.cuda()
    w(rows[:, 0], rows[:, 2], i32(torch, slots), kc.view(torch.float8_e4m3fn), vc, ks, vs)
    torch.cuda.synchronize()
    assert w.faults() == faults
    for got, scale, (codes, scales), src in ((kc, ks, (kv, kss), kx), (vc, vs, (vv, vss), vx)):
        want, want_scales = so.write(src.double().numpy(), slots, codes, scales)
        assert np.array_equal(scale.cpu().numpy(), want_scales)
        # equal as values (a zero may have either sign), NaN for NaN; nothing else is touched
        assert np.array_equal(E4M3[got.cpu().numpy()], want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim, page, heads, runs", [
    (64, 16, 1, [(0, 0, 1)]), (128, 16, 8, [(2, 15, 1), (0, 3, 1), (1, 0, 1)]), (192, 32, 3, [(0, 5, 27), (3, 0, 32), (1, 0, 7)]),
    (256, 128, 2, [(1, 100, 28), (0, 0, 128), (2, 0, 1)]), (64, 64, 5, [(0, 63, 1), (2, 0, 64), (1, 0, 64), (3, 0, 63)])])
def test_write(torch, gpu, dtype, dim, page, heads, runs):
    rs = np.random.RandomState(dim + page)
    slots = np.concatenate([p * page + np.arange(a, a + n) for p, a, n in runs] + [np.array([-1, -1])])
    x, y = (rs.normal(size=(len(slots), heads, dim)) * np.exp(rs.normal(size=(len(slots), heads, 1))) * s for s in (1.0, 300.0))
    cache = [fresh_cache(torch, rs, 5, heads, page, dim) for _ in range(2)]
    run_write(torch, gpu, x, y, slots, cache, dtype, page, dim)


def test_write_many_tokens(torch, gpu):
    """More than one page a workgroup: runs that begin in one stretch of tokens and end in the next."""
    rs = np.random.RandomState(3)
    dim, page, heads = 64, 16, 16
    slots = np.concatenate([p * page + np.arange(a, e) for p, (a, e) in enumerate(zip(rs.randint(0, 16, 200), rs.randint(1, 17, 200))) if a < e] + [[-1]])
    assert len(slots) * heads * 2 > 16384
    x, y = rs.normal(size=(2, len(slots), heads, dim)) * 5
    cache = [fresh_cache(torch, rs, 200, heads, page, dim) for _ in range(2)]
    run_write(torch, gpu, x, y, slots, cache, "bf16", page, dim)


def test_write_borders(torch, gpu):
    """Zeros, halves between codes, the largest value at the border of a scale, tiny and huge values, NaN and infinities."""
    rs = np.random.RandomState(5)
    dim, page = 64, 16
    x = np.zeros((9, 1, dim))
    x[1, 0, :2] = [448.0, 17.0]
    x[2, 0, :2] = [450.0, 18.0]          # the next scale
    x[3, 0, :] = np.arange(dim) / 512 / 2  # halves of the smallest step: ties to even
    x[3, 0, 0] = 448.0
    x[4, 0, :3] = [np.inf, -np.inf, 3.0]
    x[5, 0, :3] = [np.nan, 1.0, -2.0]
    x[6, 0, :2] = [3e38, -1e-38]
    x[7, 0, :2] = [2.0 ** -100, 2.0 ** -56]  # under the smallest scale's range
    x[8] = (16 + np.arange(dim)) * 0.5     # ties between codes
    x[8, 0, 0] = 448.0
    slots = np.arange(9) * page + np.array([0, 0, 0, 0, 0, 0, 0, 0, 0])
    cache = [fresh_cache(torch, rs, 9, 1, page, dim) for _ in range(2)]
    run_write(torch, gpu, x, -x, slots, cache, "bf16", page, dim)


def test_write_scale_moves_earlier_codes(torch, gpu):
    """Tokens one at a time into a page; the scale grows, stays, and an older scale that is no power of two is kept."""
    rs = np.random.RandomState(6)
    dim, page, heads = 128, 16, 2
    kc, ks, kv, kss = fresh_cache(torch, rs, 1, heads, page, dim)
    vc, vs, vv, vss = fresh_cache(torch, rs, 1, heads, page, dim)
    for place in range(page):
        x, y = rs.normal(size=(2, 1, heads, dim)) * 4.0 ** (place % 5)
        run_write(torch, gpu, x, y, np.array([place]), [(kc, ks, kv, kss), (vc, vs, vv, vss)], "bf16", page, dim)
        kv, kss, vv, vss = E4M3[kc.cpu().numpy()], ks.cpu().numpy(), E4M3[vc.cpu().numpy()], vs.cpu().numpy()
    ks.fill_(1000.0)
    kss = ks.cpu().numpy()
    x, y = rs.normal(size=(2, 1, heads, dim))
    x32 = torch.from_numpy(x).bfloat16().float().numpy()
    w = gpu("CacheWrite", head_dim=dim, page_size=page, dtype="bf16")
    before = kc.clone()
    w(torch.from_numpy(x).bfloat16().cuda(), torch.from_numpy(y).bfloat16().cuda(), i32(torch, [7]), kc, vc, ks, vs)
    torch.cuda.synchronize()
    assert np.array_equal(ks.cpu().numpy(), kss) and torch.equal(kc[:, :, :7], before[:, :, :7])
    # fp32 division, rounded once more
    assert np.array_equal(E4M3[kc[0, :, 7].cpu().numpy()], so.e4m3_round((x32[0] / np.float32(1000.0)).astype(np.float64)))


def test_write_again_changes_nothing(torch, gpu):
    rs = np.random.RandomState(8)
    dim, page, heads = 128, 32, 4
    slots = np.arange(10, 32)
    x, y = rs.normal(size=(2, len(slots), heads, dim)) * 100
    (kc, ks, *_), (vc, vs, *_) = [fresh_cache(torch, rs, 2, heads, page, dim) for _ in range(2)]
    w = gpu("CacheWrite", head_dim=dim, page_size=page, dtype="f16")
    args = (torch.from_numpy(x).half().cuda(), torch.from_numpy(y).half().cuda(), i32(torch, slots), kc, vc, ks, vs)
    w(*args)
    once = [t.clone() for t in args[3:]]
    w(*args)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(once, args[3:]))


def test_write_skips_slots_outside_the_cache(torch, gpu):
    rs = np.random.RandomState(9)
    dim, page, heads = 64, 16, 2
    slots = np.array([-1, 5, 3 * page, 3 * page + 1, 2 ** 31 - 1, 2 * page, -2 ** 31])
    x, y = rs.normal(size=(2, len(slots), heads, dim))
    cache = [fresh_cache(torch, rs, 3, heads, page, dim) for _ in range(2)]
    run_write(torch, gpu, x, y, slots, cache, "bf16", page, dim, faults=2)


def test_write_nothing(torch, gpu):
    w = gpu("CacheWrite", head_dim=64, page_size=16, dtype="bf16")
    rs = np.random.RandomState(1)
    (kc, ks, *_), (vc, vs, *_) = [fresh_cache(torch, rs, 1, 1, 16, 64) for _ in range(2)]
    none = torch.zeros((0, 1, 64), dtype=torch.bfloat16, device="cuda")
    w(none, none, i32(torch, []), kc, vc, ks, vs)


# ------------------------------------------------------------------------------------------------ attention

HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # torch.finfo(t).eps / 2, relative to the value


def attention_inputs(torch, dtype, dim, page, heads, group, lengths, queries, seed, value_exponents=(-4, 4), q_sigma=1.0):
    """Tensors of a batch over a cache whose unused pages, tails and table entries hold anything."""
    rs = np.random.RandomState(seed)
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    lengths, queries = np.array(lengths), np.array(queries)
    held = -(-lengths // page)
    pages = int(held.sum()) + 3
    order = rs.permutation(pages)
    width = int(held.max()) + 2
    table = rs.choice([-1, 2 ** 31 - 1, -2 ** 31, pages], size=(len(lengths), width)).astype(np.int64)
    codes = rs.randint(0, 256, (2, pages, heads, page, dim)).astype(np.uint8)
    codes[(codes & 127) == 127] = 8
    scales = np.stack([np.exp2(rs.randint(-9, -6, (pages, heads))), np.exp2(rs.randint(*value_exponents, (pages, heads)))]) * rs.choice([1.0, 1.37], (2, pages, heads))
    used = np.zeros((pages, page), dtype=bool)
    at = 0
    for b, n in enumerate(lengths):
        mine = order[at:at + held[b]]
        table[b, :held[b]] = mine
        at += held[b]
        for i, p in enumerate(mine):
            used[p, :max(0, min(page, n - i * page))] = True
    codes[:, ~used.any(axis=1)] = 127
    scales[:, ~used.any(axis=1)] = rs.choice([np.nan, np.inf], 1)
    for p in np.flatnonzero(used.any(axis=1)):
        codes[:, p][:, :, ~used[p]] = rs.choice([127, 255], 1)
    scales = scales.astype(np.float32)
    starts = np.concatenate([[0], np.cumsum(queries)])
    tokens = int(starts[-1]) + 3  # rows behind the last request
    rows = torch.from_numpy(rs.normal(size=(tokens, heads * group + 2, dim)) * q_sigma).to(t)
    out = torch.full((tokens, heads * group + 1, dim), 77.0, dtype=t, device="cuda")
    device = dict(q=rows.cuda()[:, :heads * group], k_cache=torch.from_numpy(codes[0]).cuda(), v_cache=torch.from_numpy(codes[1]).cuda(),
                  k_scales=torch.from_numpy(scales[0]).cuda(), v_scales=torch.from_numpy(scales[1]).cuda(), table=i32(torch, table), lengths=i32(torch, lengths),
                  starts=i32(torch, starts), out=out[:, :heads * group])
    host = dict(q=rows[:, :heads * group].double().numpy(), codes=E4M3[codes], scales=scales.astype(np.float64), table=table, lengths=lengths, starts=starts)
    return device, host, out


def check_attention(out, host, dtype, page, group, scale):
    o = out.double().cpu().numpy()
    tokens, starts = o.shape[0], host["starts"]
    heads, dim = host["codes"].shape[2], host["codes"].shape[4]
    assert np.array_equal(o[starts[-1]:], np.full(o[starts[-1]:].shape, 77.0)) and np.all(o[:, heads * group:] == 77.0)
    worst = 0.0
    for b, n in enumerate(host["lengths"]):
        m = starts[b + 1] - starts[b]
        pages = host["table"][b, :-(-n // page)]
        for h in range(heads):
            with np.errstate(invalid="ignore"):
                k, v = ((host["codes"][s][pages, h] * host["scales"][s][pages, h][:, None, None]).reshape(-1, dim)[:n] for s in (0, 1))
                vs = np.repeat(host["scales"][1][pages, h], page)[:n]
            for u in range(h * group, (h + 1) * group):
                q, got = host["q"][starts[b]:starts[b + 1], u], o[starts[b]:starts[b + 1], u]
                want, tol = so.attention(q, k, v, vs, n - m + np.arange(m) + 1, scale)
                tol = tol + HALF_STEP[dtype] * (np.abs(want) + tol) + 2.0 ** -25  # the result's rounding, and fp16's smallest step
                err = np.abs(got - want)
                assert np.all(np.isfinite(got)), (b, u)
                worst = max(worst, float((err / tol).max()) if m else 0.0)
                assert np.all(err <= tol), (b, u, worst)
    return worst


def run_attention(torch, gpu, dtype, dim, page, heads, group, lengths, queries, seed=0, scale=None, max_queries=None, max_length=None, faults=0, **kw):
    device, host, out = attention_inputs(torch, dtype, dim, page, heads, group, lengths, queries, seed, **kw)
    scale = scale or 1.0 / np.sqrt(dim)
    a = gpu("CacheAttention", head_dim=dim, page_size=page, dtype=dtype)
    max_queries, max_length = max_queries or max(1, max(queries)), max_length or max(1, max(lengths))
    n = a.workspace_bytes(device["q"].shape[0], len(lengths), heads * group, heads, max_queries, max_length)
    ws = torch.full((n + 64,), 255, dtype=torch.uint8, device="cuda")
    a(**device, scale=scale, max_queries=max_queries, max_length=max_length, workspace=ws)
    torch.cuda.synchronize()
    assert a.faults() == faults
    assert torch.all(ws[n:] == 255)
    check_attention(out, host, dtype, page, group, scale)
    return out, n


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim, page", [(64, 16), (64, 64), (128, 16), (128, 32), (128, 128), (192, 32), (256, 16), (256, 128)])
def test_attention_single_queries(torch, gpu, dtype, dim, page):
    run_attention(torch, gpu, dtype, dim, page, 2, 4, LENGTHS, [1] * len(LENGTHS), seed=dim + page)


@pytest.mark.parametrize("heads, group", [(1, 1), (3, 1), (1, 16), (2, 3), (1, 17), (1, 40), (5, 7)])
def test_attention_head_layouts(torch, gpu, heads, group):
    run_attention(torch, gpu, "bf16", 128, 16, heads, group, [1, 40, 129, 513], [1, 1, 1, 1], seed=heads)


@pytest.mark.parametrize("dim, page, group", [(64, 16, 4), (128, 32, 2), (192, 16, 1), (256, 64, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_several_queries(torch, gpu, dtype, dim, page, group):
    """Drafted tokens (few rows) and pieces of prompts (many); requests without queries, without keys, with more queries than keys."""
    run_attention(torch, gpu, dtype, dim, page, 2, group, [70, 5, 33, 0, 128], [3, 5, 2, 1, 4], seed=1)
    run_attention(torch, gpu, dtype, dim, page, 2, group, [0, 0, 9, 300, 150, 200, 64], [0, 2, 20, 130, 150, 1, 0], seed=2)


@pytest.mark.parametrize("dtype, dim, page, group", [("f16", 64, 16, 4), ("bf16", 128, 32, 3), ("bf16", 192, 16, 20), ("f16", 256, 64, 1)])
def test_attention_of_up_to_1024_keys(torch, gpu, dtype, dim, page, group):
    """A call of few workgroups whose keys eight wavefronts divide: lengths at the ends of their steps of 256 keys, several rows."""
    run_attention(torch, gpu, dtype, dim, page, 2, group, [1024, 513, 0, 1, 255, 256, 257, 1000, 33], [1, 3, 1, 2, 1, 1, 2, 3, 0], seed=dim)


def test_attention_rows_that_see_nothing(torch, gpu):
    for queries in (1, 100):
        device, host, out = attention_inputs(torch, "bf16", 128, 16, 1, 4, [0, 1], [queries, queries], seed=4)
        a = gpu("CacheAttention", head_dim=128, page_size=16, dtype="bf16")
        a(**device, scale=0.1, max_queries=queries, max_length=64)
        torch.cuda.synchronize()
        assert torch.all(out[:2 * queries - 1, :4] == 0)  # nothing, or queries in front of the first key
        check_attention(out, host, "bf16", 16, 4, 0.1)


@pytest.mark.parametrize("dtype, dim, page, heads, group, length, queries", [
    ("bf16", 128, 16, 1, 4, 5000, 1), ("f16", 64, 128, 2, 1, 9001, 2), ("f16", 256, 64, 1, 8, 4097, 3), ("bf16", 192, 32, 1, 2, 3001, 40), ("bf16", 64, 16, 1, 1, 70001, 1)])
def test_attention_split_keys(torch, gpu, dtype, dim, page, heads, group, length, queries):
    """Few long contexts: the keys are divided among workgroups and joined; a short request and an empty one beside them."""
    _, bytes_split = run_attention(torch, gpu, dtype, dim, page, heads, group, [length, 100, 0], [queries, 1, 1], seed=length)
    assert bytes_split > 0


def test_attention_division_does_not_matter(torch, gpu):
    """max_queries and max_length choose the division of the work; every choice is within the tolerance, and a run repeats itself to the bit."""
    for max_length in (1, 300, 1000, 5000, 1 << 20):
        for max_queries in (1, 2, 7, 500):
            out, _ = run_attention(torch, gpu, "bf16", 128, 16, 2, 3, [1000, 37], [7, 2], seed=5, max_queries=max_queries, max_length=max_length)
            again, _ = run_attention(torch, gpu, "bf16", 128, 16, 2, 3, [1000, 37], [7, 2], seed=5, max_queries=max_queries, max_length=max_length)
            assert torch.equal(out, again)


def test_attention_scales_far_apart(torch, gpu):
    """Pages of values whose scales differ by 2^60 beside one another, and sharp and flat distributions."""
    for sigma in (0.0, 0.1, 30.0):
        run_attention(torch, gpu, "bf16", 128, 16, 2, 2, [400, 33], [1, 3], seed=6, value_exponents=(-50, 10), q_sigma=sigma)


def test_attention_values_without_scale(torch, gpu):
    """A page whose scale of values is 0 weighs in the softmax and adds nothing."""
    device, host, out = attention_inputs(torch, "f16", 64, 16, 1, 2, [50, 16], [1, 1], seed=7)
    for b, p in ((0, 1), (1, 0)):
        page = host["table"][b, p]
        device["v_scales"][page] = 0.0
        host["scales"][1][page] = 0.0
    a = gpu("CacheAttention", head_dim=64, page_size=16, dtype="f16")
    a(**device, scale=0.125, max_queries=1, max_length=50)
    torch.cuda.synchronize()
    check_attention(out, host, "f16", 16, 2, 0.125)


@pytest.mark.parametrize("queries", [1, 50])
def test_attention_leaves_out_pages_outside_the_cache(torch, gpu, queries):
    dim, page = 128, 16
    device, host, out = attention_inputs(torch, "bf16", dim, page, 1, 2, [90, 64], [queries, 1], seed=8)
    for bad in (-1, device["k_cache"].shape[0], 2 ** 31 - 1):
        device["table"][0, 2] = bad
        a = gpu("CacheAttention", head_dim=dim, page_size=page, dtype="bf16")
        a(**device, scale=0.09, max_queries=queries, max_length=90)
        torch.cuda.synchronize()
        assert a.faults() > 0 and a.faults() == 0
        o = out.double().cpu().numpy()
        pages = host["table"][0, :6]
        k, v = ((host["codes"][s][pages, 0] * host["scales"][s][pages, 0][:, None, None]).reshape(-1, dim)[:90] for s in (0, 1))
        vs = np.repeat(host["scales"][1][pages, 0], page)[:90]
        kept = np.r_[0:32, 48:90]
        for i in range(queries):
            seen = kept[kept < 90 - queries + i + 1]
            for u in range(2):
                want, tol = so.attention(host["q"][i:i + 1, u], k[seen], v[seen], vs[seen], [len(seen)], 0.09)
                assert np.all(np.abs(o[i, u] - want) <= tol + HALF_STEP["bf16"] * (np.abs(want) + tol))


@pytest.mark.parametrize("dim, page, group", [(64, 16, 3), (128, 32, 1), (192, 64, 2), (256, 16, 2)])
@pytest.mark.parametrize("length, queries", [(90, 3), (90, 90), (700, 20), (1300, 300), (9000, 6)])
def test_attention_nan_stays_with_the_queries_that_see_it(torch, gpu, dim, page, group, length, queries):
    """NaN among the values, and among the keys, of tokens that the first queries do not see."""
    device, host, out = attention_inputs(torch, "bf16", dim, page, 1, group, [length, 50], [queries, 50], seed=length + dim)
    rs = np.random.RandomState(length)
    odd = np.zeros((length, dim), dtype=bool)
    for key in {length - 1, length - 2, length - 1 - queries // 2}:
        for d in (0, dim - 1, rs.randint(dim)):
            odd[key, d] = True
    codes = device["v_cache"].cpu().numpy()
    pages = host["table"][0, :-(-length // page)]
    for key, d in zip(*np.nonzero(odd)):
        codes[pages[key // page], 0, key % page, d] = rs.choice([127, 255])
    device["v_cache"] = torch.from_numpy(codes).cuda()
    a = gpu("CacheAttention", head_dim=dim, page_size=page, dtype="bf16")
    ws = torch.empty(a.workspace_bytes(device["q"].shape[0], 2, group, 1, max(queries, 50), length), dtype=torch.uint8, device="cuda")
    o = {}
    for blind in (False, True):
        if blind:  # the last token's key as well: the last query is NaN throughout
            device["k_cache"][int(pages[-1]), 0, (length - 1) % page, dim // 3] = 127
        a(**device, scale=0.09, max_queries=max(queries, 50), max_length=length, workspace=ws)
        torch.cuda.synchronize()
        assert a.faults() == 0
        o[blind] = out.double().cpu().numpy()
    for r, n in enumerate(host["lengths"]):
        at, m = host["starts"][r], host["starts"][r + 1] - host["starts"][r]
        mine = host["table"][r, :-(-n // page)]
        k, v = ((host["codes"][s][mine, 0] * host["scales"][s][mine, 0][:, None, None]).reshape(-1, dim)[:n] for s in (0, 1))
        vs = np.repeat(host["scales"][1][mine, 0], page)[:n]
        seen = n - m + np.arange(m) + 1
        nan = np.array([odd[:max(c, 0)].any(axis=0) for c in seen]) if r == 0 else np.zeros((m, dim), dtype=bool)
        for u in range(group):
            want, tol = so.attention(host["q"][at:at + m, u], k, np.where(odd, 0.0, v) if r == 0 else v, vs, seen, 0.09)
            tol = tol + HALF_STEP["bf16"] * (np.abs(want) + tol)
            for blind in (False, True):
                got, expect = o[blind][at:at + m, u], nan.copy()
                if blind and r == 0:
                    expect[m - 1] = True
                assert np.array_equal(np.isnan(got), expect), (r, u, blind)
                assert np.all(np.abs(got - want)[~expect] <= np.broadcast_to(tol, want.shape)[~expect])


def test_attention_length_beyond_the_table(torch, gpu):
    device, host, out = attention_inputs(torch, "bf16", 64, 16, 1, 1, [64, 20], [1, 1], seed=9)
    device["table"] = device["table"][:, :4].contiguous()
    device["lengths"][0] = 1000
    a = gpu("CacheAttention", head_dim=64, page_size=16, dtype="bf16")
    a(**device, scale=0.125, max_queries=1, max_length=64)
    torch.cuda.synchronize()
    assert a.faults() == 1
    check_attention(out, host, "bf16", 16, 1, 0.125)


# ------------------------------------------------------------------------------------------------ 4-bit weights

def run_matvec(torch, gpu, dtype, group, m, n, k, zeros="random", seed=0, mean=0.0):
    rs = np.random.RandomState(seed + m + n + k)
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    x = torch.from_numpy(rs.normal(size=(m, k + 8)) + mean).to(t)
    codes = rs.randint(0, 256, (n, k // 2)).astype(np.uint8)
    scales = torch.from_numpy(rs.uniform(0.005, 0.02, (k // group, n)) * rs.choice([-1.0, 1.0], (k // group, n))).to(t)
    z = {"random": rs.randint(0, 16, (k // group, n)), "wide": rs.randint(0, 256, (k // group, n)), "none": np.full((k // group, n), 8)}[zeros].astype(np.uint8)
    y = torch.full((m, n + 3), 99.0, dtype=t, device="cuda")  # rows of x and y stand in wider ones
    gpu("Matvec4", group=group, dtype=dtype)(x.cuda()[:, :k], torch.from_numpy(codes).cuda(), scales.cuda(), y[:, :n],
                                             zeros=None if zeros == "none" else torch.from_numpy(z).cuda())
    torch.cuda.synchronize()
    got = y.double().cpu().numpy()
    assert np.all(got[:, n:] == 99.0)
    want, tol = so.matvec4(x[:, :k].double().numpy(), codes, scales.double().numpy(), z.astype(np.float64), group, {"bf16": 128, "f16": 64}[dtype])
    tol = tol + HALF_STEP[dtype] * (np.abs(want) + tol) + 2.0 ** -25
    assert np.all(np.abs(got[:, :n] - want) <= tol), float((np.abs(got[:, :n] - want) / tol).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 16, 3), (2, 17, 8), (15, 33, 9), (16, 100, 2), (17, 31, 5), (33, 64, 4), (64, 129, 7), (1, 1000, 33)])
def test_matvec(torch, gpu, dtype, group, m, n, k):
    """k in groups: blocks of 128 columns that are whole, partial, and fewer than the wavefronts."""
    run_matvec(torch, gpu, dtype, group, m, n, k * group, seed=group)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m, n, k, zeros", [(1, 20000, 256, "none"), (5, 16385, 128, "wide"), (1, 48, 16384, "random"), (40, 300, 4096, "none"), (64, 5, 8192, "wide")])
def test_matvec_sizes(torch, gpu, dtype, m, n, k, zeros):
    run_matvec(torch, gpu, dtype, 128, m, n, k, zeros=zeros)


def test_matvec_activations_with_a_mean(torch, gpu):
    """The sums that the offset and the zero point take out are large then."""
    for dtype in ("bf16", "f16"):
        run_matvec(torch, gpu, dtype, 64, 3, 65, 2048, mean=4.0)


def test_matvec_row_with_nan_stays_alone(torch, gpu):
    rs = np.random.RandomState(1)
    x = torch.from_numpy(rs.normal(size=(3, 256))).bfloat16().cuda()
    x[1, 77] = float("nan")
    codes, scales = torch.from_numpy(rs.randint(0, 256, (40, 128)).astype(np.uint8)).cuda(), torch.full((2, 40), 0.01, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros((3, 40), dtype=torch.bfloat16, device="cuda")
    gpu("Matvec4", group=128, dtype="bf16")(x, codes, scales, y)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[::2]).all()
    gpu("Matvec4", group=128, dtype="bf16")(x[:0], codes, scales, y[:0])


def test_matvec_codes_beyond_32_bits(torch, gpu):
    """5.2 GB of codes: the last columns, whose rows begin behind 2^32 bytes."""
    n, k, group = 40000, 262144, 128
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randn((2, k), generator=g, device="cuda").bfloat16()
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((k // group, n), generator=g, device="cuda") * 0.01 + 0.005).bfloat16()
    y = torch.zeros((2, n), dtype=torch.bfloat16, device="cuda")
    gpu("Matvec4", group=group, dtype="bf16")(x, codes, scales, y)
    for at in (slice(0, 4), slice(n - 4, n)):
        want, tol = so.matvec4(x.double().cpu().numpy(), codes[at].cpu().numpy(), scales[:, at].double().cpu().numpy(), np.full((k // group, 4), 8.0), group, 128)
        assert np.all(np.abs(y[:, at].double().cpu().numpy() - want) <= tol + HALF_STEP["bf16"] * (np.abs(want) + tol))


# ------------------------------------------------------------------------------------------------ a step


def test_a_serving_step(torch, gpu):
    """All operators as a server calls them: projection, tables, write, attention, projection; prompts, then tokens one at a
    time, replayed from a graph in turn with eager calls."""
    dim, page, heads, group, requests, pages, hidden, columns = 128, 16, 2, 4, 3, 40, 256, 64
    rs = np.random.RandomState(12)
    tables, write, attend, project = (gpu(n, **k) for n, k in (
        ("PageTable", dict(page_size=page)), ("CacheWrite", dict(head_dim=dim, page_size=page, dtype="bf16")),
        ("CacheAttention", dict(head_dim=dim, page_size=page, dtype="bf16")), ("Matvec4", dict(group=columns, dtype="bf16"))))
    width, most, qkv_rows = 12, 60, heads * (group + 2)
    state = dict(cached=i32(torch, [0] * requests), added=i32(torch, [0] * requests), free=i32(torch, rs.permutation(pages)), count=i32(torch, [pages]),
                 table=i32(torch, np.full((requests, width), -1)), lengths=i32(torch, [0] * requests), starts=i32(torch, [0] * (requests + 1)),
                 slots=i32(torch, [0] * most), counts=i32(torch, [0, 0]))
    kc, vc = (torch.full((pages, heads, page, dim), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((pages, heads), float("nan"), device="cuda") for _ in range(2))

    def weights(n, k):
        return (torch.from_numpy(rs.randint(0, 256, (n, k // 2)).astype(np.uint8)).cuda(),
                torch.from_numpy(rs.uniform(0.005, 0.02, (k // columns, n))).bfloat16().cuda(),
                torch.from_numpy(rs.randint(4, 12, (k // columns, n)).astype(np.uint8)).cuda())

    def check_product(x, w, y):
        want, tol = so.matvec4(x.double().cpu().numpy(), w[0].cpu().numpy(), w[1].double().cpu().numpy(), w[2].double().cpu().numpy(), columns, 128)
        assert np.all(np.abs(y.double().cpu().numpy() - want) <= tol + HALF_STEP["bf16"] * (np.abs(want) + tol))

    w_in, w_out = weights(qkv_rows * dim, hidden), weights(hidden, heads * group * dim)
    x = torch.zeros((most, hidden), dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros((most, qkv_rows, dim), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((most, heads * group, dim), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros((most, hidden), dtype=torch.bfloat16, device="cuda")
    ws = torch.zeros(attend.workspace_bytes(most, requests, heads * group, heads, most, width * page), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()

    def step(stream):
        q, k, v = qkv[:, :heads * group], qkv[:, heads * group:heads * (group + 1)], qkv[:, heads * (group + 1):]
        project(x, w_in[0], w_in[1], qkv.view(most, -1), zeros=w_in[2], stream=stream)
        tables(state["cached"], state["added"], state["free"], state["count"], state["table"], state["lengths"], state["starts"], state["slots"],
               state["counts"], stream=stream)
        write(k, v, state["slots"], kc, vc, ks, vs, stream=stream)
        attend(q, kc, vc, ks, vs, state["table"], state["lengths"], state["starts"], out, dim ** -0.5, max_queries=most, max_length=width * page, workspace=ws,
               stream=stream)
        project(out.view(most, -1), w_out[0], w_out[1], y, zeros=w_out[2], stream=stream)

    with torch.cuda.stream(side):
        step(side.cuda_stream)  # adds nothing: no request has tokens yet
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)

    keys = [[np.zeros((0, heads, dim))] * 2 for _ in range(requests)]  # of each request, before they are coded
    for turn, added in enumerate([[20, 1, 33], [1, 1, 1], [1, 0, 1], [1, 16, 1], [14, 1, 0], [1, 1, 1]]):
        state["added"].copy_(i32(torch, added))
        x.copy_(torch.from_numpy(rs.normal(size=tuple(x.shape))).bfloat16())
        out.fill_(5.0)
        for t in (qkv, y):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        if turn % 2 == 0:
            graph.replay()
        else:
            step(None)
        torch.cuda.synchronize()
        assert int(state["counts"][1]) == 0 and write.faults() == 0 and attend.faults() == 0
        check_product(x, w_in, qkv.view(most, -1))
        check_product(out.view(most, -1), w_out, y)
        starts = np.concatenate([[0], np.cumsum(added)])
        assert np.array_equal(state["starts"].cpu().numpy(), starts)
        values = qkv.double().cpu().numpy()
        got = out.double().cpu().numpy()
        assert np.all(got[starts[-1]:] == 5.0)
        scales = [ks.cpu().numpy().astype(np.float64), vs.cpu().numpy().astype(np.float64)]
        table = state["table"].cpu().numpy()
        for b in range(requests):
            mine = values[starts[b]:starts[b + 1]]
            for side_of in (0, 1):
                at = heads * (group + side_of)
                keys[b][side_of] = np.concatenate([keys[b][side_of], mine[:, at:at + heads]])
            n = len(keys[b][0])
            held = table[b, :-(-n // page)]
            for h in range(heads):
                coded = []
                for side_of, codes in ((0, kc), (1, vc)):
                    value = (E4M3[codes.cpu().numpy()[held, h]] * scales[side_of][held, h][:, None, None]).reshape(-1, dim)[:n]
                    # a code is half a step from its value (2^-4 of it, or 2^-10 of the scale), once more for every time the
                    # page's scale doubled, which loses under the smallest step only
                    bound = np.abs(keys[b][side_of][:, h]) * 2.0 ** -4 + np.repeat(scales[side_of][held, h], page)[:n, None] * 2.0 ** -10 * 3
                    assert np.all(np.abs(value - keys[b][side_of][:, h]) <= bound)
                    coded.append(value)
                for u in range(h * group, (h + 1) * group):
                    want, tol = so.attention(mine[:, u], coded[0], coded[1], np.repeat(scales[1][held, h], page)[:n], n - len(mine) + np.arange(len(mine)) + 1,
                                             dim ** -0.5)
                    assert np.all(np.abs(got[starts[b]:starts[b + 1], u] - want) <= tol + HALF_STEP["bf16"] * (np.abs(want) + tol)), (turn, b, u)
        state["cached"].copy_(state["lengths"])
        state["count"].copy_(state["counts"][:1])


@pytest.mark.parametrize("queries", [1, 100])
def test_cache_beyond_32_bits(torch, gpu, queries):
    """Pages behind 2^32 bytes of codes: the same bits as from a small cache, and pages in front of them are left alone."""
    dim, page, heads, tokens, pages = 256, 128, 1, 300, 140_000
    assert pages * heads * page * dim > 2 ** 32
    rs = np.random.RandomState(30)
    write, attend = gpu("CacheWrite", head_dim=dim, page_size=page, dtype="bf16"), gpu("CacheAttention", head_dim=dim, page_size=page, dtype="bf16")
    k, v = (torch.from_numpy(rs.normal(size=(tokens, heads, dim))).bfloat16().cuda() for _ in range(2))
    q = torch.from_numpy(rs.normal(size=(queries, 4, dim))).bfloat16().cuda()
    results = []
    for total, held in ((4, [0, 3, 1]), (pages, [pages - 1, pages - 3, 7])):
        kc, vc = (torch.zeros((total, heads, page, dim), dtype=torch.uint8, device="cuda") for _ in range(2))
        ks, vs = (torch.ones((total, heads), device="cuda") for _ in range(2))
        slots = np.array(held).repeat(page)[:tokens] * page + np.arange(tokens) % page
        write(k, v, i32(torch, slots), kc, vc, ks, vs)
        out = torch.zeros_like(q)
        attend(q, kc, vc, ks, vs, i32(torch, [held]), i32(torch, [tokens]), i32(torch, [0, queries]), out, 0.06, max_queries=queries)
        torch.cuda.synchronize()
        assert write.faults() == 0 and attend.faults() == 0
        assert int(kc.view(torch.int64).count_nonzero()) <= 3 * page * dim // 8
        results.append((out.clone(), kc[held].clone(), vc[held].clone(), ks[held].clone()))
        del kc, vc
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_attention_in_place(torch, gpu):
    """The result may take the queries' place."""
    for queries in (1, 60):
        device, host, out = attention_inputs(torch, "bf16", 128, 32, 2, 4, [700, 90], [queries, 2], seed=31)
        a = gpu("CacheAttention", head_dim=128, page_size=32, dtype="bf16")
        a(**device, scale=0.1, max_queries=queries, max_length=700)
        device["out"] = device["q"]
        a(**device, scale=0.1, max_queries=queries, max_length=700)
        torch.cuda.synchronize()
        n = int(host["starts"][-1])
        assert torch.equal(device["q"][:n], out[:n, :8])


def test_two_streams_at_a_time(torch, gpu):
    """One pipeline on two streams, each with its own buffers and workspace; the same results as one after the other."""
    a = gpu("CacheAttention", head_dim=128, page_size=16, dtype="bf16")
    runs = []
    for seed in (20, 21):
        device, host, out = attention_inputs(torch, "bf16", 128, 16, 2, 4, [5000, 300], [1, 2], seed=seed)
        n = a.workspace_bytes(device["q"].shape[0], 2, 8, 2, 2, 5000)
        runs.append((device, host, out, torch.empty(n, dtype=torch.uint8, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for device, _, _, ws, stream in runs:
            a(**device, scale=0.1, max_queries=2, max_length=5000, workspace=ws, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for _, host, out, _, _ in runs:
        check_attention(out, host, "bf16", 16, 4, 0.1)


@pytest.mark.parametrize("dim, scale", [(64, -0.2), (128, 0.0), (192, -0.05), (256, 0.5)])
def test_attention_scales_of_any_sign(torch, gpu, dim, scale):
    for queries in (2, 70):
        device, host, out = attention_inputs(torch, "f16", dim, 32, 1, 3, [120, 33], [queries, 1], seed=dim)
        a = gpu("CacheAttention", head_dim=dim, page_size=32, dtype="f16")
        a(**device, scale=scale, max_queries=queries, max_length=120)
        torch.cuda.synchronize()
        o, starts = out.double().cpu().numpy(), host["starts"]
        for b, n in enumerate(host["lengths"]):
            pages, m = host["table"][b, :-(-n // 32)], starts[b + 1] - starts[b]
            k, v = ((host["codes"][s][pages, 0] * host["scales"][s][pages, 0][:, None, None]).reshape(-1, dim)[:n] for s in (0, 1))
            vs = np.repeat(host["scales"][1][pages, 0], 32)[:n]
            for u in range(3):
                q = host["q"][starts[b]:starts[b + 1], u]
                want, tol = so.attention(np.sign(scale) * q, k, v, vs, n - m + np.arange(m) + 1, abs(scale))
                assert np.all(np.abs(o[starts[b]:starts[b + 1], u] - want) <= tol + HALF_STEP["f16"] * (np.abs(want) + tol) + 2.0 ** -25)
