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


@pytest.mark.parametrize("cached, added", [([0], [0]), ([0], [1]), ([16], [1]), ([15], [1]), ([15], [2]), ([0, 0, 0], [0, 0, 0]), ([5, 0, 7], [0, 40, 0]),
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
