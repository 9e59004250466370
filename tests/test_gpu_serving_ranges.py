"""The operators of a serving step where weights, scales and activations leave the ordinary range, against 64 bits."""
import numpy as np
import pytest

import serving_oracle as so
from test_gpu_serving import E4M3, HALF_STEP, gpu, i32, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def code_of(x):
    """The e4m3 code nearest to each value."""
    import torch
    return torch.from_numpy(np.asarray(x, dtype=np.float32)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def attention_of(q, k, v, v_scales, limits, scale):
    """One head of one request, as serving_oracle.attention: the result, and how far a kernel may be from it before it rounds
    its result.  Weights are p * (scale of the value), the largest of a row 2^15: fp16 keeps 11 bits of them down to 2^-14, that
    is 2^-29 of the largest, and is off by 2^-25, that is 2^-40 of the largest, under it."""
    n, dim = q.shape
    o, tol = np.zeros((n, dim)), np.zeros((n, dim))
    codes = np.abs(v) / np.where(v_scales > 0, v_scales, 1.0)[:, None]
    for i in range(n):
        m = int(limits[i])
        if m <= 0:
            continue
        z = (k[:m] @ q[i]) * scale
        exponent = ((dim / 32 + 8) * 2.0 ** -24 * (np.abs(k[:m]) @ np.abs(q[i])) * scale + 8 * 2.0 ** -24 * (np.abs(z) + 128)).max()
        p = np.exp(z - z.max())
        p /= p.sum()
        o[i] = p @ v[:m]
        tol[i] = (2.0 ** -11 + 2 * exponent + (m / 32 + 16) * 2.0 ** -24) * (p @ np.abs(v[:m])) + 2.0 ** -40 * codes[:m].sum(axis=0) * (p * v_scales[:m]).max()
    return o, tol


class Request:
    """One request over pages in order, one head of keys; kc and vc [length, dim] codes, scales a page."""

    def __init__(self, torch, dtype, page, kc, vc, k_scales, v_scales, q):
        length, dim = kc.shape
        pages = -(-length // page)
        t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
        self.page, self.dim, self.length, self.dtype = page, dim, length, dtype
        codes = np.zeros((2, pages, 1, page, dim), dtype=np.uint8)
        codes.reshape(2, -1, dim)[:, :length] = np.stack([kc, vc])
        self.k_cache, self.v_cache = (torch.from_numpy(c).cuda() for c in codes)
        scales = np.stack([k_scales, v_scales]).astype(np.float32)
        self.k_scales, self.v_scales = (torch.from_numpy(s[:, None].copy()).cuda() for s in scales)
        self.q = torch.from_numpy(q).to(t)  # [queries, heads, dim]
        of = np.repeat(scales.astype(np.float64), page, axis=1)[:, :length]
        self.k, self.v, self.vs = E4M3[kc] * of[0][:, None], E4M3[vc] * of[1][:, None], of[1]

    def run(self, torch, gpu, scale, few=True, splits=True):
        """The result.  `few`: the program for few rows.  Not `splits`: as among so many workgroups that keys are not divided (requests
        without tokens and room for 64 rows each, whose parts would take too much memory, or room for more queries)."""
        queries, heads, dim = self.q.shape
        requests = 1 if splits or not few or self.length <= 1024 else 16384
        max_queries = (queries if requests == 1 else 64 // heads) if few else 100 if splits else 1 << 17
        a = gpu("CacheAttention", head_dim=dim, page_size=self.page, dtype=self.dtype)
        n = a.workspace_bytes(queries, requests, heads, 1, max_queries, self.length)
        assert (n > 0) == splits
        table = np.tile(np.arange(self.k_cache.shape[0]), (requests, 1))
        out = torch.zeros((queries, heads, dim), dtype=self.q.dtype, device="cuda")
        a(self.q.cuda(), self.k_cache, self.v_cache, self.k_scales, self.v_scales, i32(torch, table), i32(torch, [self.length] + [0] * (requests - 1)),
          i32(torch, [0] + [queries] * requests), out, scale, max_queries=max_queries, max_length=self.length,
          workspace=torch.empty(n, dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        assert a.faults() == 0
        return out.double().cpu().numpy()

    def check(self, out, scale):
        queries, heads, _ = self.q.shape
        for h in range(heads):
            want, tol = attention_of(self.q[:, h].double().numpy(), self.k, self.v, self.vs, self.length - queries + np.arange(queries) + 1, scale)
            tol = tol + HALF_STEP[self.dtype] * (np.abs(want) + tol) + (2.0 ** -25 if self.dtype == "f16" else 2.0 ** -134)
            assert np.all(np.abs(out[:, h] - want) <= tol), float((np.abs(out[:, h] - want) / tol).max())


@pytest.mark.parametrize("few, splits", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("length, above, ratio, spread", [(32768, 12, 16, 0.0), (131072, 13, 64, 0.0), (131072, 13, 64, 1.0), (20000, 9, 2 ** 12, 0.5)])
def test_attention_keeps_small_weights(torch, gpu, few, splits, length, above, ratio, spread):  # noqa: F811
    """One key far above the others, whose value is 0 in most dimensions, on a page of a larger scale: what the others add up
    to there is the result."""
    dim, page, queries = 64, 128 if few and not splits else 16, 2 if few else 100
    rs = np.random.RandomState(length + above)
    q = rs.normal(size=(queries, 2, dim))
    q[..., 0] = 1.0
    k = rs.normal(size=(length, dim)) * spread / dim ** 0.5
    k[:, 0], k[0] = 0.0, 0.0
    k[0, 0] = above
    pages = -(-length // page)
    v_scales = np.full(pages, 2.0 ** -4)
    v_scales[0] *= ratio
    v = 32.0 * (1.0 + 0.3 * rs.normal(size=(length, dim)))  # in units of their page's scale
    v[:page] /= ratio
    v[0] = 0.0
    v[0, 0] = 256.0
    r = Request(torch, "bf16", page, code_of(k), code_of(v), np.ones(pages), v_scales, q)
    r.check(r.run(torch, gpu, 1.0, few, splits), 1.0)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("length", [8000, 9000])
def test_attention_nan_in_keys_of_no_weight(torch, gpu, few, length):  # noqa: F811
    """A value that is NaN makes its dimension of the result NaN also where its part of the keys has a weight of 0 beside the
    others (16 parts, joined by a wavefront, and 18, by a workgroup)."""
    dim, page, queries, high = 64, 32, 2 if few else 100, length - 700
    rs = np.random.RandomState(length)
    q = rs.normal(size=(queries, 2, dim))
    q[..., 0] = 1.0
    k = np.zeros((length, dim))
    k[high, 0] = 144.0  # 207 in base 2: 2^-207 of it is 0
    v = code_of(rs.normal(size=(length, dim)))
    v[100, 5], v[101, 63] = 127, 255
    pages = -(-length // page)
    for nan in (True, False):
        out = Request(torch, "bf16", page, code_of(k), v, np.ones(pages), np.ones(pages), q).run(torch, gpu, 1.0, few)
        odd = np.zeros(dim, dtype=bool)
        odd[[5, 63]] = nan
        assert np.array_equal(np.isnan(out), np.broadcast_to(odd, out.shape))
        assert np.array_equal(out[..., ~odd], np.broadcast_to(E4M3[v[high]][~odd], out[..., ~odd].shape))
        v[100, 5], v[101, 63] = 0, 0


def random_request(torch, dtype, dim, page, length, v_scales, queries, heads=2, seed=0):  # noqa: F811
    rs = np.random.RandomState(seed)
    k, v = (code_of(rs.normal(size=(length, dim)) * 16) for _ in range(2))
    return Request(torch, dtype, page, k, v, np.full(-(-length // page), 1 / 64), v_scales, rs.normal(size=(queries, heads, dim)))


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("dim, length, splits", [(64, 600, False), (128, 5000, True), (192, 200, False), (256, 3000, True)])
def test_attention_small_scales_of_values(torch, gpu, few, dim, length, splits):  # noqa: F811
    """Scales of values down to 2^-80; what is under that, 0 among it, weighs in the softmax and adds nothing."""
    page, queries, scale = 16, 2 if few else 90, dim ** -0.5
    pages = -(-length // page)
    rs = np.random.RandomState(length)
    for scales in (np.full(pages, 2.0 ** -70), np.full(pages, 1.37 * 2.0 ** -80), np.exp2(rs.randint(-80, -60, pages)), np.exp2(rs.randint(-80, 4, pages))):
        r = random_request(torch, "bf16", dim, page, length, scales, queries, seed=length)
        r.check(r.run(torch, gpu, scale, few, splits), scale)
        none = rs.rand(pages) < 0.4
        for small in (0.0, 2.0 ** -140, 2.0 ** -81):
            r.v_scales[torch.from_numpy(none).cuda()] = small
            r.v[np.repeat(none, page)[:length]] = 0.0
            r.check(r.run(torch, gpu, scale, few, splits), scale)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("dim, length, splits", [(64, 600, False), (128, 5000, True), (256, 100, False)])
def test_attention_values_of_no_scale(torch, gpu, few, dim, length, splits):  # noqa: F811
    """No page has a scale: the result is 0, but for dimensions in which a key that is seen has NaN."""
    page, queries = 32, 3 if few else 90
    r = random_request(torch, "bf16", dim, page, length, np.zeros(-(-length // page)), queries, seed=length)
    assert np.all(r.run(torch, gpu, 0.1, few, splits) == 0.0)
    codes = r.v_cache.view(-1, dim)
    codes[7, 3], codes[length - 2, dim - 1] = 127, 255  # the last but one key: all but the first `queries - 2` see it
    out = r.run(torch, gpu, 0.1, few, splits)
    odd = np.zeros(out.shape, dtype=bool)
    odd[:, :, 3] = True
    odd[queries - 2:, :, dim - 1] = True
    assert np.array_equal(np.isnan(out), odd) and np.all(out[~odd] == 0.0)


@pytest.mark.parametrize("few", [True, False])
def test_attention_small_scales_of_keys(torch, gpu, few):  # noqa: F811
    """Large queries and keys of a small scale: the scores are ordinary.  Keys of scale 0 have the score 0."""
    dim, page, length, queries = 128, 16, 400, 2 if few else 90
    rs = np.random.RandomState(3)
    k, v = (code_of(rs.normal(size=(length, dim)) * 16) for _ in range(2))
    q = rs.normal(size=(queries, 2, dim)) * 2.0 ** 100
    pages = -(-length // page)
    k_scales = np.exp2(rs.randint(-108, -103, pages))
    k_scales[3] = 0.0
    r = Request(torch, "bf16", page, k, v, k_scales, np.ones(pages), q)
    r.check(r.run(torch, gpu, dim ** -0.5, few, False), dim ** -0.5)


@pytest.mark.parametrize("m", [1, 3, 4, 5, 16, 20, 40])
@pytest.mark.parametrize("group, k", [(32, 96), (64, 320), (128, 1024)])
@pytest.mark.parametrize("zeros", [True, False])
def test_matvec_large_activations(torch, gpu, m, group, k, zeros):  # noqa: F811
    """Activations up to the largest of bf16 whose products with the weights are finite: no sum on the way overflows."""
    rs = np.random.RandomState(m + k)
    n = 50
    for x, size in ((rs.normal(size=(m, k)) * 1e36, 0.01), (np.full((m, k), 2.0 ** 127), 2.0 ** -20), (rs.choice([-3.3e38, 3.3e38], (m, k)), 2.0 ** -20)):
        x = torch.from_numpy(x).bfloat16()
        codes = rs.randint(0, 256, (n, k // 2)).astype(np.uint8)
        scales = torch.from_numpy(rs.uniform(0.5, 2.0, (k // group, n)) * size).bfloat16()
        z = rs.randint(0, 256, (k // group, n)).astype(np.uint8) if zeros else np.full((k // group, n), 8, dtype=np.uint8)
        y = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
        gpu("Matvec4", group=group, dtype="bf16")(x.cuda(), torch.from_numpy(codes).cuda(), scales.cuda(), y, zeros=torch.from_numpy(z).cuda() if zeros else None)
        torch.cuda.synchronize()
        want, tol = so.matvec4(x.double().numpy(), codes, scales.double().numpy(), z.astype(np.float64), group, 128)
        assert np.abs(want).max() < 3e38
        assert np.all(np.abs(y.double().cpu().numpy() - want) <= tol + HALF_STEP["bf16"] * (np.abs(want) + tol))


@pytest.mark.parametrize("m", [1, 4, 13, 40])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_matvec_small_activations(torch, gpu, m, group):  # noqa: F811
    """Activations around 2^-112: the sums are taken of 2^-16 of the products, in steps of 2^-149 at least."""
    rs = np.random.RandomState(m + group)
    n, k = 50, 1024
    x = torch.from_numpy(rs.normal(size=(m, k)) * 2.0 ** -112).bfloat16()
    codes = rs.randint(0, 256, (n, k // 2)).astype(np.uint8)
    scales = torch.from_numpy(rs.uniform(0.5, 2.0, (k // group, n))).bfloat16()
    z = rs.randint(0, 256, (k // group, n)).astype(np.uint8)
    y = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    gpu("Matvec4", group=group, dtype="bf16")(x.cuda(), torch.from_numpy(codes).cuda(), scales.cuda(), y, zeros=torch.from_numpy(z).cuda())
    torch.cuda.synchronize()
    want, tol = so.matvec4(x.double().numpy(), codes, scales.double().numpy(), z.astype(np.float64), group, 128)
    # half steps of 2^-149: 8 + group / 32 of a group's products, as many of its sum of x, which counts 3 times (383 / 128), and one
    # where the group is added; all times 2^16
    steps = 2.0 ** -150 * (4 * (8 + group / 32) + 1) * scales.double().numpy().sum(axis=0) * 2.0 ** 16
    assert np.all(np.abs(y.double().cpu().numpy() - want) <= tol + steps + HALF_STEP["bf16"] * (np.abs(want) + tol + steps))


@pytest.mark.parametrize("few, length, splits", [(True, 300, False), (True, 5000, True), (False, 300, False), (False, 5000, True)])
@pytest.mark.parametrize("power", [10, 18, 20, 22, 24, 26, 30, 50, 90])
def test_attention_large_scores(torch, gpu, few, length, splits, power):  # noqa: F811
    """Scores of both signs up to 2^98: with gaps beyond what 32 bits leave between them, a query's result is its best key's value."""
    dim, page, queries = 64, 16, 2 if few else 90
    rs = np.random.RandomState(power)
    k = np.zeros((length, dim))
    k[:, 0] = rs.randint(-8, 8, length) + 0.5  # ties share the row
    k[:, 1] = rs.choice([-0.5, 0.0, 0.5], length)
    q = np.zeros((queries, 2, dim))
    q[..., 0], q[..., 1] = 2.0 ** power * rs.choice([-1.25, 1.0, 1.5], (queries, 2)), 2.0 ** (power - 3)
    pages = -(-length // page)
    r = Request(torch, "bf16", page, code_of(k), code_of(rs.normal(size=(length, dim)) * 16), np.full(pages, 16.0), 1.37 * np.exp2(rs.randint(-9, 4, pages)), q)
    out = r.run(torch, gpu, 1.0, few, splits)
    for h in range(2):
        q = r.q[:, h].double().numpy()
        for i in range(queries):
            n = length - queries + i + 1
            z = r.k[:n] @ q[i]
            best = z == z.max()
            assert np.sort(z[~best])[-1] < z.max() - 200.0  # nothing else has a weight
            want = r.v[:n][best].mean(axis=0)
            # the best keys' scores are equal, and so are their exponents but for their scales' logarithms, which are added in 32 bits
            step = 2.0 ** -24 * (np.abs(z.max()) * 1.4427 + 16)
            if best.sum() == 1 or step < 2.0 ** -6:
                size = np.abs(r.v[:n][best]).mean(axis=0)
                tol = (2.0 ** -11 + (8 * step if best.sum() > 1 else 0.0) + 2.0 ** -18) * size
                assert np.all(np.abs(out[i, h] - want) <= tol + HALF_STEP["bf16"] * (np.abs(want) + tol)), (i, h)
            else:
                # weights of ties are off by the rounding of their exponents: the result is between the ties' values
                lo, hi = r.v[:n][best].min(axis=0), r.v[:n][best].max(axis=0)
                slack = HALF_STEP["bf16"] * np.maximum(np.abs(lo), np.abs(hi)) * 1.01
                assert np.all(out[i, h] >= lo - slack) and np.all(out[i, h] <= hi + slack), (i, h)
