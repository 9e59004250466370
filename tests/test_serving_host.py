"""The operators of a serving step without a GPU: what is generated compiles for gfx950, every refusal is an error with a
message, and the plain loops that the device is checked against agree with torch's conversions."""
import ctypes as C

import numpy as np
import pytest
import torch

import gern_amd
import serving_oracle as so

ONLY = gern_amd.COMPILE_ONLY


@pytest.fixture(scope="module")
def pipe():
    return dict(tables=gern_amd.PageTable(16, flags=ONLY), write=gern_amd.CacheWrite(64, 16, "bf16", flags=ONLY),
                attention=gern_amd.CacheAttention(64, 16, "bf16", flags=ONLY), matvec=gern_amd.Matvec4(64, "bf16", flags=ONLY))


# ------------------------------------------------------------------------------------------------ creation

@pytest.mark.parametrize("make, call", [
    (lambda: gern_amd.PageTable(64, flags=ONLY), "gernels::extend_page_table<page, threads, per>"),
    (lambda: gern_amd.CacheWrite(192, 32, "f16", flags=ONLY), "gernels::write_cache<head_dim, page, threads>"),
    (lambda: gern_amd.CacheAttention(256, 128, "f16", flags=ONLY), "gernels::attend_few_rows<head_dim, page, waves>"),
    (lambda: gern_amd.Matvec4(32, "f16", flags=ONLY), "gernels::multiply_4bit<group, row_tiles, column_tiles, waves>")])
def test_generated_programs(make, call):
    p = make()
    assert call in p.source and "__launch_bounds__(" in p.source and p.kernel_name.startswith("function_")


@pytest.mark.parametrize("make", [
    lambda: gern_amd.PageTable(8, flags=ONLY), lambda: gern_amd.PageTable(48, flags=ONLY), lambda: gern_amd.PageTable(256, flags=ONLY),
    lambda: gern_amd.CacheWrite(96, 16, flags=ONLY), lambda: gern_amd.CacheWrite(320, 16, flags=ONLY), lambda: gern_amd.CacheWrite(64, 20, flags=ONLY),
    lambda: gern_amd.CacheWrite(64, 16, "f32", flags=ONLY), lambda: gern_amd.CacheAttention(32, 16, flags=ONLY),
    lambda: gern_amd.CacheAttention(64, 512, flags=ONLY), lambda: gern_amd.CacheAttention(64, 16, "fp16", flags=ONLY),
    lambda: gern_amd.Matvec4(16, flags=ONLY), lambda: gern_amd.Matvec4(256, flags=ONLY), lambda: gern_amd.Matvec4(64, "int8", flags=ONLY)])
def test_creation_refuses(make):
    with pytest.raises(gern_amd.GernError, match="must be"):
        make()


def test_creation_refuses_types_and_null():
    lib, h = gern_amd.pipelines_lib(), C.c_void_p()
    for rc in (lib.gern_cache_write_create(64, 16, 2, ONLY, C.byref(h)), lib.gern_cache_attention_create(64, 16, -1, ONLY, C.byref(h)),
               lib.gern_matvec4_create(64, 7, ONLY, C.byref(h)), lib.gern_page_table_create(16, ONLY, None)):
        assert rc != 0 and not h


# ------------------------------------------------------------------------------------------------ the C ABI's checks

def refused(rc, *words):
    assert rc != 0
    message = gern_amd._pipe_error()
    for w in words:
        assert w in message, message


A = 1 << 20  # an address that is aligned; nothing is read in these calls


def tables_args(pipe, **kw):
    a = dict(cached=A, added=A + 4096, requests=4, free=A + 8192, capacity=100, count=A + 12288, table=A + 16384, width=8, lengths=A + 20480,
             starts=A + 24576, slots=A + 28672, tokens=10, counts=A + 32768)
    a.update(kw)
    return [pipe["tables"].h] + list(a.values()) + [None]


@pytest.mark.parametrize("kw, word", [
    (dict(), "compile-only"), (dict(requests=-1), "requests"), (dict(requests=8193), "8192"), (dict(width=0), "table_width"), (dict(tokens=-1), "tokens"),
    (dict(capacity=2 ** 31), "free_capacity"), (dict(cached=None), "null"), (dict(count=None), "null"), (dict(slots=None), "null"), (dict(free=None), "null"),
    (dict(added=A + 2), "aligned"), (dict(counts=A + 32769), "aligned"), (dict(lengths=A), "shares memory"), (dict(counts=A + 12288), "shares memory"),
    (dict(table=A + 20480 - 64), "two results"), (dict(starts=A + 28672), "two results"), (dict(slots=A + 8192), "shares memory"),
    (dict(requests=0, cached=None, added=None, table=None, lengths=None), "compile-only"), (dict(tokens=0, slots=None), "compile-only")])
def test_tables_run_refuses(pipe, kw, word):
    refused(gern_amd.pipelines_lib().gern_page_table_run(*tables_args(pipe, **kw)), "gern_page_table_run", word)


def write_args(pipe, **kw):
    a = dict(K=A, ldk=128, V=A, ldv=128, slots=A, tokens=3, heads=2, k=A, v=A, ks=A, vs=A, pages=5)
    a.update(kw)
    return [pipe["write"].h] + list(a.values()) + [None]


@pytest.mark.parametrize("kw, word", [
    (dict(), "compile-only"), (dict(k=None), "null"), (dict(vs=None), "null"), (dict(K=None), "null"), (dict(slots=None), "null"), (dict(k=A + 8), "aligned"),
    (dict(ks=A + 2), "aligned"), (dict(K=A + 2), "aligned"), (dict(V=A + 8), "aligned"), (dict(ldk=132), "multiples of 8"), (dict(ldv=120), "less than"),
    (dict(heads=0), "heads"), (dict(heads=65536), "heads"), (dict(pages=0), "pages"), (dict(pages=2 ** 27), "pages"), (dict(tokens=-1), "tokens"),
    (dict(slots=A + 1), "aligned"), (dict(ldk=-128), "less than"), (dict(tokens=2 ** 31 - 1, heads=60000, ldk=64 * 60000, ldv=64 * 60000), "2^30")])
def test_write_run_refuses(pipe, kw, word):
    refused(gern_amd.pipelines_lib().gern_cache_write_run(*write_args(pipe, **kw)), "gern_cache_write_run", word)


def attention_args(pipe, **kw):
    a = dict(Q=A, ldq=256, k=A, v=A, ks=A, vs=A, pages=5, table=A, width=4, lengths=A, starts=A, requests=2, tokens=3, q_heads=4, heads=2, O=A, ldo=256,
             scale=0.1, max_queries=2, max_length=64, workspace=None, workspace_bytes=0)
    a.update(kw)
    return [pipe["attention"].h] + list(a.values()) + [None]


@pytest.mark.parametrize("kw, word", [
    (dict(), "compile-only"), (dict(k=None), "null"), (dict(Q=None), "null"), (dict(O=None), "null"), (dict(table=None), "null"), (dict(lengths=None), "null"),
    (dict(starts=None), "null"), (dict(Q=A + 8), "aligned"), (dict(O=A + 4), "aligned"), (dict(table=A + 2), "aligned"), (dict(ldq=260), "multiples of 8"),
    (dict(ldq=248), "less than"), (dict(ldo=128), "less than"), (dict(q_heads=3), "multiple"), (dict(heads=0), "heads"), (dict(q_heads=1), "multiple"),
    (dict(requests=65536), "requests"), (dict(requests=-1), "requests"), (dict(tokens=-1), "tokens"), (dict(tokens=2 ** 30), "2^31"),
    (dict(max_queries=0), "max_queries"), (dict(max_length=0), "max_length"), (dict(max_length=2 ** 30 + 1), "max_length"), (dict(width=0), "table_width"),
    (dict(width=2 ** 27), "table_width"), (dict(pages=0), "pages"), (dict(max_length=100000), "workspace"),
    (dict(max_length=100000, workspace=A + 8, workspace_bytes=2 ** 40), "workspace"), (dict(max_length=100000, workspace=A, workspace_bytes=1000), "workspace"),
    (dict(max_length=100000, workspace=A, workspace_bytes=2 ** 40), "shares memory")])
def test_attention_run_refuses(pipe, kw, word):
    refused(gern_amd.pipelines_lib().gern_cache_attention_run(*attention_args(pipe, **kw)), "gern_cache_attention_run", word)


def matvec_args(pipe, **kw):
    a = dict(X=A, ldx=128, codes=A, scales=A, zeros=None, Y=A * 8, ldy=40, M=3, N=40, K=128)
    a.update(kw)
    return [pipe["matvec"].h] + list(a.values()) + [None]


@pytest.mark.parametrize("kw, word", [
    (dict(), "compile-only"), (dict(X=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(Y=None), "null"), (dict(M=65), "64"),
    (dict(M=-1), "M must"), (dict(N=0), "N in"), (dict(K=96), "group"), (dict(K=0), "K in"), (dict(K=2 ** 24 + 64), "2^24"), (dict(X=A + 8), "aligned"),
    (dict(codes=A + 8), "aligned"), (dict(scales=A + 1), "aligned"), (dict(ldx=132), "multiple of 8"), (dict(ldx=120), "less than"), (dict(ldy=39), "less than"),
    (dict(ldx=2 ** 26), "more than"), (dict(Y=A), "shares memory"), (dict(zeros=A * 8 + 50), "shares memory")])
def test_matvec_run_refuses(pipe, kw, word):
    refused(gern_amd.pipelines_lib().gern_matvec4_run(*matvec_args(pipe, **kw)), "gern_matvec4_run", word)


def test_runs_refuse_other_pipelines(pipe):
    lib = gern_amd.pipelines_lib()
    other = gern_amd.Softmax(256, flags=ONLY).h
    n = C.c_int64()
    for rc in (lib.gern_page_table_run(other, *tables_args(pipe)[1:]), lib.gern_cache_write_run(other, *write_args(pipe)[1:]),
               lib.gern_cache_attention_run(other, *attention_args(pipe)[1:]), lib.gern_matvec4_run(other, *matvec_args(pipe)[1:]),
               lib.gern_cache_attention_workspace(other, 1, 1, 1, 1, 1, 1, C.byref(n)), lib.gern_page_table_run(None, *tables_args(pipe)[1:])):
        refused(rc, "bad pipeline")
    # and the others refuse these
    assert lib.gern_softmax_run(pipe["matvec"].h, A, A, 1, 256, None) != 0


def test_nothing_to_do_is_no_error(pipe):
    lib = gern_amd.pipelines_lib()
    assert lib.gern_cache_write_run(*write_args(pipe, tokens=0, K=None, V=None, slots=None)) == 0
    assert lib.gern_cache_attention_run(*attention_args(pipe, tokens=0, Q=None)) == 0
    assert lib.gern_cache_attention_run(*attention_args(pipe, requests=0, lengths=None)) == 0
    assert lib.gern_matvec4_run(*matvec_args(pipe, M=0, X=None)) == 0


def test_workspace(pipe):
    a = pipe["attention"]
    sizes = dict(tokens=2, requests=2, q_heads=8, kv_heads=2, max_queries=1, max_length=512)
    assert a.workspace_bytes(**sizes) == 0  # one launch
    sizes["max_length"] = 65536
    n = a.workspace_bytes(**sizes)
    assert n > 0 and n % (2 * 8 * (64 + 2) * 4) == 0  # a part and two statistics a row and split
    assert a.workspace_bytes(**dict(sizes, requests=0)) == 0
    for bad in (dict(q_heads=3), dict(max_queries=0), dict(max_length=0), dict(requests=70000), dict(tokens=-1)):
        with pytest.raises(gern_amd.GernError, match="gern_cache_attention_workspace"):
            a.workspace_bytes(**dict(sizes, **bad))


# ------------------------------------------------------------------------------------------------ the Python view's checks

def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_python_checks(pipe):
    half, cache, scales = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 16, 64, dtype=torch.uint8), torch.zeros(5, 2)
    good = dict(
        tables=[i32(4), i32(4), i32(100), i32(1), i32(4, 8), i32(4), i32(5), i32(10), i32(2)],
        write=[half, half, i32(3), cache, cache, scales, scales],
        attention=[half, cache, cache, scales, scales, i32(2, 4), i32(2), i32(3), half, 0.1],
        matvec=[torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(40, 64, dtype=torch.uint8), torch.zeros(2, 40, dtype=torch.bfloat16),
                torch.zeros(3, 40, dtype=torch.bfloat16)])
    for name, args in good.items():
        with pytest.raises(gern_amd.GernError, match="GPU"):  # what is on the CPU is refused last
            pipe[name](*args)
    bad = [("tables", 0, i32(4).long(), "int32"), ("tables", 1, i32(5), "must be"), ("tables", 4, i32(8, 4).t(), "contiguous"), ("tables", 6, i32(4), "must be"),
           ("tables", 8, i32(3), "must be"), ("tables", 0, i32(2, 2), "must be"), ("write", 0, half.half(), "bfloat16"), ("write", 1, half[:, :1], "must be"),
           ("write", 0, torch.zeros(3, 2, 128, dtype=torch.bfloat16)[..., ::2], "contiguous"), ("write", 2, i32(4), "must be"), ("write", 3, cache[:, :, :8], "page_size"),
           ("write", 5, scales.double(), "float32"), ("write", 6, scales[:, :1], "scales"), ("write", 4, torch.zeros(5, 2, 16, 64), "must be"),
           ("attention", 0, half[..., :32], "must be"), ("attention", 8, half.half(), "bfloat16"), ("attention", 5, i32(3, 4), "must be"), ("attention", 7, i32(2), "must be"),
           ("matvec", 1, torch.zeros(40, 64, dtype=torch.int8), "uint8"), ("matvec", 2, torch.zeros(2, 40), "must be"), ("matvec", 3, torch.zeros(2, 40, dtype=torch.bfloat16), "must be")]
    for name, at, wrong, word in bad:
        args = list(good[name])
        args[at] = wrong
        with pytest.raises(gern_amd.GernError, match=word):
            pipe[name](*args)


# ------------------------------------------------------------------------------------------------ the oracle

def test_oracle_codes_and_rounding():
    codes = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(so.e4m3_table(), codes.view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)
    x = torch.arange(0, 2 ** 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[x.isfinite()]
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(so.e4m3_round(x.double().numpy()), want)
    for amax, scale in ((448.0, 1.0), (448.5, 2.0), (224.0, 0.5), (225.0, 1.0), (1e-30, 2.0 ** -64), (0.0, 2.0 ** -64), (448.0 * 2.0 ** -64, 2.0 ** -64)):
        assert so.scale_for(amax) == scale


def test_oracle_attention_is_softmax():
    rs = np.random.RandomState(0)
    q, k, v = rs.normal(size=(3, 8)), rs.normal(size=(10, 8)), rs.normal(size=(10, 8))
    o, tol = so.attention(q, k, v, np.ones(10), [0, 4, 10], 0.5)
    p = torch.softmax(torch.from_numpy(k @ q[2]) * 0.5, dim=0).numpy()
    assert np.all(o[0] == 0) and np.allclose(o[2], p @ v, rtol=1e-12) and np.all(tol[2] < 1e-2)


def test_refuses_launches_of_too_many_threads(pipe):
    """2^32 threads and more are no launch; such sizes are refused by name."""
    lib = gern_amd.pipelines_lib()
    refused(lib.gern_cache_write_run(*write_args(pipe, tokens=2 ** 25, heads=128, ldk=128 * 128, ldv=128 * 128)), "gern_cache_write_run", "2^23")
    refused(lib.gern_matvec4_run(*matvec_args(pipe, M=1, N=2 ** 31 - 1, Y=1 << 50)), "gern_matvec4_run", "2^27")
    refused(lib.gern_cache_attention_run(*attention_args(pipe, tokens=2 ** 25, requests=1, max_length=100000, O=1 << 52, workspace=1 << 40, workspace_bytes=2 ** 50)),
            "gern_cache_attention_run", "2^24")
