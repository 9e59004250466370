"""Calls of the serving operators whose buffers share memory are refused before anything is launched; the arithmetic is
tests/cpp/test_memory_ranges.cpp's."""
import numpy as np
import pytest

from test_gpu_serving import attention_inputs, gpu, i32, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def bytes_as(torch, flat, at, like):  # noqa: F811
    """A tensor of like's type and shape over flat's bytes from `at` on."""
    return flat[at:at + like.numel() * like.element_size()].view(like.dtype).view(like.shape)


@pytest.mark.parametrize("one, other", [("k", "k_cache"), ("v", "v_cache"), ("k", "v_scales"), ("slots", "v_cache"), ("slots", "k_scales"), ("k_cache", "v_cache"),
                                        ("k_cache", "k_scales"), ("v_scales", "k_scales"), ("v_cache", "k_scales")])
def test_write_refuses_shared_memory(torch, gpu, one, other):  # noqa: F811
    w = gpu("CacheWrite", head_dim=64, page_size=16, dtype="bf16")
    half = dict(dtype=torch.bfloat16, device="cuda")
    t = dict(k=torch.ones((4, 2, 64), **half), v=torch.ones((4, 2, 64), **half), slots=i32(torch, np.arange(4)),
             k_cache=torch.zeros((3, 2, 16, 64), dtype=torch.uint8, device="cuda"), v_cache=torch.zeros((3, 2, 16, 64), dtype=torch.uint8, device="cuda"),
             k_scales=torch.ones((3, 2), device="cuda"), v_scales=torch.ones((3, 2), device="cuda"))
    w(**t)
    a, b = t[one], t[other]
    na, nb = (x.numel() * x.element_size() for x in (a, b))
    flat = torch.zeros(na + nb + 64, dtype=torch.uint8, device="cuda")
    for at in (0, nb - 16 if nb >= 16 else 0):  # at the start, and in the last bytes
        t[other], t[one] = bytes_as(torch, flat, 0, b), bytes_as(torch, flat, at // 16 * 16, a)
        with pytest.raises(gpu.error, match="share memory"):
            w(**t)
    t[one] = bytes_as(torch, flat, -(-nb // 16) * 16, a)  # side by side
    w(**t)
    torch.cuda.synchronize()


@pytest.mark.parametrize("result", ["out", "workspace"])
@pytest.mark.parametrize("other", ["k_cache", "v_cache", "k_scales", "v_scales", "table", "lengths", "starts"])
def test_attention_refuses_shared_memory(torch, gpu, result, other):  # noqa: F811
    a = gpu("CacheAttention", head_dim=64, page_size=16, dtype="bf16")
    device, _, out = attention_inputs(torch, "bf16", 64, 16, 1, 2, [2000, 30], [1, 1], seed=1)
    device["out"] = torch.zeros_like(device["q"])
    n = a.workspace_bytes(device["q"].shape[0], 2, 2, 1, 1, 2000)
    assert n > 0
    run = dict(device, workspace=torch.zeros(n, dtype=torch.uint8, device="cuda"))
    a(**run, scale=0.1, max_length=2000)
    b, r = run[other], run[result]
    nb, nr = (x.numel() * x.element_size() for x in (b, r))
    flat = torch.zeros(nb + nr + 64, dtype=torch.uint8, device="cuda")
    run[other], run[result] = bytes_as(torch, flat, 0, b).copy_(b), bytes_as(torch, flat, (nb - 1) // 16 * 16, r)
    with pytest.raises(gpu.error, match="shares memory"):
        a(**run, scale=0.1, max_length=2000)
    run[result] = bytes_as(torch, flat, -(-nb // 16) * 16, r)
    a(**run, scale=0.1, max_length=2000)
    torch.cuda.synchronize()
    assert a.faults() == 0


def test_attention_out_beside_its_queries(torch, gpu):  # noqa: F811
    """O in Q's place or in other columns of the same rows is fine, anything else of Q is not."""
    a = gpu("CacheAttention", head_dim=64, page_size=16, dtype="bf16")
    device, host, out = attention_inputs(torch, "bf16", 64, 16, 1, 2, [40, 33], [2, 3], seed=2)
    q = device["q"].contiguous()
    tokens, heads, dim = q.shape
    device["q"] = q
    a(**device, scale=0.1, max_queries=3, max_length=40)
    torch.cuda.synchronize()
    want, n = device["out"].clone(), int(host["starts"][-1])
    rows = torch.zeros((tokens + 1, 2 * heads, dim), dtype=q.dtype, device="cuda")
    device["q"] = rows[:tokens, :heads]
    for good in (rows[:tokens, heads:], rows[1:, heads:], rows[:tokens, :heads]):
        rows[:tokens, :heads] = q
        device["out"] = good
        a(**device, scale=0.1, max_queries=3, max_length=40)
        torch.cuda.synchronize()
        assert torch.equal(good[:n], want[:n])
    wider = torch.zeros((tokens, 3 * heads, dim), dtype=q.dtype, device="cuda")
    for q_at, bad in ((rows[:tokens, :heads], rows[:tokens, 1:1 + heads]), (rows[:tokens, :heads], rows[1:, :heads]),
                      (wider.view(-1, heads, dim)[:tokens], wider[:, :heads])):
        device["q"], device["out"] = q_at, bad
        with pytest.raises(gpu.error, match="not in its place"):
            a(**device, scale=0.1, max_queries=3, max_length=40)
    n = a.workspace_bytes(tokens, 2, heads, 1, 3, 2000)
    flat = torch.zeros(n + q.numel() * 2, dtype=torch.uint8, device="cuda")
    device["q"], device["out"] = bytes_as(torch, flat, n - 16, q), torch.zeros_like(q)
    with pytest.raises(gpu.error, match="workspace shares memory with Q"):
        a(**device, scale=0.1, max_queries=3, max_length=2000, workspace=flat[:n])
