"""Attention over the cache of batches whose requests differ much, and of more queries than a call says."""
import numpy as np
import pytest

import serving_oracle as so
from test_gpu_serving import HALF_STEP, attention_inputs, check_attention, gpu, run_attention, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim, heads, group, queries", [(64, 8, 4, 1), (128, 16, 1, 3)])
def test_one_long_request_of_many(torch, gpu, dim, heads, group, queries):  # noqa: F811
    requests, page = 128, 16
    rs = np.random.RandomState(dim)
    lengths = rs.randint(1, 60, requests)
    lengths[[0, 70, 127]] = [9000, 0, 4100]
    counts = np.minimum(rs.randint(1, queries + 1, requests), np.maximum(lengths, 1))
    device, host, out = attention_inputs(torch, "bf16", dim, page, heads, group, lengths, counts, seed=dim)
    a = gpu("CacheAttention", head_dim=dim, page_size=page, dtype="bf16")
    tokens, scale = device["q"].shape[0], dim ** -0.5
    n = a.workspace_bytes(tokens, requests, heads * group, heads, queries, 9000)
    assert n == 3 * tokens * heads * group * (dim + 2) * 4  # pieces of 3072 keys
    for workspace in (torch.full((n,), 255, dtype=torch.uint8, device="cuda"), None, torch.empty(n - 16, dtype=torch.uint8, device="cuda"),
                      torch.empty(n + 8, dtype=torch.uint8, device="cuda")[8:]):
        out.fill_(77.0)
        a(**device, scale=scale, max_queries=queries, max_length=9000, workspace=workspace)
        torch.cuda.synchronize()
        assert a.faults() == 0
        o, starts = out.double().cpu().numpy(), host["starts"]
        assert np.all(o[starts[-1]:] == 77.0) and np.all(o[starts[70]:starts[71], :heads * group] == 0.0)
        for b in (0, 1, 69, 127):
            length, m = lengths[b], counts[b]
            pages = host["table"][b, :-(-length // page)]
            for h in (0, heads - 1):
                k, v = ((host["codes"][s][pages, h] * host["scales"][s][pages, h][:, None, None]).reshape(-1, dim)[:length] for s in (0, 1))
                vs = np.repeat(host["scales"][1][pages, h], page)[:length]
                for u in range(h * group, (h + 1) * group):
                    want, tol = so.attention(host["q"][starts[b]:starts[b] + m, u], k, v, vs, length - m + np.arange(m) + 1, scale)
                    assert np.all(np.abs(o[starts[b]:starts[b] + m, u] - want) <= tol + HALF_STEP["bf16"] * (np.abs(want) + tol)), (b, u)


@pytest.mark.parametrize("dim, group", [(64, 1), (128, 2), (192, 1), (256, 1)])
def test_whole_prompts(torch, gpu, dim, group):  # noqa: F811
    """As many queries as keys: the first one sees one key."""
    run_attention(torch, gpu, "bf16", dim, 32, 1, group, [400, 1, 257, 0], [400, 1, 257, 0], seed=dim)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("length, said", [(600, 1), (600, 70), (3000, 1), (3000, 70)])
def test_more_queries_and_keys_than_said(torch, gpu, dim, length, said):  # noqa: F811
    """Workgroups of either program that take rows after rows, the keys undivided and divided."""
    device, host, out = attention_inputs(torch, "f16", dim, 16, 1, 1, [length, 300], [300, 2], seed=length + dim)
    a = gpu("CacheAttention", head_dim=dim, page_size=16, dtype="f16")
    n = a.workspace_bytes(device["q"].shape[0], 2, 1, 1, said, length // 2 + 300)
    for _ in range(2):  # the second run finds the first one's parts
        a(**device, scale=dim ** -0.5, max_queries=said, max_length=length // 2 + 300, workspace=torch.empty(n, dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        assert a.faults() == 0 and (n > 0) == (length > 1500)
        check_attention(out, host, "f16", 16, 1, dim ** -0.5)
