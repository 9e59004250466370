"""How attention over the cache divides the keys, seen through the workspace that it asks for, without a GPU."""
import pytest

import gern_amd


def splits(attend, tokens, requests, q_heads, kv_heads, max_queries, max_length):
    n = attend.workspace_bytes(tokens=tokens, requests=requests, q_heads=q_heads, kv_heads=kv_heads, max_queries=max_queries, max_length=max_length)
    part = tokens * q_heads * (attend.head_dim + 2) * 4
    assert n % part == 0
    return max(1, n // part)


@pytest.fixture(scope="module")
def attend():
    return gern_amd.CacheAttention(128, 16, "bf16", flags=gern_amd.COMPILE_ONLY)


@pytest.mark.parametrize("requests, kv_heads, group, queries", [(128, 8, 4, 1), (1024, 1, 4, 1), (128, 8, 16, 1), (64, 16, 4, 3), (200, 8, 4, 4)])
@pytest.mark.parametrize("max_length", [5000, 20000, 100000, 262144])
def test_a_long_request_in_a_large_batch_is_divided(attend, requests, kv_heads, group, queries, max_length):
    """No piece of the longest request is more than 8192 keys while the parts stay under 256 MiB."""
    n = splits(attend, requests * queries, requests, kv_heads * group, kv_heads, queries, max_length)
    most = (256 << 20) // (requests * queries * kv_heads * group * 130 * 4)
    assert n >= min(-(-max_length // 8192), most) and n <= max(1, most)


def test_short_requests_of_a_large_batch_are_whole(attend):
    for max_length in (1000, 2000, 4096):
        assert splits(attend, 128, 128, 32, 8, 1, max_length) == 1


def test_workspace_grows_with_the_tokens(attend):
    """A workspace for more tokens serves fewer of the same requests."""
    sizes = dict(requests=256, q_heads=32, kv_heads=8, max_queries=8, max_length=262144)
    n = [attend.workspace_bytes(tokens=t, **sizes) for t in (1, 256, 700, 2048)]
    assert n == sorted(n) and n[0] > 0 and n[-1] <= 256 << 20
