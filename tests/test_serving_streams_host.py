"""The stream that a call of the serving operators' Python view hands to the C ABI, without a GPU."""
import pytest
import torch

import gern_amd


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("named, handed", [({}, 4711), (dict(stream=0), 0), (dict(stream=99), 99), (dict(stream=None), 4711)])
def test_stream_of_a_call(named, handed):
    only = gern_amd.COMPILE_ONLY
    half, cache, scales = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 16, 64, dtype=torch.uint8), torch.zeros(5, 2)
    calls = [(gern_amd.PageTable(16, flags=only), [i32(4), i32(4), i32(100), i32(1), i32(4, 8), i32(4), i32(5), i32(10), i32(2)]),
             (gern_amd.CacheWrite(64, 16, "bf16", flags=only), [half, half, i32(3), cache, cache, scales, scales]),
             (gern_amd.CacheAttention(64, 16, "bf16", flags=only), [half, cache, cache, scales, scales, i32(2, 4), i32(2), i32(3), half, 0.1]),
             (gern_amd.Matvec4(64, "bf16", flags=only), [torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(40, 64, dtype=torch.uint8),
                                                         torch.zeros(2, 40, dtype=torch.bfloat16), torch.zeros(3, 40, dtype=torch.bfloat16)])]
    for pipeline, args in calls:
        taken = []
        pipeline._device, pipeline._current_stream = -1, lambda device: 4711 + (device + 1)  # the device of tensors on the CPU
        pipeline._run = lambda *a: taken.append(a[-1]) or 0
        pipeline(*args, **named)
        assert taken == [handed]
