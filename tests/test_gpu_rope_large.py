"""rope_append where a workgroup takes all heads that share a key/value head (1024 blocks and heads or more), with many
tokens a block: its threads step over tokens and heads there."""

import pytest
import torch

from tests.test_gpu_rope import check

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
LENS = [(1 + 37 * i % 121, 1 + 37 * i % 121 + 53 * i % 400) for i in range(24)] + [(0, 9), (200, 200)]


def blocks(lens):
    return sum(n for n, _ in lens) // 32 + 2 * len(lens)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("D,H,KV,rot", [(64, 33, 11, 64), (64, 24, 12, 20), (128, 48, 12, 128), (128, 24, 12, 40),
                                        (256, 55, 11, 64), (256, 11, 11, 256), (64, 120, 12, 0)])
def test_all_heads_a_workgroup(gpu, D, H, KV, rot, interleaved, dtype):
    assert blocks(LENS) * KV >= 1024
    check(gpu, LENS, H, KV, D, rot=rot, interleaved=interleaved, dtype=dtype, norm=rot != 64, m=1.25)


@pytest.mark.parametrize("pad", [1, 4, 8])
def test_strides(gpu, pad):
    check(gpu, LENS, 24, 12, 128, rot=40, norm=True, pad=pad, interleaved=pad == 4)


def test_blocks_of_every_count_of_tokens(gpu):
    """1 to 32 tokens in a block, at every place in it."""
    lens = [(1 + i % 32, 1 + i % 32 + 7 * i) for i in range(96)]
    assert blocks(lens) * 8 >= 1024
    check(gpu, lens, 24, 8, 64, rot=64, page=96)
    check(gpu, lens, 8, 8, 256, rot=20, interleaved=True, norm=True, page=32, dtype=BF16)


def test_rows_before_position_zero_and_pages_that_are_not_there(gpu):
    lens = LENS + [(90, 40), (70, 200)]
    check(gpu, lens, 22, 11, 64, page=32, break_pages=[(len(lens) - 1, 4), (len(lens) - 1, 5)])
