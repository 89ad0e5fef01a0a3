"""How much scratch an attention call asks for, without a GPU: it goes by the tiles whose keys are split, not by
the call's rows, since every layer's call allocates it beside a cache that was given the rest of the memory."""

import random

import pytest

from raceline_amd import ops

MB = 1 << 20


@pytest.mark.parametrize("H,KV,D,tokens", [(20, 4, 256, 8200), (16, 4, 256, 10267), (32, 8, 128, 6172), (20, 4, 256, 8192)])
def test_a_prompts_first_tiles_are_not_split(H, KV, D, tokens):
    """Tiles past a whole number for the CUs are the prompt's shortest."""
    assert ops.attention_workspace_bytes(tokens, H, KV, D, 1, tokens, tokens) == 0


@pytest.mark.parametrize("H,KV,D,T,B,max_q,max_kv,most", [
    (20, 4, 256, 8216, 1, 8216, 32768, 64), (20, 4, 256, 2048, 1, 2048, 8192, 64), (16, 4, 256, 32 * 65, 32, 65, 4000, 256),
    (20, 4, 256, 2049, 2, 2048, 8192, 128), (20, 4, 256, 2079, 32, 2048, 16000, 300), (32, 8, 128, 4095, 1000, 3096, 8000, 300)])
def test_scratch_of_long_calls(H, KV, D, T, B, max_q, max_kv, most):
    assert ops.attention_workspace_bytes(T, H, KV, D, B, max_q, max_kv) <= most * MB


def test_scratch_is_bounded():
    """Split tiles of many rows: 256 MB. Of few rows: at most 511 workgroups and one a tile, and at most twice as many
    tiles as are counted (2044 runs of 32 rows of D + 2 floats), with 16 bytes a tile."""
    rng = random.Random(3)
    for _ in range(20000):
        KV, G, D = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 5, 8, 16, 33]), rng.choice([64, 128, 256])
        B, max_q = int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 13))
        T = min(65536, rng.randint(1, B * max_q))
        max_kv = int(2 ** rng.uniform(0, 20))
        window = rng.choice([0, 0, 1000])
        n = ops.attention_workspace_bytes.__wrapped__(T, G * KV, KV, D, B, max_q, max_kv, window)
        assert n <= 257 * MB + 2044 * 32 * (D + 2) * 4 + 2044 * 16, (T, G * KV, KV, D, B, max_q, max_kv, window)
