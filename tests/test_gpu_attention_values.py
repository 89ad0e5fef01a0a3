"""Attention over extreme values, in every plan (one tile's rows or many, keys in one run or split over
workgroups): NaN that a row sees is NaN in that row and nowhere else."""

import numpy as np
import pytest
import torch

from tests.paged import attend, attention_tolerance, pack_keys, pack_values
from tests.test_gpu_attention import make, run

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

# new and cached tokens, and whether the keys are split over workgroups
PLANS = {"few": ([(1, 100), (3, 50)], False), "few-split": ([(2, 6000), (1, 4000)], True),
         "many": ([(100, 150), (40, 90)], False), "many-split": ([(60, 5000)], True),
         "both": ([(100, 3000), (1, 5000)], True)}


def planned(gpu, name, D, dtype=F16, seed=0):
    from raceline_amd import ops

    lens, split = PLANS[name]
    s = make(gpu, lens, 4, 2, D, dtype=dtype, seed=seed)
    assert (ops.attention_workspace_bytes(s.T, 4, 2, D, len(lens), s.max_q, s.max_kv) > 0) == split
    return s


def put(s, b, pos, dim, value, keys=False, head=None):
    """Writes one dimension of a cached position (of all key/value heads, or one)."""
    page = s.page
    mark = np.zeros((1, 1, page, s.D), np.float32)
    mark[0, 0, pos % page, dim] = 1
    m = torch.from_numpy((pack_keys if keys else pack_values)(mark)).to(s.kc.device)[0, 0].bool()
    c = (s.kc if keys else s.vc)[int(s.table[b, pos // page])]
    for h in range(c.shape[0]) if head is None else [head]:
        c[h][m] = value


def rows_of(s, out, out_dtype=F16):
    """Per sequence: rows, the 64-bit rows without what was put in, and their tolerance."""
    got = out.double().cpu().numpy().reshape(s.T, -1, s.D)
    for b, (n, kv) in enumerate(s.lens):
        r = slice(s.cu[b], s.cu[b] + n)
        ref, size = attend(s.q[r], s.keys[b], s.values[b], kv, s.D ** -0.5)
        yield got[r], ref, attention_tolerance(ref, size, s.q[r], s.keys[b], kv, s.D ** -0.5, 0.0, s.dtype, out_dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("plan", PLANS)
def test_a_query_with_nan_gives_a_row_of_nan(gpu, plan, D):
    s = planned(gpu, plan, D)
    bad = [(0, 0), (s.T - 1, 3)]                             # (row, head)
    for row, head in bad:
        s.dq[row, head * D + 5] = float("nan")
    out = run(s, gpu)
    assert all(out[row, head * D:(head + 1) * D].isnan().all() for row, head in bad)
    at = 0
    for got, ref, tol in rows_of(s, out):
        fine = np.ones(got.shape[:2], bool)
        for row, head in bad:
            if at <= row < at + len(got):
                fine[row - at, head] = False
        assert (np.abs(got - ref) <= tol)[fine].all()
        at += len(got)


@pytest.mark.parametrize("n,kv", [(1, 33), (1, 34), (1, 129), (3, 65), (1, 4097), (2, 6001), (40, 41), (129, 193),
                                  (60, 4097), (100, 8200)])
@pytest.mark.parametrize("D", [64, 256])
def test_a_lone_nan_key_reaches_the_rows_that_see_it(gpu, D, n, kv):
    """The newest key, alone in its block, wave or run of keys: only the last row sees it."""
    s = make(gpu, [(n, kv)], 4, 2, D)
    put(s, 0, kv - 1, 7, float("nan"), keys=True)
    (got, ref, tol), = rows_of(s, run(s, gpu))
    assert np.isnan(got[-1]).all()
    assert (np.abs(got[:-1] - ref[:-1]) <= tol[:-1]).all()


@pytest.mark.parametrize("plan", PLANS)
def test_a_block_of_nan_keys_reaches_the_rows_that_see_it(gpu, plan):
    """32 keys that one wave takes together, seen by every row of its sequence."""
    s = planned(gpu, plan, 128)
    for pos in range(32):
        put(s, 0, pos, 3, float("nan"), keys=True, head=1)   # query heads 2 and 3
    for b, (got, ref, tol) in enumerate(rows_of(s, run(s, gpu))):
        hit = slice(2, 4) if b == 0 else slice(0, 0)
        assert np.isnan(got[:, hit]).all()
        rest = np.delete(np.arange(4), hit)
        assert (np.abs(got - ref) <= tol)[:, rest].all()
