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


TYPES = [(F16, F16), (BF16, F16), (BF16, BF16), (F16, BF16)]
INF = float("inf")


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=["f16", "bf16-f16", "bf16", "f16-bf16"])
@pytest.mark.parametrize("plan", PLANS)
def test_an_infinite_value_is_infinite_in_the_rows_that_see_it(gpu, plan, dtype, out_dtype):
    """In a block that all rows see, and in the newest, that they see in part; two of them with different
    signs are NaN."""
    s = planned(gpu, plan, 64, dtype)
    n, kv = s.lens[0]
    put(s, 0, 40, 3, INF)
    put(s, 0, 41, 4, -INF)
    put(s, 0, 40, 9, INF)
    put(s, 0, 45, 9, -INF)
    put(s, 0, kv - 1, 17, -INF)                              # the last row alone
    for b, (got, ref, tol) in enumerate(rows_of(s, run(s, gpu, out_dtype=out_dtype), out_dtype)):
        if b == 0:
            assert (got[:, :, 3] == INF).all() and (got[:, :, 4] == -INF).all() and np.isnan(got[:, :, 9]).all()
            assert (got[-1, :, 17] == -INF).all()
            ok = np.abs(got - ref) <= tol
            ok[:, :, [3, 4, 9]] = ok[-1, :, 17] = True
            assert ok.all()
        else:
            assert (np.abs(got - ref) <= tol).all()


@pytest.mark.parametrize("dtype,full", [(F16, False), (F16, True), (BF16, True)], ids=["f16", "f16-full", "bf16-full"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("plan", PLANS)
def test_infinite_values_in_every_tile_of_dimensions(gpu, plan, D, dtype, full):
    """In the first and last dimensions of larger heads, seen by the rows from one position on (in one plan not
    by its first 20, whose positions are 50 to 69) and by the last alone, beside a row whose scores are NaN."""
    s = planned(gpu, plan, D, dtype)
    n, kv = s.lens[0]
    place = 70 if kv > 100 else 40
    for dim in (0, 31, 32, D // 2 + 5, D - 1):
        put(s, 0, place, dim, INF)
    put(s, 0, kv - 1, D - 2, -INF)
    s.dq[0, D + 5] = float("nan")                            # row 0, head 1
    for b, (got, ref, tol) in enumerate(rows_of(s, run(s, gpu, out_dtype=dtype, full_weights=full), dtype)):
        ok = np.abs(got - ref) <= tol
        if b == 0:
            assert np.isnan(got[0, 1]).all()
            rest = np.ones(got.shape[:2], bool)
            rest[0, 1] = False
            seen = rest & (np.arange(kv - n, kv) >= place)[:, None]
            for dim in (0, 31, 32, D // 2 + 5, D - 1):
                assert (got[:, :, dim][seen] == INF).all()
                ok[:, :, dim][seen] = True
            last = rest.copy()
            last[:-1] = False
            assert (got[:, :, D - 2][last] == -INF).all()
            ok[:, :, D - 2][last] = True
            ok[0, 1] = True
        assert ok.all()


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=["f16", "bf16-f16", "bf16", "f16-bf16"])
@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("below", [-6, -20])
def test_an_infinite_value_of_a_small_weight_is_infinite(gpu, plan, below, dtype, out_dtype):
    """The keys of positions 32 to 63 (one wave's) score 48 or 160 under the others: weights of 2^-69 and
    2^-230, under what 16 and 32 bits hold and over nothing."""
    s = planned(gpu, plan, 64, dtype)
    s.dq.fill_(1.0), s.q.fill(1.0)
    for pos in range(32, 64):
        for d in range(64):
            put(s, 0, pos, d, float(below), keys=True)
        s.keys[0][pos] = below
    put(s, 0, 40, 3, INF)
    for b, (got, ref, tol) in enumerate(rows_of(s, run(s, gpu, out_dtype=out_dtype), out_dtype)):
        if b == 0:
            assert (got[:, :, 3] == INF).all()
            got, ref, tol = (np.delete(x, 3, -1) for x in (got, ref, tol))
        assert (np.abs(got - ref) <= tol).all()


@pytest.mark.parametrize("plan", ["few-split", "many-split"])
def test_an_infinite_value_of_a_run_of_small_weights_is_infinite(gpu, plan):
    """As above, with the first 2560 keys, more than a workgroup's run."""
    s = planned(gpu, plan, 64)
    s.dq.fill_(1.0), s.q.fill(1.0)
    for pos in range(0, 2560, s.page):
        s.kc[int(s.table[0, pos // s.page])] = -20.0
    s.keys[0][:2560] = -20.0
    put(s, 0, 40, 3, INF)
    for b, (got, ref, tol) in enumerate(rows_of(s, run(s, gpu))):
        if b == 0:
            assert (got[:, :, 3] == INF).all()
            got, ref, tol = (np.delete(x, 3, -1) for x in (got, ref, tol))
        assert (np.abs(got - ref) <= tol).all()


def check_weights(gpu, lens, D, dtype, out_dtype, **kw):
    """Queries with one dimension, so that a score is one product, exact in fp32 but for two roundings of
    2^-24 of at most 16 (base 2): 2^-19; exp2 2^-22; weights of two terms 2^-16 (bf16) or 2^-21 (fp16); the sum
    over at most 6000 keys, whose partial sums of 4 x 4 x 32 keys and runs are short, 2^-17. The rows are off by half
    a step of their own, by its size there, and those."""
    s = make(gpu, lens, 4, 2, D, dtype=dtype)
    keep = np.arange(s.T * 4).reshape(s.T, 4, 1) * 7 % D == np.arange(D)
    s.q = np.where(keep, np.clip(s.q, -3, 3), 0.0)
    s.dq = torch.from_numpy(s.q.reshape(s.T, 4 * D)).to(dtype).to(gpu)
    s.q = s.dq.double().cpu().numpy().reshape(s.T, 4, D)
    out = run(s, gpu, scale=0.5, out_dtype=out_dtype, **kw).double().cpu().numpy().reshape(s.T, 4, D)
    bits = 10 if out_dtype == F16 else 7
    for b, (n, kv) in enumerate(lens):
        r = slice(s.cu[b], s.cu[b] + n)
        ref, size = attend(s.q[r], s.keys[b], s.values[b], kv, 0.5)
        off = (2.0 ** -16 if dtype == BF16 else 2.0 ** -21) + 2.0 ** -18 + 2.0 ** -22 + 2.0 ** -17
        _, e = np.frexp(np.abs(ref) + off * size)
        half_step = 2.0 ** np.maximum(e - 2 - bits, -25 if out_dtype == F16 else -134)
        assert (np.abs(out[r] - ref) <= half_step + off * size).all(), np.max((np.abs(out[r] - ref) - half_step) / size)


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=["f16", "bf16-f16", "bf16", "f16-bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 1), (1, 700), (1, 65)], [(5, 333), (8, 900)], [(2, 6000)]],
                         ids=["tokens", "drafts", "split"])
def test_weights_of_few_rows_keep_more_bits_than_the_rows(gpu, lens, D, dtype, out_dtype):
    check_weights(gpu, lens, D, dtype, out_dtype)


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=["f16", "bf16-f16", "bf16", "f16-bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(70, 333), (129, 129)], [(60, 6000)], [(40, 3000), (1, 5000)]], ids=["many", "split", "both"])
def test_full_weights_of_many_rows_keep_more_bits_than_the_rows(gpu, lens, D, dtype, out_dtype):
    check_weights(gpu, lens, D, dtype, out_dtype, full_weights=True)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n,q_scale", [(2, 1.5), (60, 1.5), (2, 12.0), (60, 12.0)], ids=["few", "many", "few-wide", "many-wide"])
@pytest.mark.parametrize("cap", [0.25, 2.0, 12.0, 30.0, 88.0, 89.0, 1e3, 1e4, 1e5, 1e6, 1e8, 1e12, 1e30, 1e38, 3.4e38])
def test_a_cap_of_any_size_keeps_the_weights(gpu, cap, n, q_scale, dtype):
    """Queries with one dimension and one-hot values: a score is one product, exact in fp32, and the rows are the
    weights themselves. A score is off by three roundings of 2^-24, the polynomial's 2^-24.4 and its
    evaluation's 2^-22 of itself, or 2^-20.6 where the other form gives it: 2^-20 of the largest capped score, or,
    for caps up to 88.8 (128 in base 2), by 2^-21.5 of 88.8: 2^-15. That is what a weight is off by,
    and so is their sum; a weight's 16 bits, the row's, 64 additions and exp2 come on top. Weights are held
    as fp16 with the largest at 2^7 or more, those under 2^-14 in steps of 2^-24: half of one is 2^-32 of the row."""
    D = kv = 64
    s = make(gpu, [(n, kv)], 4, 2, D, dtype=dtype, q_scale=q_scale)
    keep = np.arange(n * 4).reshape(n, 4, 1) * 7 % D == np.arange(D)
    s.q = np.where(keep, s.q, 0.0)
    s.dq = torch.from_numpy(s.q.reshape(n, 4 * D)).to(dtype).to(gpu)
    s.values[0] = np.repeat(np.eye(kv)[:, None], 2, 1)
    page = torch.from_numpy(pack_values(np.repeat(np.eye(kv)[None, None], 2, 1))).to(gpu).to(dtype)
    s.vc[int(s.table[0, 0])] = page[0]
    got = run(s, gpu, scale=0.5, softcap=cap).double().cpu().numpy().reshape(n, 4, D)
    ref, _ = attend(s.q, s.keys[0], s.values[0], kv, 0.5, 0, cap)
    score = np.einsum("nhd,khd->nhk", s.q, np.repeat(s.keys[0].astype(np.float64), 2, 1)) * 0.5
    most = np.abs(cap * np.tanh(score / cap)).max()
    off = 2 * (2.0 ** -15 + 2.0 ** -20 * most + 2.0 ** -22) + 2.0 ** -18
    weight = 2.0 ** -16 if dtype == BF16 else 2.0 ** -11     # two terms where rows leave with more bits
    assert (np.abs(got - ref) <= (off + weight + 2.0 ** -11) * ref + 2.0 ** -25 + 2.0 ** -32).all(), \
        np.nanmax(np.abs(got - ref) / (ref + 2.0 ** -14))


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("lens", [[(1, 1), (3, 40)], [(2, 6000)], [(70, 90), (1, 1)], [(60, 5000)]],
                         ids=["few", "few-split", "many", "many-split"])
def test_values_near_the_largest_of_bf16(gpu, lens, D):
    """Values of up to 4.5 2^118, the rows' among them; and one key whose value is the largest there is."""
    s = make(gpu, lens, 4, 2, D, dtype=BF16)
    s.vc *= 2.0 ** 118
    s.values = [v.astype(np.float64) * 2.0 ** 118 for v in s.values]
    for got, ref, tol in rows_of(s, run(s, gpu, out_dtype=BF16), BF16):
        assert (np.abs(got - ref) <= tol).all()
    s = make(gpu, [(n, n) for n, _ in lens], 4, 2, D, dtype=BF16)
    most = float(torch.finfo(BF16).max)
    for b, (n, _) in enumerate(s.lens):
        put(s, b, 0, 3, most)
        s.values[b][0, :, 3] = most
    out = run(s, gpu, out_dtype=BF16)
    for got, ref, tol in rows_of(s, out, BF16):
        assert (np.abs(got - ref) <= tol).all()
        assert (got[0, :, 3] == most).all()                  # the row that sees it alone


def test_large_values_of_no_weight_add_nothing(gpu):
    """Keys that score 160 under the others (2^-230) hold values of 2^120, in one wave's block and in a run."""
    for lens, upto in (([(1, 100)], 32), ([(2, 6000)], 2560)):
        s = make(gpu, lens, 4, 2, 64, dtype=BF16)
        s.dq.fill_(1.0), s.q.fill(1.0)
        for pos in range(upto):
            s.keys[0][pos] = -20.0
        for at in range(-(-upto // 64)):
            page, n = int(s.table[0, at]), min(64, upto - at * 64)
            mark = np.zeros((1, 1, 64, 64), np.float32)
            mark[0, 0, :n] = 1
            for c, pack, x in ((s.kc, pack_keys, -20.0), (s.vc, pack_values, 2.0 ** 120)):
                c[page][:, torch.from_numpy(pack(mark)).to(gpu)[0, 0].bool()] = x
        # the sums of such values times 2^-230 are 2^-110
        s.values[0][:upto] = 0.0
        for got, ref, tol in rows_of(s, run(s, gpu, out_dtype=BF16), BF16):
            assert (np.abs(got - ref) <= tol).all()


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("plan", PLANS)
def test_sums_of_the_largest_values_of_bf16_stay_in_range(gpu, plan, D):
    """Every value one of the largest bf16 numbers, all of one sign in a dimension: rows of them."""
    s = planned(gpu, plan, D, BF16)
    most = float(torch.finfo(BF16).max)
    for b in range(len(s.lens)):
        s.values[b] = np.broadcast_to(np.where(np.arange(D) % 3 == 0, -most, most), s.values[b].shape)
    big = np.broadcast_to(np.where(np.arange(D) % 3 == 0, -most, most).astype(np.float32), (s.vc.shape[0], 2, s.page, D))
    s.vc = torch.from_numpy(pack_values(np.ascontiguousarray(big))).to(gpu).to(BF16)
    for got, ref, tol in rows_of(s, run(s, gpu, out_dtype=BF16), BF16):
        assert (np.abs(got - ref) <= tol).all()
