"""sample against its definition in 64 bits: every filter alone and together, ties, masks that leave one token or none,
infinities and NaN, rows from one token to a whole vocabulary."""

import numpy as np
import pytest
import torch

from tests import recurrent as R

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def run(gpu, x, u, T=None, k=None, p=None, m=None, pad=0):
    from raceline_amd import ops

    rows, V = x.shape
    wide = torch.full((rows, V + pad), 1e9, device=gpu)
    wide[:, :V] = torch.from_numpy(x).to(gpu)
    vec = lambda v, t: None if v is None else torch.tensor(np.broadcast_to(v, rows).copy(), dtype=t, device=gpu)  # noqa: E731
    probs = torch.empty(rows, device=gpu)
    f = torch.float32
    tokens = ops.sample(wide[:, :V], vec(u, torch.float64), temperature=vec(T, f), top_k=vec(k, torch.int32),
                        top_p=vec(p, f), min_p=vec(m, f), probs=probs)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), probs.cpu().numpy()


def check(gpu, x, u, T=None, k=None, p=None, m=None, pad=0):
    x = np.asarray(x, np.float32)
    rows = len(x)
    tokens, probs = run(gpu, x, u, T, k, p, m, pad)
    at = lambda v, r, d, t: d if v is None else t(np.broadcast_to(v, rows)[r])                # noqa: E731
    f32 = lambda v: float(np.float32(v))                                                      # noqa: E731
    for r in range(rows):
        with np.errstate(over="ignore"):
            want, share, near = R.choose(x[r], at(u, r, 0.0, float), at(T, r, 1.0, f32), at(k, r, 0, int), at(p, r, 1.0, f32),
                                         at(m, r, 0.0, f32))
        if near > 1e-9:        # steps of 2^-44 and their sums: what a border can be off by
            assert tokens[r] == want, f"row {r}: {tokens[r]} for {want}"
            # a weight's step is off by 2^-45 of the largest: nothing beside fp32 where a token is likely enough
            # to be drawn; the share is rounded once
            assert abs(probs[r] - share) <= share * 2.0 ** -23 + 2.0 ** -40
    return tokens


def rows_of(rng, rows, V, spread=2.5):
    return (rng.standard_normal((rows, V)) * spread).astype(np.float32)


FILTERS = {"none": {}, "k": dict(k=7), "p": dict(p=0.8), "m": dict(m=0.05), "kp": dict(k=50, p=0.9),
           "all": dict(k=60, p=0.95, m=0.02, T=0.7), "hot": dict(T=3.0, p=0.5), "cold": dict(T=0.05, k=5),
           "wide": dict(p=0.999), "k1": dict(k=1), "large k": dict(k=900), "k past the row": dict(k=10**9)}


@pytest.mark.parametrize("filters", FILTERS)
@pytest.mark.parametrize("V", [1, 2, 5, 63, 1000, 4096, 4097, 12345])
def test_filters(gpu, V, filters):
    rng = np.random.default_rng(V)
    check(gpu, rows_of(rng, 9, V), rng.random(9), **FILTERS[filters])


@pytest.mark.parametrize("filters", ["none", "kp", "p", "m", "wide"])
def test_a_whole_vocabulary(gpu, filters):
    rng = np.random.default_rng(5)
    check(gpu, rows_of(rng, 5, 248320), rng.random(5), **FILTERS[filters])


def test_parameters_of_each_row(gpu):
    rng = np.random.default_rng(6)
    n = 40
    check(gpu, rows_of(rng, n, 3001), rng.random(n), T=rng.uniform(0.1, 3, n), k=rng.integers(-1, 400, n),
          p=rng.uniform(0.01, 1.2, n), m=rng.uniform(-0.1, 0.3, n))


@pytest.mark.parametrize("pad", [1, 2, 3, 4])
def test_strides(gpu, pad):
    rng = np.random.default_rng(pad)
    check(gpu, rows_of(rng, 5, 5001), rng.random(5), k=40, p=0.9, pad=pad)


def test_every_number_gives_its_token(gpu):
    """One row, many numbers: the kept tokens come out in order of index, each with its share."""
    rng = np.random.default_rng(3)
    x = np.repeat(rows_of(rng, 1, 700), 2000, 0)
    u = (np.arange(2000) + 0.5) / 2000
    got = check(gpu, x, u, k=20, p=0.95)
    assert (np.diff(got) >= 0).all() and len(set(got)) > 5


def test_ties_go_to_the_lowest_index(gpu):
    V = 9000
    x = np.zeros((6, V), np.float32)
    x[:, 100::7] = 1.0
    x[2, ::2] = -0.0                       # both zeros are one
    u = np.array([0.0, 0.3, 0.99, 0.5, 0.9, 0.1])
    for f in (dict(k=10), dict(k=1300), dict(p=0.2), dict(p=0.5), dict(k=1300, p=0.9), dict(T=0.0), dict(m=0.5), dict(m=1.0)):
        check(gpu, x, u, **f)
    y = np.full((3, 248320), 2.5, np.float32)
    check(gpu, y, [0.0, 0.5, 0.9999], p=0.7)
    check(gpu, y, [0.0, 0.5, 0.9999], k=12345)


def test_greedy(gpu):
    rng = np.random.default_rng(1)
    x = np.round(rows_of(rng, 30, 20000) * 2) / 2          # many ties for the largest
    for T in (0.0, -1.0, NAN):
        assert np.array_equal(run(gpu, x, rng.random(30), T=T)[0], x.argmax(1))


def test_masked_rows(gpu):
    rng = np.random.default_rng(2)
    x = rows_of(rng, 8, 6000)
    x[0] = -INF                                            # nothing is left
    x[1, :4321] = -INF
    x[1, 4322:] = -INF                                     # one token
    x[2, ::2] = NAN
    x[3] = NAN
    x[4] = np.finfo(np.float32).min                        # a mask of the lowest value leaves all alike
    x[5, 1:] = np.finfo(np.float32).min
    x[6, 50:] = -INF
    x[7, 17] = INF
    for f in ({}, dict(k=5), dict(p=0.9), dict(k=100, p=0.5, m=0.1, T=0.3), dict(T=0.0), dict(T=INF)):
        tokens = check(gpu, x, rng.random(8), **f)
        assert tokens[0] == -1 and tokens[3] == -1 and tokens[1] == 4321 and tokens[7] == 17
        assert (tokens[[2, 4, 5, 6]] >= 0).all() and tokens[6] < 50 and tokens[2] % 2


def test_two_infinite_logits_share(gpu):
    x = np.zeros((2, 500), np.float32)
    x[:, [7, 300]] = INF
    assert list(run(gpu, x, [0.2, 0.8])[0]) == [7, 300]
    assert list(run(gpu, x, [0.2, 0.8], p=0.4)[0]) == [7, 7]


def test_parameters_out_of_range(gpu):
    rng = np.random.default_rng(4)
    x = rows_of(rng, 8, 900)
    u = rng.random(8)
    free = run(gpu, x, u)[0]
    for f in (dict(k=-5), dict(k=0), dict(p=1.0), dict(p=7.0), dict(p=NAN), dict(m=0.0), dict(m=-1.0), dict(m=NAN), dict(T=1.0)):
        assert np.array_equal(run(gpu, x, u, **f)[0], free), f
    first = x.argmax(1)
    for f in (dict(p=0.0), dict(p=-1.0), dict(m=1.0), dict(m=5.0), dict(k=1), dict(T=1e-30), dict(T=1e-45)):
        assert np.array_equal(run(gpu, x, u, **f)[0], first), f
    last = run(gpu, x, np.ones(8))[0]                      # a number past the range: the last kept token
    assert np.array_equal(last, run(gpu, x, np.full(8, 5.0))[0]) and (last >= 0).all()
    assert np.array_equal(run(gpu, x, np.full(8, -1.0))[0], run(gpu, x, np.zeros(8))[0])
    assert np.array_equal(run(gpu, x, np.full(8, NAN))[0], run(gpu, x, np.zeros(8))[0])


def test_sharp_and_flat_rows(gpu):
    rng = np.random.default_rng(7)
    x = rows_of(rng, 6, 30000)
    check(gpu, x * 1e3, rng.random(6), p=0.9)
    check(gpu, x * 1e-6, rng.random(6), p=0.9)
    check(gpu, x * 1e30, rng.random(6), T=1e30, p=0.6)
    check(gpu, x * 1e-3, rng.random(6), k=29999)


def test_after_adjust_logits(gpu):
    """The end of a step: biases and a grammar's mask, then the choice."""
    from raceline_amd import ops

    rng = np.random.default_rng(9)
    x = torch.from_numpy(rows_of(rng, 4, 5000)).to(gpu)
    mask = rng.integers(-2**31, 2**31, (4, 157)).astype(np.int32)
    mask[3] = 0
    y = ops.adjust_logits(x, allowed=torch.from_numpy(mask).to(gpu))
    got = check(gpu, y.cpu().numpy(), rng.random(4), p=0.9)
    assert got[3] == -1 and all(mask.view(np.uint32)[r][t // 32] >> (t % 32) & 1 for r, t in enumerate(got[:3]))


@pytest.mark.parametrize("V", [2**18 + 1, 2**22])
def test_the_largest_vocabularies(gpu, V):
    """Past 2^18 tokens a weight is held in steps of 2^-(62 - ceil(log2 V)) of the largest: each is off by half a step and their
    sum by V / 2 of them, so a share of a weight of W is off by less than V steps / W, and a number that lies farther from a
    border is on the right side of it."""
    rng = np.random.default_rng(V)
    step = 2.0 ** -(62 - int(np.ceil(np.log2(V))))
    flat = np.full((2, V), 2.5, np.float32)
    x = np.concatenate([rows_of(rng, 1, V), np.round(rows_of(rng, 1, V))])
    u = rng.random(2)
    told = 0
    for rows, f in ((flat, {}), (flat, dict(p=0.7)), (flat, dict(k=V - 1000)), (flat, dict(k=V // 3, p=0.5)), (x, {}), (x, dict(p=0.9)),
                    (x, dict(m=0.001)), (x, dict(k=100000, p=0.99, m=1e-4, T=0.9)), (x, dict(T=0.0))):
        tokens, probs = run(gpu, rows, u, **f)
        for r in range(2):
            T, p, m = (float(np.float32(f.get(n, d))) for n, d in (("T", 1.0), ("p", 1.0), ("m", 0.0)))
            want, share, border = R.choose(rows[r], u[r], T, f.get("k", 0), p, m)
            w = 1.0 if not T > 0 else np.exp((float(rows[r][want]) - float(rows[r].max())) / T)
            near = V * step * share / w
            if border > near:
                told += 1
                assert tokens[r] == want, (f, r)
                assert abs(probs[r] - share) <= share * 2.0 ** -23 + near, (f, r)
    assert told >= 16                                              # of 18
