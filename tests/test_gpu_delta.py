"""gated_delta against the rule token by token in 64 bits: head layouts, lengths around the chunks' borders,
states, kept rows, strides, strong and weak fades, keys that are alike, zero or huge."""

import numpy as np
import pytest
import torch

from tests import recurrent as R

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
HEADS = {"k128": (2, 4, 128, 128), "one": (1, 1, 128, 64), "h64": (3, 3, 64, 64), "wide": (1, 3, 64, 256),
         "mixed": (2, 2, 64, 128), "256": (1, 2, 128, 256)}


def draw(lens, heads, dtype, seed=0, alike=0.7, size=1.0, fade=1.0, state=0.3):
    Hk, Hv, Dk, Dv = HEADS[heads]
    rng = np.random.default_rng(seed)
    s = R.Sequences(lens, seed=seed)
    T = max(s.T, 1)
    to = lambda x: torch.from_numpy(x).to(dtype).double().numpy()                        # noqa: E731
    c = dict(q=to(rng.standard_normal((T, Hk, Dk)) * size), v=to(rng.standard_normal((T, Hv, Dv)) * size),
             k=to((rng.standard_normal((T, Hk, Dk)) + alike * rng.standard_normal((Hk, Dk))) * size),
             a=rng.standard_normal((T, Hv)), b=rng.standard_normal((T, Hv)) * 2,
             a_log=np.log(rng.uniform(0.01, 4, Hv) * fade), dt_bias=rng.standard_normal(Hv) - 2,
             z=rng.standard_normal((T, Hv, Dv)) * 2, norm=1 + 0.2 * rng.standard_normal(Dv),
             state=rng.standard_normal((s.n_slots, Hv, Dk, Dv)) * state)
    for n in ("a", "b", "a_log", "dt_bias", "z", "norm", "state"):
        c[n] = c[n].astype(np.float32).astype(np.float64)
    return s, c


def check(gpu, s, c, dtype, gate=False, out_dtype=F16, keep=None, max_q=None, pad=0, more_rows=0, eps=1e-6, scale=None,
          norm_eps=1e-6):
    from raceline_amd import ops

    T, (Hk, Dk), (Hv, Dv) = s.T + more_rows, c["q"].shape[1:], c["v"].shape[1:]

    def rows(x, t):
        """A slice of wider rows, NaN behind the sequences' own."""
        x = x.reshape(len(x), -1)
        y = torch.full((T, x.shape[1] + pad), float("nan"), dtype=t)
        y[:s.T, :x.shape[1]] = torch.from_numpy(x[:s.T]).to(t)
        return y.to(gpu)[:, :x.shape[1]]

    f = torch.float32
    dev = lambda x: torch.from_numpy(x.copy()).to(f).to(gpu)                             # noqa: E731
    st, out = dev(c["state"]), torch.full((T, Hv * Dv + pad), 7.0, dtype=out_dtype, device=gpu)
    kw = dict(z=rows(c["z"], f), norm=dev(c["norm"])) if gate else {}
    kp = None if keep is None else torch.tensor(keep, dtype=torch.int32, device=gpu)
    ops.gated_delta(rows(c["q"], dtype), rows(c["k"], dtype), rows(c["v"], dtype), rows(c["a"], f), rows(c["b"], f),
                    dev(c["a_log"]), dev(c["dt_bias"]), st, *s.dev(gpu), max_q=s.max_q if max_q is None else max_q,
                    scale=scale, eps=eps, norm_eps=norm_eps, keep=kp, out=out[:, :Hv * Dv], **kw)
    torch.cuda.synchronize()
    y, got = out.double().cpu().numpy(), st.double().cpu().numpy()
    want = c["state"].copy()
    for i, (n, kv) in enumerate(s.lens):
        at, mine = slice(s.cu[i], s.cu[i] + n), s.has_state(i)
        S0 = c["state"][s.slots[i]] if mine and kv > n else np.zeros((Hv, Dk, Dv))
        extra = dict(z=c["z"][at], norm=c["norm"], norm_eps=norm_eps) if gate else {}
        ref, S, tol, off = R.delta(c["q"][at], c["k"][at], c["v"][at], c["a"][at], c["b"][at], c["a_log"], c["dt_bias"],
                                   S0, Dk ** -0.5 if scale is None else scale, eps,
                                   keep=None if keep is None else keep[i], **extra)
        tol = tol + R.half_step(out_dtype, np.abs(ref) + tol)
        wrong = np.abs(y[at, :Hv * Dv].reshape(n, Hv, Dv) - ref) > tol
        assert not wrong.any(), f"sequence {i}: rows {np.unique(np.nonzero(wrong)[0])[:8]}"
        if mine and n and (keep is None or keep[i] > 0):
            slot = s.slots[i]
            assert (np.abs(got[slot] - S) <= off[:, None, :] + 1e-37).all(), f"state of sequence {i}"
            want[slot] = got[slot]
    assert np.array_equal(got, want)                           # the other slots stay as they were
    assert (y[s.T:] == 7).all() and (y[:, Hv * Dv:] == 7).all()
    return y, got


LENS = [(1, 1), (1, 50), (0, 9), (2, 2), (63, 100), (64, 64), (65, 65), (0, 0), (130, 200), (17, 17)]


@pytest.mark.parametrize("gate", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads", HEADS)
def test_lengths_and_heads(gpu, heads, dtype, gate):
    s, c = draw(LENS, heads, dtype, seed=len(heads))
    check(gpu, s, c, dtype, gate, out_dtype=BF16 if gate and dtype is BF16 else F16)


@pytest.mark.parametrize("max_q", [0, 1, 8, 64, 100000])
def test_results_stay_right_past_max_q(gpu, max_q):
    s, c = draw([(3, 3), (70, 90), (1, 4)], "k128", F16, seed=4)
    check(gpu, s, c, F16, True, max_q=max_q)


@pytest.mark.parametrize("lens", [[(1, 7)], [(5, 50)] * 9, [(1, 30)] * 70], ids=["token", "drafts", "users"])
def test_decoding(gpu, lens):
    s, c = draw(lens, "k128", BF16, seed=7)
    check(gpu, s, c, BF16, True)


@pytest.mark.parametrize("pad", [1, 2, 4, 8, 24])
def test_strides(gpu, pad):
    s, c = draw([(5, 9), (70, 70)], "one", F16, seed=pad)
    check(gpu, s, c, F16, True, pad=pad)
    check(gpu, s, c, F16, True, pad=pad, max_q=1)


def test_kept_rows(gpu):
    s, c = draw([(5, 30)] * 6 + [(5, 5)], "k128", F16, seed=1)
    check(gpu, s, c, F16, True, keep=[0, 1, 4, 5, 9, -2, 3])
    check(gpu, s, c, F16, True, keep=[0, 1, 4, 5, 9, -2, 3], max_q=1000)
    s, c = draw([(150, 300)] * 6 + [(1, 9), (70, 70)], "h64", F16, seed=2)
    check(gpu, s, c, F16, False, keep=[0, 1, 63, 64, 65, 149, 0, 69])


def test_kept_rows_are_the_start_of_the_next_call(gpu):
    """A draft of which three of five tokens are taken leaves what those three alone leave, bit for bit."""
    s, c = draw([(5, 30), (5, 5)], "k128", F16, seed=9)
    t, d = draw([(3, 28), (3, 3)], "k128", F16, seed=9)
    for n in ("q", "k", "v", "a", "b", "z"):
        d[n] = np.concatenate([c[n][:3], c[n][5:8]])
    for n in ("a_log", "dt_bias", "norm", "state"):
        d[n] = c[n]
    y, got = check(gpu, s, c, F16, True, keep=[3, 3])
    y3, got3 = check(gpu, t, d, F16, True)
    assert (got == got3).all() and (y[[0, 1, 2, 5, 6, 7]] == y3).all()


def test_sequences_without_a_state(gpu):
    s, c = draw([(3, 30), (70, 90), (2, 9), (2, 2)], "h64", F16)
    s.slots[:] = [-1, 6, 1, 2**31 - 1]
    check(gpu, s, c, F16)


def test_padded_batch_and_no_rows(gpu):
    s, c = draw([(3, 30), (70, 90)], "one", F16)
    check(gpu, s, c, F16, True, more_rows=80)
    s, c = draw([(0, 3), (0, 0)], "one", F16)
    check(gpu, s, c, F16, more_rows=2, max_q=100)


@pytest.mark.parametrize("fade", [1e-6, 1.0, 1e3, 1e30], ids=["none", "some", "strong", "all"])
def test_fades(gpu, fade):
    s, c = draw([(150, 200), (3, 9)], "h64", F16, seed=5, fade=fade)
    check(gpu, s, c, F16, True)
    check(gpu, s, c, F16, True, max_q=1)


def test_a_fade_that_comes_and_goes(gpu):
    """Tokens that forget all, between tokens that forget nothing: sums of logarithms that differ widely."""
    s, c = draw([(200, 300)], "h64", F16, seed=6)
    c["a"][:] = -30
    c["a"][::7] = 90
    c["a"][3::31] = 3e4
    check(gpu, s, c, F16)


@pytest.mark.parametrize("alike", [0.0, 30.0, 1e3])
def test_keys_that_are_alike(gpu, alike):
    s, c = draw([(140, 140), (64, 90)], "k128", BF16, seed=8, alike=alike)
    c["b"][:] = 40                                             # beta 1: corrections as strong as they get
    c["a"][:] = -40                                            # no fade
    check(gpu, s, c, BF16)


@pytest.mark.parametrize("size", [1e-3, 30.0, 6000.0])
def test_sizes_of_rows(gpu, size):
    s, c = draw([(90, 100), (2, 5)], "k128", F16, seed=3, size=size, state=size)
    check(gpu, s, c, F16 if size < 6000 else F16, out_dtype=BF16)
    check(gpu, s, c, F16, True, max_q=1)


@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_sizes_of_bf16_rows(gpu, size):
    s, c = draw([(90, 100), (2, 5)], "h64", BF16, seed=3)
    c["q"], c["k"] = c["q"] * 2.0 ** 60, c["k"] * 2.0 ** -40    # lengths of 2^63, and far below eps
    c["v"] = torch.from_numpy(c["v"] * size).bfloat16().double().numpy()
    c["state"] = (c["state"] * size).astype(np.float32).astype(np.float64)
    check(gpu, s, c, BF16, out_dtype=BF16, eps=1e-30)


@pytest.mark.parametrize("size", [2.0 ** -70, 2.0 ** -90, 2.0 ** -120])
def test_rows_whose_squares_pass_below_fp32(gpu, size):
    """Keys and queries far shorter than eps: the state takes next to nothing, and nothing overflows."""
    s, c = draw([(90, 100), (70, 70)], "h64", BF16, seed=4)
    c["k"][::3] *= size
    c["q"][::2] *= size
    check(gpu, s, c, BF16, out_dtype=BF16)
    check(gpu, s, c, BF16, out_dtype=BF16, max_q=1)


def test_runs_of_chunks(gpu):
    """A prompt of more chunks than the scratch holds at a time, in one call and in two: the state goes from run to
    run as it goes from call to call, but for the power of two its parts are held at (two terms of 2^-22)."""
    from raceline_amd import ops

    Hk, Hv, Dk, Dv, T, cut = 16, 32, 128, 128, 6400, 64 * 40
    assert ops.gated_delta_workspace_bytes(T, Hk, Hv, Dk, Dv, 1, T) == ops.gated_delta_workspace_bytes(2 * T, Hk, Hv, Dk, Dv, 1, T)
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    rnd = lambda *n: torch.randn(n, generator=g, device=gpu)                             # noqa: E731
    x, ba, z = rnd(T, 2 * Hk * Dk + Hv * Dv).half(), rnd(T, 2 * Hv), rnd(T, Hv * Dv)
    a_log, dt, norm, start = rnd(Hv) - 2, rnd(Hv) - 3, rnd(Dv), rnd(1, Hv, Dk, Dv) * 0.3

    def run(state, lo, hi, slot=0):
        ints = dict(dtype=torch.int32, device=gpu)
        r = slice(lo, hi)
        return ops.gated_delta(x[r, :Hk * Dk], x[r, Hk * Dk:2 * Hk * Dk], x[r, 2 * Hk * Dk:], ba[r, :Hv], ba[r, Hv:], a_log, dt,
                               state, torch.tensor([0, hi - lo], **ints), torch.tensor([hi + 9], **ints),
                               torch.tensor([slot], **ints), max_q=T, z=z[r], norm=norm, out_dtype=BF16)

    one, two, none = start.clone(), start.clone(), start.clone()
    whole = run(one, 0, T)
    parts = torch.cat([run(two, 0, cut), run(two, cut, T)])
    assert (one - two).norm() <= 2.0 ** -18 * two.norm()
    assert (whole.float() - parts.float()).norm() <= 2.0 ** -8 * parts.float().norm()
    # a sequence without a slot goes through the runs all the same, from zeros
    free = run(none, 0, T, slot=-1)
    zeros = torch.zeros_like(start)
    assert torch.equal(none, start) and torch.equal(free, run(zeros, 0, T))


def test_runs_of_chunks_over_many_sequences(gpu):
    """More sequences than a run of chunks can touch, some without rows, one longer than a run: each as if alone (as in
    test_runs_of_chunks where a run ends inside one, else to the bit)."""
    from raceline_amd import ops

    Hk, Hv, Dk, Dv = 16, 32, 128, 128
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(0, 150, 100)]
    lens[3], lens[40], lens[99] = 0, 64 * 70 + 5, 1
    B, cu = len(lens), np.concatenate([[0], np.cumsum(lens)])
    T = int(cu[-1]) + 3                                        # rows behind the last sequence too
    ints = dict(dtype=torch.int32, device=gpu)
    g = torch.Generator(device=gpu)
    g.manual_seed(2)
    rnd = lambda *n: torch.randn(n, generator=g, device=gpu)                             # noqa: E731
    x, ba = rnd(T, 2 * Hk * Dk + Hv * Dv).half(), rnd(T, 2 * Hv)
    a_log, dt, start = rnd(Hv) - 2, rnd(Hv) - 3, rnd(B, Hv, Dk, Dv) * 0.3
    most = 1 << 20
    assert ops.gated_delta_workspace_bytes(T, Hk, Hv, Dk, Dv, B, most) == ops.gated_delta_workspace_bytes(2 * T, Hk, Hv, Dk, Dv, B, most)

    def run(state, lo, hi, cu, kv, slots):
        r = slice(lo, hi)
        out = torch.full((hi - lo, Hv * Dv), 7.0, dtype=F16, device=gpu)
        return ops.gated_delta(x[r, :Hk * Dk], x[r, Hk * Dk:2 * Hk * Dk], x[r, 2 * Hk * Dk:], ba[r, :Hv], ba[r, Hv:], a_log, dt,
                               state, torch.tensor(cu, **ints), torch.tensor(kv, **ints), torch.tensor(slots, **ints),
                               max_q=most, out=out)

    kv = [n + 5 * (i % 2) for i, n in enumerate(lens)]
    together, alone = start.clone(), start.clone()
    whole = run(together, 0, T, cu.tolist(), kv, list(range(B)))
    assert (whole[cu[-1]:] == 7).all()
    same = 0
    for i, n in enumerate(lens):
        if not n:
            assert torch.equal(together[i], start[i])
            continue
        rows = run(alone, int(cu[i]), int(cu[i + 1]), [0, n], [kv[i]], [i])
        same += torch.equal(rows, whole[cu[i]:cu[i + 1]]) and torch.equal(alone[i], together[i])
        assert (alone[i] - together[i]).norm() <= 2.0 ** -18 * alone[i].norm(), i
        assert (rows.float() - whole[cu[i]:cu[i + 1]].float()).norm() <= 2.0 ** -10 * rows.float().norm(), i
    runs = -(-(T // 64 + 2 * B) // 60)                         # a run holds 60 chunks or more
    assert same >= sum(n > 0 for n in lens) - runs


def test_zero_rows_and_eps(gpu):
    s, c = draw([(80, 100), (2, 5)], "k128", F16, seed=3)
    c["k"][5:9] = 0
    c["q"][7:20] = 0
    c["v"][70:] = 0
    check(gpu, s, c, F16)
    check(gpu, s, c, F16, True, eps=3.0, scale=0.5, norm_eps=0.1)


def test_other_sequences_do_not_reach_a_row(gpu):
    from raceline_amd import ops

    s, c = draw([(6, 20), (70, 90), (66, 66)], "h64", F16)
    f = lambda n, t=torch.float32: torch.from_numpy(c[n]).to(t).to(gpu)                  # noqa: E731
    args = {n: f(n, F16).reshape(s.T, -1) for n in "qkv"} | {n: f(n) for n in "ab"}

    def run(args, state):
        return ops.gated_delta(*args.values(), f("a_log"), f("dt_bias"), state, *s.dev(gpu), max_q=s.max_q)

    good = f("state")
    want = run(args, good)
    for name in args:
        for value in (float("nan"), float("inf"), -float("inf")):
            bad = {n: x.clone() for n, x in args.items()}
            bad[name][6:76] = value
            state = f("state")
            state[int(s.slots[1])] = value
            state[int(s.slots[2])] = value                     # begins from zeros all the same
            got = run(bad, state)
            assert torch.equal(got[:6], want[:6]) and torch.equal(got[76:], want[76:]), (name, value)
            for b in (0, 2):
                assert torch.equal(state[int(s.slots[b])], good[int(s.slots[b])])


def test_the_same_call_gives_the_same_bits(gpu):
    s, c = draw([(130, 200), (5, 9), (64, 64)], "k128", F16, seed=2)
    first = check(gpu, s, c, F16, True)
    again = check(gpu, s, c, F16, True)
    assert all(np.array_equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("where", ["value", "state", "kept"])
def test_what_is_not_finite_stays_in_its_column(gpu, where, value):
    """In chunks a head's values are held by the size of the largest one; the others keep their bits beside an infinity."""
    from raceline_amd import ops

    s, c = draw([(70, 90), (130, 130)], "k128", BF16, seed=6)
    f = lambda n, t=torch.float32: torch.from_numpy(c[n]).to(t).to(gpu)                  # noqa: E731
    keep = torch.tensor([66, 100], dtype=torch.int32, device=gpu) if where == "kept" else None

    def run(x):
        v, state = f("v", BF16), f("state")
        if where == "state":
            state[int(s.slots[0]), 1, :, 5] = x
        else:
            v[67, 1, 5] = v[70 + 69, 2, 100] = x
        out = ops.gated_delta(f("q", BF16).flatten(1), f("k", BF16).flatten(1), v.flatten(1), f("a"), f("b"), f("a_log"),
                              f("dt_bias"), state, *s.dev(gpu), max_q=s.max_q, keep=keep)
        return out.reshape(s.T, 4, 128), state

    (out, state), (want, kept) = run(value), run(0.0)
    touched = torch.zeros_like(want, dtype=torch.bool)
    of_state = torch.zeros_like(kept, dtype=torch.bool)
    first = 0 if where == "state" else 66 if where == "kept" else 64
    touched[first:70, 1, 5] = of_state[int(s.slots[0]), 1, :, 5] = True
    if where != "state":
        touched[70 + 64:, 2, 100] = of_state[int(s.slots[1]), 2, :, 100] = True
    if where == "kept":
        of_state[int(s.slots[0])] = False                      # the row lies behind the kept ones
    assert torch.equal(out[~touched], want[~touched]) and torch.equal(state[~of_state], kept[~of_state])
    assert not out[69, 1, 5].isfinite() and (not of_state.any() or not state[of_state].isfinite().any())


def test_a_largest_value_is_forgotten_with_its_rows(gpu):
    """Rates are 0.01 at least, so a token fades by e^-9.9 or more: the first chunk's last tokens, which are held by its
    largest value, still reach the second chunk, and nothing of them the third (e^-600 is 0 in fp32)."""
    from raceline_amd import ops

    s, c = draw([(200, 200)], "h64", BF16, seed=7)
    f = lambda n, t=torch.float32: torch.from_numpy(c[n]).to(t).to(gpu)                  # noqa: E731

    def run(x):
        v, state = f("v", BF16), f("state")
        v[3, 1, 5] = x
        out = ops.gated_delta(f("q", BF16).flatten(1), f("k", BF16).flatten(1), v.flatten(1), f("a") + 1e3, f("b"), f("a_log"),
                              f("dt_bias"), state, *s.dev(gpu), max_q=s.max_q)
        return out[128:], state

    for x, y in zip(run(torch.finfo(BF16).max), run(0.0)):
        assert x.isfinite().all() and torch.equal(x, y)
