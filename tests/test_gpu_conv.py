"""causal_conv against its definition in 64 bits: taps, lengths from none to many runs, states, kept rows,
strides and channel counts that the wide loads do not take."""

import numpy as np
import pytest
import torch

from tests import recurrent as R

pytestmark = pytest.mark.gpu


def check(gpu, lens, C, taps=4, dtype=torch.float16, bias=False, silu=True, keep=None, pad=0, seed=0, slots=None,
          more_rows=0, scale=1.0):
    from raceline_amd import ops

    rng = np.random.default_rng(seed)
    s = R.Sequences(lens, seed=seed)
    if slots is not None:
        s.slots[:] = slots
    T = s.T + more_rows
    rows = (rng.standard_normal((max(T, 1), C + pad)) * scale).astype(np.float32)
    rows[s.T:] = np.nan
    w = rng.standard_normal((C, taps)).astype(np.float32)
    bs = rng.standard_normal(C).astype(np.float32) if bias else None
    state = rng.standard_normal((s.n_slots, taps - 1, C)).astype(np.float32)
    dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(gpu)      # noqa: E731
    st, out = dev(state), torch.full((T, C + pad), 7.0, dtype=dtype, device=gpu)
    kp = None if keep is None else dev(np.array(keep, np.int32))
    got = ops.causal_conv(dev(rows)[:T, :C], dev(w), st, *s.dev(gpu), bias=dev(bs), silu=silu, keep=kp, out=out[:, :C])
    torch.cuda.synchronize()
    y = got.float().cpu().numpy()
    want_state = state.copy()
    for b, (n, kv) in enumerate(lens):
        at, mine = s.cu[b], s.has_state(b)
        before = state[s.slots[b]] if mine and kv > n else np.zeros((taps - 1, C), np.float32)
        x = rows[at:at + n, :C]
        ref, size = R.conv(*(v.astype(np.float64) for v in (x, w)), None if bs is None else bs.astype(np.float64), silu,
                           before.astype(np.float64))
        # the sums: taps products and additions; SiLU's slope is below 1.1; its exponential's argument is
        # off by |y| 2^-24, which moves y sigmoid(y) by less than |y| 2^-24, and a few roundings
        tol = 1.1 * (2 * taps + 1) * R.EPS * size + 8 * R.EPS * np.abs(size) + R.half_step(dtype, ref)
        assert (np.abs(y[at:at + n] - ref) <= tol).all(), f"sequence {b}"
        end = n if keep is None else max(0, min(keep[b], n))
        if mine and end:
            want_state[s.slots[b]] = np.concatenate([before, x])[end:end + taps - 1]
    assert np.array_equal(st.cpu().numpy(), want_state)
    assert (out.float().cpu().numpy()[s.T:] == 7).all() and (out.float().cpu().numpy()[:, C:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("taps", [2, 3, 4])
def test_lengths_and_taps(gpu, taps, dtype):
    lens = [(1, 1), (1, 9), (2, 2), (0, 5), (3, 40), (15, 15), (16, 17), (17, 17), (33, 70), (0, 0), (100, 100)]
    check(gpu, lens, 64, taps, dtype, bias=taps == 3, seed=taps)


@pytest.mark.parametrize("C,pad", [(1, 0), (7, 0), (260, 0), (1000, 3), (8192, 4096), (64, 1)])
def test_channels_and_strides(gpu, C, pad):
    check(gpu, [(5, 60), (19, 19)], C, 4, pad=pad, seed=C)


def test_without_the_activation(gpu):
    check(gpu, [(9, 30), (40, 41)], 128, silu=False, bias=True)


def test_kept_rows(gpu):
    keep = [0, 1, 2, 3, 4, 5, 9, -3, 1]
    check(gpu, [(5, 30), (5, 30), (5, 5), (5, 30), (5, 30), (5, 30), (5, 30), (5, 30), (50, 60)], 64, keep=keep)


def test_sequences_without_a_state(gpu):
    check(gpu, [(4, 30), (20, 30), (2, 2)], 64, slots=[-1, 5, 1])     # 5 is behind the last slot
    check(gpu, [(4, 30)], 64, slots=[2**31 - 1])


def test_padded_batch_and_no_rows(gpu):
    check(gpu, [(4, 30), (20, 30)], 64, more_rows=37)
    check(gpu, [(0, 3), (0, 0)], 64, more_rows=2)


def test_many_sequences(gpu):
    check(gpu, [(1 + i % 3, 1 + i % 3 + (i % 5) * 7) for i in range(200)], 32, seed=3)


def test_large_and_small_values(gpu):
    check(gpu, [(30, 60)], 64, dtype=torch.bfloat16, scale=1e30, silu=False)
    check(gpu, [(30, 60)], 64, dtype=torch.bfloat16, scale=30.0)
    check(gpu, [(30, 60)], 64, scale=1e-6)


def test_other_sequences_do_not_reach_a_row(gpu):
    """NaN in one sequence's rows and state stays there."""
    from raceline_amd import ops

    s = R.Sequences([(6, 20), (7, 20), (5, 5)])
    rows, w = torch.randn((s.T, 64), device=gpu), torch.randn((64, 4), device=gpu)
    state = torch.randn((s.n_slots, 3, 64), device=gpu)
    want_state = state.clone()
    want = ops.causal_conv(rows, w, want_state, *s.dev(gpu))
    rows[6:13] = float("nan")
    state[int(s.slots[1])] = float("inf")
    state[int(s.slots[2])] = float("nan")            # begins from zeros all the same
    got = ops.causal_conv(rows, w, state, *s.dev(gpu))
    assert torch.equal(got[:6], want[:6]) and torch.equal(got[13:], want[13:]) and got[6:13].isnan().all()
    for b in (0, 2):
        assert torch.equal(state[int(s.slots[b])], want_state[int(s.slots[b])])


LONG = [(15, 15), (16, 40), (17, 17), (33, 60), (0, 3), (1, 9), (1050, 1050), (31, 32), (2, 2), (1040, 3000)]


@pytest.mark.parametrize("taps,C,pad", [(4, 8192, 0), (3, 8192, 0), (2, 8192, 4), (4, 2051, 0), (3, 2048, 1), (2, 2048, 3), (4, 8196, 0)])
def test_long_calls_in_runs_of_sixteen(gpu, taps, C, pad):
    """Calls of 2048 waves and more take runs of 16 tokens: with wide loads 8192 channels a wave of 256, else a wave of 64."""
    rows = sum(n for n, _ in LONG)
    wide = C % 4 == 0 and pad % 4 == 0
    assert rows // 16 * -(-C // (64 * (4 if wide else 1))) >= 2048
    check(gpu, LONG, C, taps, torch.bfloat16 if taps == 3 else torch.float16, bias=taps != 2, pad=pad, seed=C + taps, more_rows=9)


@pytest.mark.parametrize("C", [8192, 2049])
def test_kept_rows_of_long_calls(gpu, C):
    check(gpu, LONG, C, keep=[15, 3, 0, 32, 7, 1, 1049, 16, 1, 2], silu=C != 2049, seed=C, slots=[0, 1, 2, 3, 4, 5, 6, -1, 7, 8])
