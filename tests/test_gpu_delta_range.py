"""gated_delta over the range of fp32: values that fade by more than fp32 spans, rows
whose squares pass fp32, values next to the smallest ones, columns far smaller than others of their head."""

import numpy as np
import pytest
import torch

from tests import recurrent as R
from tests.test_gpu_delta import BF16, check, draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_q", [1, 300], ids=["tokens", "chunks"])
@pytest.mark.parametrize("state,first,later", [
    (1e6, 0.0, 0.0), (1e8, 0.0, 0.0), (1e9, 0.0, 0.0), (2.0 ** 116, 0.0, 0.0), (2.0 ** 116, 0.0, 2.0 ** -30),
    (0.3, 2.0 ** 116, 2.0 ** -30), (0.0, 2.0 ** 116, 2.0 ** -60), (2.0 ** 100, 2.0 ** 100, 2.0 ** -100)])
@pytest.mark.parametrize("heads", ["h64", "k128"])
def test_what_is_forgotten_leaves_no_trace(gpu, heads, state, first, later, max_q):
    """A chunk that forgets all, in front of values that may be smaller by more than fp32 spans. Every token fades by e^-9.9
    or more, so nothing of the first 64 rows reaches those behind the next 64 (e^-630), and these and the state are held to
    the rule's own bounds; what stands in front has to be finite."""
    from raceline_amd import ops

    s, c = draw([(200, 300), (70, 70)], heads, BF16, seed=11, state=1.0)
    Hv, Dk, Dv = c["state"].shape[1:]
    c["a"] = c["a"] + 1e3
    c["state"] = (np.clip(c["state"], -4, 4) * state).astype(np.float32).astype(np.float64)
    size = np.where(np.arange(len(c["v"])) < 64, first, later)[:, None, None]
    c["v"] = torch.from_numpy(np.clip(c["v"], -4, 4) * size).bfloat16().double().numpy()
    f = lambda n, t=torch.float32: torch.from_numpy(c[n]).to(t).to(gpu)                  # noqa: E731
    st = f("state")
    out = ops.gated_delta(*(f(n, BF16).flatten(1) for n in "qkv"), f("a"), f("b"), f("a_log"), f("dt_bias"), st, *s.dev(gpu),
                          max_q=max_q, out_dtype=BF16)
    torch.cuda.synchronize()
    assert out.isfinite().all() and st.isfinite().all()
    args = [c[n][:200] for n in "qkvab"]
    ref, S, tol, off = R.delta(*args, c["a_log"], c["dt_bias"], c["state"][s.slots[0]], Dk ** -0.5)
    tol = (tol + R.half_step(BF16, np.abs(ref) + tol))[128:]
    got = out[128:200].double().cpu().numpy().reshape(72, Hv, Dv)
    assert (np.abs(got - ref[128:]) <= tol).all()
    assert (np.abs(st[int(s.slots[0])].double().cpu().numpy() - S) <= off[:, None, :] + 1e-37).all()


@pytest.mark.parametrize("max_q", [1, 300], ids=["tokens", "chunks"])
@pytest.mark.parametrize("heads", ["h64", "wide", "256", "one"])
@pytest.mark.parametrize("size", [2.0 ** 58, 2.0 ** 70, 2.0 ** 110])
def test_rows_whose_squares_pass_fp32_are_normalised(gpu, size, heads, max_q):
    s, c = draw([(90, 100), (2, 5), (70, 70)], heads, BF16, seed=5)
    c["v"] = torch.from_numpy(c["v"] * size).bfloat16().double().numpy()
    c["state"] = (c["state"] * size).astype(np.float32).astype(np.float64)
    c["v"][:, 0] /= 2.0 ** 60                                  # another head of ordinary rows beside them
    c["state"][:, 0] /= 2.0 ** 60
    check(gpu, s, c, BF16, True, out_dtype=BF16, max_q=max_q)


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -112, 2.0 ** -118])
@pytest.mark.parametrize("heads", ["h64", "k128"])
def test_values_next_to_the_smallest(gpu, size, heads):
    s, c = draw([(90, 100), (2, 5), (70, 70)], heads, BF16, seed=6)
    c["v"] = torch.from_numpy(c["v"] * size).bfloat16().double().numpy()
    c["state"] = (c["state"] * size).astype(np.float32).astype(np.float64)
    for max_q in (1, 300):
        check(gpu, s, c, BF16, out_dtype=BF16, max_q=max_q)


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("gate", [False, True], ids=["plain", "gated"])
def test_small_columns_keep_their_bits_without_a_fade(gpu, dk, gate):
    """Keys and queries of one element, weights of 1 and no fade: after each token the state's row of its key is its value,
    and its output that row. Every number on the way is a whole one of at most 8 bits times a power of two, so fp32 and
    the operands of chunks hold it exactly, unless its unit lies below the last bit that they keep: 2^-39 of the bound that
    a head's values are held by. Values here are up to 127; after n chunks the bound is 127 (9 + 8 sqrt(n)) at most,
    and units of 2^-21 (2^-28 of the largest value) are kept for 32768 rows; 127 (9 + 8 n), a sum of lengths in place of their
    squares', would lose them from 130 chunks on."""
    from raceline_amd import ops

    T, dv = 32768, 64
    g = torch.Generator(device=gpu)
    g.manual_seed(3)
    order = torch.cat([torch.randperm(dk, generator=g, device=gpu) for _ in range(T // dk)])
    rows = torch.zeros(T, dk, device=gpu, dtype=BF16)
    rows[torch.arange(T, device=gpu), order] = 1
    v = torch.randint(-127, 128, (T, dv), generator=g, device=gpu).float()
    v[:, 0] = 127
    v[:, 1::2] *= 2.0 ** -21
    ints = dict(dtype=torch.int32, device=gpu)
    a, b, zero = torch.full((T, 1), -1e30, device=gpu), torch.full((T, 1), 1e30, device=gpu), torch.zeros(1, device=gpu)
    state = ops.delta_state(1, 1, dk, dv)
    extra = dict(z=torch.full((T, dv), 1e30, device=gpu), norm=torch.ones(dv, device=gpu)) if gate else {}
    out = ops.gated_delta(rows, rows, v.bfloat16(), a, b, zero, zero, state, torch.tensor([0, T], **ints), torch.tensor([T], **ints),
                          torch.tensor([0], **ints), max_q=T, scale=1.0, eps=1e-37, out_dtype=BF16, **extra)
    want = torch.empty(dk, dv, device=gpu)
    want[order[-dk:]] = v[-dk:]
    assert torch.equal(state[0, 0], want)
    if not gate:
        assert torch.equal(out.float(), v)


def test_more_sequences_than_chunks_are_for(gpu):
    """A batch whose heads are past the chunked form takes a large max_q too: every sequence as in a call of its own."""
    from raceline_amd import ops

    Hk, Hv, Dk, Dv, B, most = 1, 32, 64, 128, 33000, 1 << 20
    rng = np.random.default_rng(8)
    lens = np.zeros(B, np.int64)
    lens[rng.choice(B, 40, replace=False)] = rng.integers(1, 4, 40)
    lens[[0, 777, B - 1]] = 5, 150, 2
    cu = np.concatenate([[0], np.cumsum(lens)])
    T, used = int(cu[-1]), np.nonzero(lens)[0]
    slots = np.full(B, -1)
    slots[used] = rng.permutation(len(used))
    assert ops.gated_delta_workspace_bytes(T, Hk, Hv, Dk, Dv, B, most) == 0
    ints = dict(dtype=torch.int32, device=gpu)
    g = torch.Generator(device=gpu)
    g.manual_seed(4)
    rnd = lambda *n: torch.randn(n, generator=g, device=gpu)                             # noqa: E731
    x, ba = rnd(T, 2 * Hk * Dk + Hv * Dv).bfloat16(), rnd(T, 2 * Hv)
    a_log, dt, start = rnd(Hv) - 2, rnd(Hv) - 3, rnd(len(used), Hv, Dk, Dv)

    def run(state, lo, hi, cu, kv, slots, max_q):
        r = slice(lo, hi)
        return ops.gated_delta(x[r, :Dk], x[r, Dk:2 * Dk], x[r, 2 * Dk:], ba[r, :Hv], ba[r, Hv:], a_log, dt, state,
                               torch.tensor(cu, **ints), torch.tensor(kv, **ints), torch.tensor(slots, **ints), max_q=max_q,
                               out_dtype=BF16)

    together, alone = start.clone(), start.clone()
    whole = run(together, 0, T, cu, lens + 3, slots, most)
    for b in used:
        rows = run(alone, int(cu[b]), int(cu[b + 1]), [0, lens[b]], [lens[b] + 3], [slots[b]], 1)
        assert torch.equal(rows, whole[cu[b]:cu[b + 1]]), b
    assert torch.equal(together, alone)


@pytest.mark.parametrize("max_q", [1, 300], ids=["tokens", "chunks"])
@pytest.mark.parametrize("heads,size,norm_eps", [("256", 2.0 ** 61, 1e38), ("256", 2.0 ** 62, 3e38), ("h64", 2.0 ** 64, 3e38), ("h64", 1.0, 3e38)])
def test_large_rows_beside_a_large_norm_eps(gpu, heads, size, norm_eps, max_q):
    """Squares whose sum, or whose mean with eps, passes fp32."""
    s, c = draw([(90, 100), (2, 5), (70, 70)], heads, BF16, seed=5)
    c["v"] = torch.from_numpy(c["v"] * size).bfloat16().double().numpy()
    c["state"] = (c["state"] * size).astype(np.float32).astype(np.float64)
    c["norm"] = c["norm"] * 2.0 ** 10
    check(gpu, s, c, BF16, True, out_dtype=BF16, max_q=max_q, scale=1.0, norm_eps=float(np.float32(norm_eps)))
