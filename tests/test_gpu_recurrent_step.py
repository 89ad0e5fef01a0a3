"""The recurrent layer's operators together, as a decoding step runs them: the stacked in projection, causal_conv,
gated_delta with its gate, the out projection into the residual stream, over a prompt, drafts of which a part is
taken, and single tokens; and the choice of the tokens at the end. Every operator is held to 64 bits on what the one
before it gave, so each keeps its own tolerance."""

import numpy as np
import pytest
import torch

import oracle as O
from raceline_amd.model import Engine
from tests import model_files as MF
from tests import recurrent as R
from tests.qdata import make_layer, upload_mlx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_prompt_drafts_and_tokens(gpu, dtype):
    from raceline_amd import ops

    Hk, Hv, D, hid, taps = 2, 4, 64, 256, 4
    C, E = (2 * Hk + Hv) * D, Hv * D
    # rows of the in projection: the convolution's channels, z, b and a
    lay = {n: make_layer(i + 5, N, K) for i, (n, N, K) in enumerate([("in", C + E + 2 * Hv, hid), ("out", hid, E)])}
    pw = {n: ops.pack_affine(*upload_mlx(*w, "f16", gpu)) for n, w in lay.items()}
    W = {n: ops.dequant(p).cpu().numpy().astype(np.float64) for n, p in pw.items()}
    rng = np.random.default_rng(3)
    par = {n: rng.standard_normal(s).astype(np.float32) for n, s in dict(w=(C, taps), a_log=Hv, dt=Hv, norm=D).items()}
    par["dt"] -= 3
    p = {n: torch.from_numpy(x).to(gpu) for n, x in par.items()}
    P = {n: x.astype(np.float64) for n, x in par.items()}
    cs, ds = ops.conv_state(5, C, taps, gpu), ops.delta_state(5, Hv, D, D, gpu)
    cs.fill_(float("nan")), ds.fill_(float("nan"))
    n = lambda t: t.float().cpu().numpy().astype(np.float64)                             # noqa: E731
    # (rows, tokens with them) of two sequences, and how many rows are kept: a prompt, a draft looked at and then taken
    # in part, tokens, a second prompt chunk
    steps = [([(70, 70), (33, 33)], None), ([(4, 74), (1, 34)], [0, 1]), ([(4, 74), (0, 34)], [2, 0]),
             ([(1, 73), (3, 37)], [1, 3]), ([(1, 74), (1, 38)], None), ([(50, 124), (1, 39)], None)]
    for step, (lens, keep) in enumerate(steps):
        s = R.Sequences(lens)
        s.slots[:], s.n_slots = [3, 1], 5
        seqs = s.dev(gpu)
        kp = None if keep is None else torch.tensor(keep, dtype=torch.int32, device=gpu)
        x = torch.from_numpy(rng.standard_normal((s.T, hid)).astype(np.float16)).to(gpu)
        h0 = rng.standard_normal((s.T, hid)).astype(np.float32)
        h = torch.from_numpy(h0.copy()).to(gpu)
        before = n(cs), n(ds)
        rows = ops.linear(x, pw["in"])
        y = ops.causal_conv(rows[:, :C], p["w"], cs, *seqs, keep=kp, out_dtype=dtype)
        o = ops.gated_delta(y[:, :Hk * D], y[:, Hk * D:2 * Hk * D], y[:, 2 * Hk * D:], rows[:, C + E + Hv:], rows[:, C + E:C + E + Hv],
                            p["a_log"], p["dt"], ds, *seqs, max_q=s.max_q, z=rows[:, C:C + E], norm=p["norm"], keep=kp)
        ops.linear(o, pw["out"], out=h, accum=True)
        torch.cuda.synchronize()

        O.check_close(n(rows), n(x) @ W["in"].T, 1e-3, f"step {step}: in")
        r, got = n(rows), (n(cs), n(ds))
        for b, (m, kv) in enumerate(lens):
            at, slot = slice(s.cu[b], s.cu[b] + m), s.slots[b]
            goes_on, end = kv > m, m if keep is None else max(0, min(keep[b], m))
            old = before[0][slot] if goes_on else np.zeros((taps - 1, C))
            ref, size = R.conv(r[at, :C], P["w"], None, True, old)
            tol = 1.1 * (2 * taps + 1) * R.EPS * size + 8 * R.EPS * size + R.half_step(dtype, ref)
            assert (np.abs(n(y)[at] - ref) <= tol).all(), f"step {step}: convolution"
            if end:
                assert np.array_equal(got[0][slot], np.concatenate([old, r[at, :C]])[end:end + taps - 1])
            heads = lambda v, H: v.reshape(m, H, D)                                      # noqa: E731
            yy = n(y)[at]
            S0 = before[1][slot] if goes_on else np.zeros((Hv, D, D))
            ref, S, tol, off = R.delta(heads(yy[:, :Hk * D], Hk), heads(yy[:, Hk * D:2 * Hk * D], Hk), heads(yy[:, 2 * Hk * D:], Hv),
                                       r[at, C + E + Hv:], r[at, C + E:C + E + Hv], P["a_log"], P["dt"], S0, D ** -0.5,
                                       z=heads(r[at, C:C + E], Hv), norm=P["norm"], keep=end)
            tol = tol + R.half_step(torch.float16, np.abs(ref) + tol)
            assert (np.abs(n(o)[at].reshape(m, Hv, D) - ref) <= tol).all(), f"step {step}: delta rule"
            if end:
                assert (np.abs(got[1][slot] - S) <= off[:, None, :]).all(), f"step {step}: state"
            elif m:
                assert np.array_equal(got[1][slot], before[1][slot], equal_nan=True)
        O.check_close(n(h) - h0, n(o) @ W["out"].T, 1e-3, f"step {step}: out")


def test_the_choice_at_the_end_of_a_step(gpu, tmp_path):
    """Head, adjustments and choice: tokens by the definition from the logits that the step gave."""
    from raceline_amd import ops

    m = MF.write_dense_model(str(tmp_path / "m.rlm"), vocab=1000)
    rng = np.random.default_rng(8)
    h = torch.from_numpy(rng.standard_normal((3, m.cfg["hidden_size"])).astype(np.float32)).to(gpu)
    dev = lambda a: torch.from_numpy(a).to(gpu)                                          # noqa: E731
    with Engine(m.path, max_chunk=16) as e:
        logits = e.head(h)[:, :e.vocab]
        mask = rng.integers(-2**31, 2**31, (3, -(-e.vocab // 32))).astype(np.int32)
        logits = ops.adjust_logits(logits, tokens=dev(rng.integers(0, e.vocab, (3, 40)).astype(np.int32)),
                                   repetition=dev(np.full(3, 1.3, np.float32)), allowed=dev(mask))
        u, p, t = rng.random(3), np.array([0.9, 0.5, 1.0], np.float32), np.array([0.7, 1.2, 0.0], np.float32)
        tokens = ops.sample(logits, dev(u), temperature=dev(t), top_p=dev(p)).cpu().numpy()
        x = logits.cpu().numpy()
        for r in range(3):
            want, _, near = R.choose(x[r], u[r], float(t[r]), 0, float(p[r]))
            assert near > 1e-9 and tokens[r] == want
            assert mask.view(np.uint32)[r][tokens[r] // 32] >> (tokens[r] % 32) & 1
        assert tokens[2] == e.top_k_device(logits[2].contiguous(), 1)[0][0]
