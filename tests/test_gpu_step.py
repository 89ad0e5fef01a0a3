"""The operators together, as a decoding step runs them: the stacked qkv linear, rope_append, attention,
the o linear into the residual stream, over a prompt, a draft's tokens and single tokens of two
sequences; and the head's logits through adjust_logits into the top-k. Every operator is held to 64
bits on what the one before it gave, so each keeps its own tolerance."""

import numpy as np
import pytest
import torch

import oracle as O
from raceline_amd.model import Engine, top_k
from tests import model_files as MF
from tests.paged import Sequences, attend, attention_tolerance, unpack_keys, unpack_values
from tests.qdata import make_layer, upload_mlx
from tests.test_gpu_logits import reference
from tests.test_gpu_rope import rotate, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_prompt_draft_and_tokens(gpu, dtype):
    from raceline_amd import ops

    H, KV, D, hid, page = 4, 2, 64, 256, 32
    lay = {n: make_layer(i + 5, N, K) for i, (n, N, K) in enumerate([("qkv", (H + 2 * KV) * D, hid), ("o", hid, H * D)])}
    pw = {n: ops.pack_affine(*upload_mlx(*w, "f16", gpu)) for n, w in lay.items()}
    W = {n: ops.dequant(p).cpu().numpy().astype(np.float64) for n, p in pw.items()}
    freq = ops.rope_frequencies(32, scaling="parts", factor=4, low=1, high=8, original=64, device=gpu)
    kc, vc = ops.kv_cache(20, KV, D, page, dtype, gpu)
    kc.fill_(float("nan")), vc.fill_(float("nan"))
    rng = np.random.default_rng(3)
    steps = [[(70, 70), (33, 33)], [(3, 73), (1, 34)], [(1, 72), (4, 38)], [(1, 73), (0, 38)], [(40, 113), (1, 39)]]
    order = rng.permutation(20)
    for step, lens in enumerate(steps):         # the third takes one of the draft's tokens back
        s = Sequences(lens, page)
        s.table = np.stack([order[:10], order[10:]]).astype(np.int32)
        cu, kv, table = s.dev(gpu)
        x = torch.from_numpy(rng.standard_normal((s.T, hid)).astype(np.float16)).to(gpu)
        h0 = rng.standard_normal((s.T, hid)).astype(np.float32)
        h = torch.from_numpy(h0.copy()).to(gpu)
        rows = ops.linear(x, pw["qkv"])
        q = ops.rope_append(rows[:, :H * D], rows[:, H * D:(H + KV) * D], rows[:, (H + KV) * D:], kc, vc, cu, kv, table,
                            freq, mscale=1.1)
        a = ops.attention(q, kc, vc, cu, kv, table, s.max_q, s.max_kv, window=90)
        ops.linear(a, pw["o"], out=h, accum=True)
        torch.cuda.synchronize()

        n = lambda t: t.float().cpu().numpy().astype(np.float64)                   # noqa: E731
        O.check_close(n(rows), n(x) @ W["qkv"].T, 1e-3, f"step {step}: qkv")
        pos = np.concatenate([np.arange(k - m, k) for m, k in lens])
        r = n(rows).reshape(s.T, H + 2 * KV, D)
        y, size = rotate(r[:, :H + KV], pos, freq.cpu().numpy(), False, 1.1)
        tol = tolerance(y, size, False, dtype)
        assert (np.abs(n(q).reshape(s.T, H, D) - y[:, :H]) <= tol[:, :H]).all()
        K, V = unpack_keys(n(kc)), unpack_values(n(vc))
        for b, (m, length) in enumerate(lens):
            at = slice(s.cu[b], s.cu[b] + m)
            keys, vals = (c.transpose(0, 2, 1, 3)[s.table[b]].reshape(-1, KV, D)[:length] for c in (K, V))
            assert (np.abs(keys[length - m:] - y[at, H:]) <= tol[at, H:]).all()
            assert np.isfinite(keys).all() and np.isfinite(vals).all()
            qs = n(q)[at].reshape(m, H, D)
            ref, size = attend(qs, keys, vals, length, D ** -0.5, 90)
            ok = attention_tolerance(ref, size, qs, keys, length, D ** -0.5, 0.0, dtype, torch.float16)
            assert (np.abs(n(a)[at].reshape(m, H, D) - ref) <= ok).all(), f"step {step}: attention"
        O.check_close(n(h) - h0, n(a) @ W["o"].T, 1e-3, f"step {step}: o")


def test_logits_before_the_top_k(gpu, tmp_path):
    from raceline_amd import ops

    m = MF.write_dense_model(str(tmp_path / "m.rlm"), vocab=1000)
    rng = np.random.default_rng(8)
    h = torch.from_numpy(rng.standard_normal((3, m.cfg["hidden_size"])).astype(np.float32)).to(gpu)
    with Engine(m.path, max_chunk=16) as e:
        logits = e.head(h)[:, :e.vocab]
        tokens = rng.integers(0, e.vocab, (3, 40)).astype(np.int32)
        mask = rng.integers(-2**31, 2**31, (3, -(-e.vocab // 32))).astype(np.int32)
        dev = lambda a: torch.from_numpy(a).to(gpu)                                # noqa: E731
        rep = np.full(3, 1.3, np.float32)
        out = ops.adjust_logits(logits, tokens=dev(tokens), repetition=dev(rep), allowed=dev(mask))
        x = logits.cpu().numpy()
        for r in range(3):
            ids, vals = e.top_k_device(out[r].contiguous(), 5)
            y, size = reference(x[r], tokens[r], rep=rep[r], allowed=mask[r])
            want, _ = top_k(out[r].cpu().numpy(), 5)
            assert list(want) == ids
            best = np.sort(y)[::-1][:5]
            assert np.abs(np.array(vals) - best).max() <= 6 * 2.0 ** -24 * size.max()
            assert all(mask.view(np.uint32)[r][i // 32] >> (i % 32) & 1 for i in ids)
