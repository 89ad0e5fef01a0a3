"""adjust_logits against its definition in 64 bits, and in front of the engine's top-k."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, tokens=None, n=None, prompt=None, rep=None, pres=None, freq=None, ids=None, bias=None, allowed=None):
    """The adjusted row in 64 bits and the size that fp32's rounding goes by."""
    V = len(x)
    y = x.astype(np.float64)
    size = np.abs(y)
    t = np.array([], int) if tokens is None else np.asarray(tokens)[:len(tokens) if n is None else max(0, n)]
    made_t = t[max(0, prompt or 0):]
    said = np.bincount(t[(t >= 0) & (t < V)], minlength=V) > 0
    made = np.bincount(made_t[(made_t >= 0) & (made_t < V)], minlength=V)
    rep, pres, freq = (d if v is None else float(v) for v, d in ((rep, 1.0), (pres, 0.0), (freq, 0.0)))
    with np.errstate(invalid="ignore"):
        y = np.where(said, np.where(y > 0, y / rep, y * rep), y)
        size = np.maximum(size, np.abs(y))
        y = np.where(made > 0, y - freq * made - pres, y)
        size = size + np.where(made > 0, abs(freq) * made + abs(pres), 0)
        if ids is not None:
            for i, v in zip(ids, bias):
                if 0 <= i < V:
                    y[i] += float(v)
                    size[i] += abs(float(v)) * (np.asarray(ids) == i).sum()
    if allowed is not None:
        v = np.arange(V)
        y = np.where(allowed.view(np.uint32)[v // 32] >> (v % 32).astype(np.uint32) & 1, y, -np.inf)
    # past fp32's range by half a step or more (its lowest value times a penalty): rounds to infinity
    y = np.where(np.abs(y) >= 2.0 ** 128 * (1 - 2.0 ** -25), np.copysign(np.inf, y), y)
    return y, size


def check(gpu, rows, V, n=0, biases=0, mask=False, penalties=True, prompt=None, seed=0, pad=0, shared=False,
          edit=None, in_place=False):
    from raceline_amd import ops

    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, V)) * 4).astype(np.float32)
    kw, per = {}, 1 if shared else rows
    if n:
        kw["tokens"] = (rng.random((per, n)) ** 4 * (V + 3) - 2).astype(np.int32)    # some outside the vocabulary
        kw["n_tokens"] = rng.integers(0, n + 1, rows).astype(np.int32)
        kw["n_tokens"][0] = n
        if prompt is not None:
            kw["n_prompt"] = np.minimum(kw["n_tokens"], prompt).astype(np.int32)
    if penalties:
        kw["repetition"] = (0.7 + rng.random(rows)).astype(np.float32)
        kw["presence"], kw["frequency"] = (rng.random((2, rows)) - 0.3).astype(np.float32)
    if biases:
        kw["bias_ids"] = rng.integers(-1, V + 1, (per, biases)).astype(np.int32)
        kw["bias_ids"][:, biases // 2:] = kw["bias_ids"][:, :biases - biases // 2]   # half of them twice
        kw["bias"] = (rng.standard_normal((per, biases)) * 5).astype(np.float32)
    if mask:
        kw["allowed"] = rng.integers(-2**31, 2**31, (per, -(-V // 32) + pad)).astype(np.int32)
    if edit:
        edit(x, kw)
    big = torch.full((rows, V + pad), 9.0, device=gpu)
    big[:, :V] = torch.from_numpy(x).to(gpu)
    dev = {k: torch.from_numpy(np.ascontiguousarray(v)).to(gpu) for k, v in kw.items()}
    logits = big[:, :V]
    out = ops.adjust_logits(logits, **dev, out=logits if in_place else None)
    torch.cuda.synchronize()
    assert (big[:, V:] == 9).all()
    if not in_place:
        assert torch.equal(logits.cpu().nan_to_num(), torch.from_numpy(x).nan_to_num())
    got = out.cpu().numpy().astype(np.float64)
    for r in range(rows):
        row = {k: v[r if len(v) == rows else 0] for k, v in kw.items()}
        y, size = reference(x[r], row.get("tokens"), row.get("n_tokens"), row.get("n_prompt"), row.get("repetition"),
                            row.get("presence"), row.get("frequency"), row.get("bias_ids"), row.get("bias"),
                            row.get("allowed"))
        fin = np.isfinite(y)
        assert np.array_equal(got[r][~fin], y[~fin], equal_nan=True)
        # a quotient or product, two subtractions, a product and two additions: six half steps of fp32
        with np.errstate(invalid="ignore"):
            assert (np.abs(got[r] - y) <= 6 * 2.0 ** -24 * size)[fin].all()
    return out


@pytest.mark.parametrize("V", [1, 31, 33, 4095, 4096, 4097, 50001])
def test_vocabularies(gpu, V):
    check(gpu, 3, V, n=200, biases=7, mask=True, prompt=90)


@pytest.mark.parametrize("n", [1, 2, 255, 257, 5000])
@pytest.mark.parametrize("prompt", [None, 0, 100, 10**6])
def test_histories(gpu, n, prompt):
    check(gpu, 4, 9001, n=n, prompt=prompt)


@pytest.mark.parametrize("biases", [1, 2, 300, 1024])
def test_biases_with_ids_that_come_twice(gpu, biases):
    check(gpu, 3, 5000, biases=biases, penalties=False)


def test_the_same_token_always(gpu):
    def edit(x, kw):
        kw["tokens"][:] = 77

    check(gpu, 2, 300, n=70000, edit=edit)


def test_nothing_to_do(gpu):
    out = check(gpu, 2, 1000, penalties=False)
    assert out.shape == (2, 1000)


@pytest.mark.parametrize("pad", [1, 3])
def test_strides_shared_rows_and_in_place(gpu, pad):
    check(gpu, 5, 8193, n=60, biases=9, mask=True, pad=pad, shared=True, in_place=True)


def test_infinities_nan_and_a_mask_that_leaves_nothing(gpu):
    def edit(x, kw):
        x[0, ::7], x[0, 1::7], x[1, ::5] = np.inf, -np.inf, np.nan
        x[1, 1::5] = np.finfo(np.float32).min
        kw["allowed"][2] = 0

    out = check(gpu, 3, 3000, n=100, mask=True, edit=edit)
    assert (out[2] == -float("inf")).all()


def test_the_whole_vocabulary(gpu):
    check(gpu, 2, 248320, n=3000, biases=100, mask=True, prompt=1000)


def test_graph_and_stream(gpu):
    from raceline_amd import ops

    x = torch.randn((2, 9000), device=gpu)
    tokens = torch.randint(0, 9000, (2, 50), device=gpu, dtype=torch.int32)
    n = torch.tensor([50, 20], dtype=torch.int32, device=gpu)
    rep = torch.tensor([1.5, 1.1], device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = ops.adjust_logits(x, tokens, n, repetition=rep)
    other = ops.adjust_logits(x, tokens, n, repetition=rep, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(want, other)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.adjust_logits(x, tokens, n, repetition=rep)
    for k in (3, 40, 0):
        n.fill_(k)
        want = ops.adjust_logits(x, tokens, n, repetition=rep)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_masks_of_unsigned_words_and_one_row_for_all(gpu):
    from raceline_amd import ops

    x = torch.randn((3, 100), device=gpu)
    bits = np.array([0xF0F0F0F0, 1, 0x80000000, 0xF], np.uint32)
    want = np.where(np.unpackbits(bits.view(np.uint8), bitorder="little")[:100] == 1, x.cpu().numpy(), -np.inf)
    signed = torch.from_numpy(bits.view(np.int32)).to(gpu)
    for allowed in (signed, signed[None], signed.view(torch.uint32), signed.repeat(3, 1)):
        assert np.array_equal(ops.adjust_logits(x, allowed=allowed).cpu().numpy(), want)


def test_more_biases_than_threads_share_one_id(gpu):
    """1024 entries for one token add up in list order, in fp32."""
    from raceline_amd import ops

    rng = np.random.default_rng(5)
    b = rng.standard_normal(1024).astype(np.float32)
    total = np.float32(0)
    for v in b:
        total = np.float32(total + v)
    x = torch.zeros((1, 50), device=gpu)
    out = ops.adjust_logits(x, bias_ids=torch.full((1, 1024), 7, dtype=torch.int32, device=gpu),
                            bias=torch.from_numpy(b[None]).to(gpu)).cpu().numpy()
    assert out[0, 7] == total and (np.delete(out[0], 7) == 0).all()
