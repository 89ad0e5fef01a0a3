"""Attention calls whose tiles are partly whole and partly split over their keys, and calls whose sequences are
found by other means, against 64 bits."""

import numpy as np
import pytest
import torch

from tests.paged import Sequences, attention_tolerance, pack_keys, pack_values

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def check(gpu, lens, H, KV, D, dtype=F16, out_dtype=F16, max_q=None, max_kv=None, window=0, cap=0.0, seed=0):
    """The call against attention in 64 bits on the GPU, one sequence and key/value head at a time."""
    from raceline_amd import ops

    s = Sequences(lens, 64, seed)
    g = torch.Generator(device=gpu).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device=gpu).to(dtype)    # noqa: E731
    q, k, v = rand(s.T, H * D) * 1.5, rand(s.n_pages, KV, 64, D), rand(s.n_pages, KV, 64, D)
    kc, vc = (torch.from_numpy(pack(x.float().cpu().numpy())).to(gpu).to(dtype) for x, pack in ((k, pack_keys), (v, pack_values)))
    out = torch.full((s.T + 1, H * D), 7.0, dtype=out_dtype, device=gpu)
    max_q, max_kv = max_q or s.max_q, max_kv or s.max_kv
    cu, kv, table = s.dev(gpu)
    for o in (out, again := out.clone()):
        ops.attention(q, kc, vc, cu, kv, table, max_q, max_kv, window=window, softcap=cap, out=o[:s.T])
    torch.cuda.synchronize()
    assert torch.equal(out, again) and (out[s.T:] == 7).all()
    G, scale = H // KV, D ** -0.5
    for b, (n, length) in enumerate(lens):
        if not n:
            continue
        pages = torch.from_numpy(s.table[b, :-(-length // 64)].astype(np.int64)).to(gpu)
        r = slice(s.cu[b], s.cu[b] + n)
        pos = torch.arange(length - n, length, device=gpu)[:, None]
        at = torch.arange(length, device=gpu)
        hide = at > pos
        if window:
            hide |= at <= pos - window
        for h in range(KV):
            K, V = (c[pages, h].reshape(-1, D)[:length].double() for c in (k, v))
            Q = q[r].view(n, KV, G, D)[:, h].double().reshape(n * G, D)
            x = torch.matmul(Q, K.t().contiguous()) * scale
            if cap:
                x = cap * torch.tanh(x / cap)
            w = torch.softmax(x.view(n, G, length).masked_fill(hide[:, None], -float("inf")), -1).view(n * G, length)
            ref, size = torch.matmul(w, V), torch.matmul(w, V.abs())
            tol = attention_tolerance(ref.cpu().numpy(), size.cpu().numpy(), Q.cpu().numpy(), K.cpu().numpy()[:, None],
                                      length, scale, cap, dtype, out_dtype)
            got = out[r].view(n, KV, G, D)[:, h].double().reshape(n * G, D)
            assert ((got - ref).abs().cpu().numpy() <= tol).all(), f"sequence {b}, head {h}"


def scratch(lens, H, KV, D):
    from raceline_amd import ops

    T, tiles = sum(n for n, _ in lens), sum(-(-n * (H // KV) // 128) for n, _ in lens)
    n = ops.attention_workspace_bytes(T, H, KV, D, len(lens), max(n for n, _ in lens), max(k for _, k in lens))
    return n, tiles * KV * 2 * 128 * (D + 2) * 4            # and what splitting all tiles in two would take


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (BF16, F16), (BF16, BF16)], ids=["f16", "bf16-f16", "bf16"])
@pytest.mark.parametrize("lens,H,KV,D", [([(2048, 4096)], 20, 4, 256), ([(1230, 5000)], 64, 8, 128), ([(1100, 5000)], 64, 2, 64),
                                         ([(1200, 4000), (860, 3000)], 20, 4, 256)],
                         ids=["256", "128", "64", "two"])
def test_whole_and_split_tiles_in_one_call(gpu, lens, H, KV, D, dtype, out_dtype):
    some, all_ = scratch(lens, H, KV, D)
    assert 0 < some < all_                                  # fewer than all of them are split
    check(gpu, lens, H, KV, D, dtype, out_dtype)


def test_whole_and_split_tiles_beside_sequences_of_few_rows(gpu):
    lens = [(1, 3000), (2048, 4096), (5, 2500), (0, 40), (1, 1)]
    some, all_ = scratch(lens, 20, 4, 256)
    assert 0 < some < all_
    check(gpu, lens, 20, 4, 256)


@pytest.mark.parametrize("window,cap", [(1500, 0.0), (0, 20.0), (0, 1e5)])
def test_whole_and_split_tiles_with_windows_and_caps(gpu, window, cap):
    check(gpu, [(2048, 4096)], 20, 4, 256, window=window, cap=cap)


@pytest.mark.parametrize("lens", [[(7 + 13 * i % 90, 1500 + 97 * i % 1500) for i in range(20)],
                                  [(1 + 29 * i % 300, 1 + 29 * i % 300 + 61 * i % 700) for i in range(40)],
                                  [(33 * (i % 3), 900 + i) for i in range(63)],
                                  [(8 + i % 9, 3000 - i) for i in range(64)]], ids=["20", "40", "63", "64"])
def test_more_sequences_than_are_ranked(gpu, lens):
    """More split tiles than the plan counts, sequences without rows, the last that fit a wave's lanes and one more."""
    check(gpu, lens, 20, 4, 128)


@pytest.mark.parametrize("max_q,max_kv", [(1, 3000), (1, 1), (300, 100), (10**6, 10**6)])
def test_split_calls_with_wrong_bounds(gpu, max_q, max_kv):
    check(gpu, [(300, 2900), (1, 3000), (40, 41)], 16, 4, 128, max_q=max_q, max_kv=max_kv)
