"""rope_append against the same in 64 bits: pair layouts, rotated parts of the head, norms, chunks that
begin and end inside blocks and pages, far positions, pages that are not there."""

import numpy as np
import pytest
import torch

from tests.paged import HALF_STEP, TINY, Sequences, unpack_keys, unpack_values

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def rotate(x, pos, freq, interleaved, m, w=None, eps=1e-6):
    """x [T][heads][D] in 64 bits; also, per element, the size that fp32's errors go by."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y, size, half = x.copy(), np.abs(x), len(freq)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    angle = pos[:, None].astype(np.float64) * freq
    c, s = m * np.cos(angle)[:, None], m * np.sin(angle)[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = m * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size


def tolerance(y, size, norm, dtype):
    """Half a step of the stored type, and fp32's: the angle is at most half a turn, off by 2^-25 of
    a turn (2 pi 2^-25 < 2^-22 radians), sincospi by 2^-22, the products and sum by 2^-23; the norm of up
    to 256 squares summed eight, then in pairs: under 2^-20."""
    return HALF_STEP[dtype] * np.abs(y) + (2.0 ** -20 + (2.0 ** -20 if norm else 0)) * size + TINY[dtype]


def check(gpu, lens, H, KV, D, page=64, dtype=F16, rot=None, interleaved=False, m=1.0, norm=False, base=1e4,
          pad=0, break_pages=(), seed=0, stream=None):
    from raceline_amd import ops

    rng = np.random.default_rng(seed)
    s = Sequences(lens, page, seed)
    for b, at in break_pages:
        s.table[b, at] = -1
    rot = D if rot is None else rot
    freq = base ** (-np.arange(0, rot, 2) / max(rot, 1))
    width = (H + 2 * KV) * D
    rows = torch.full((s.T + 2, width + pad), float("nan"), device=gpu)
    x = (rng.standard_normal((s.T, H + 2 * KV, D)) * 2).astype(np.float32)
    rows[:s.T, pad:] = torch.from_numpy(x.reshape(s.T, width)).to(gpu)
    rows = rows[:, pad:]
    w = [(1 + 0.3 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in range(2)]
    dw = [torch.from_numpy(t).to(gpu) if norm else None for t in w]
    kc, vc = ops.kv_cache(s.n_pages, KV, D, page, dtype, gpu)
    kc.fill_(3.0), vc.fill_(5.0)
    out = torch.full((s.T + 2, H * D + pad), 7.0, dtype=dtype, device=gpu)
    df = torch.from_numpy(freq).to(gpu) if rot else None
    cu, kv, table = s.dev(gpu)
    ops.rope_append(rows[:, :H * D], rows[:, H * D:(H + KV) * D], rows[:, (H + KV) * D:], kc, vc, cu, kv, table, df,
                    interleaved=interleaved, mscale=m, q_norm=dw[0], k_norm=dw[1], eps=1e-5, out=out[:, pad:],
                    stream=stream)
    torch.cuda.synchronize()
    assert (out[s.T:] == 7).all() and (out[:, :pad] == 7).all()
    pos = np.concatenate([np.arange(k - n, k) for n, k in lens]).astype(np.int64)
    x = x.astype(np.float64)
    q, qs = rotate(x[:, :H], pos, freq, interleaved, m, w[0], 1e-5)
    k, ks = rotate(x[:, H:H + KV], pos, freq, interleaved, m, w[1], 1e-5)
    got = out[:s.T, pad:].float().cpu().numpy().reshape(s.T, H, D)
    assert (np.abs(got - q) <= tolerance(q, qs, norm, dtype)).all()
    kk, vv = unpack_keys(kc.float().cpu().numpy()), unpack_values(vc.float().cpu().numpy())
    ktol, fresh = tolerance(k, ks, norm, dtype), np.ones((s.n_pages, page), bool)
    v = torch.from_numpy(x[:, H + KV:].astype(np.float32)).to(dtype).float().numpy()
    for b, (n, length) in enumerate(lens):
        for i in range(n):
            p, r = length - n + i, s.cu[b] + i
            at = s.table[b, p // page] if 0 <= p < page * s.table.shape[1] else -1
            if at < 0:
                continue
            fresh[at, p % page] = False
            assert (np.abs(kk[at, :, p % page] - k[r]) <= ktol[r]).all()
            assert np.array_equal(vv[at, :, p % page], v[r])
    # nothing else was touched
    assert (kk.transpose(0, 2, 1, 3)[fresh] == 3).all() and (vv.transpose(0, 2, 1, 3)[fresh] == 5).all()


LENS = [(1, 1), (1, 33), (5, 70), (40, 40), (70, 131), (0, 12), (2, 64), (33, 97)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("D,H,KV,rot", [(64, 6, 2, 64), (128, 4, 4, 32), (256, 5, 1, 64), (128, 8, 2, 128),
                                        (256, 4, 2, 256), (64, 3, 3, 20), (128, 2, 1, 126), (64, 2, 2, 2),
                                        (64, 2, 2, 0)])
def test_parity(gpu, D, H, KV, rot, interleaved, dtype):
    check(gpu, LENS, H, KV, D, rot=rot, interleaved=interleaved, dtype=dtype)


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(64, 20), (128, 128), (256, 64)])
def test_norms(gpu, D, rot, interleaved):
    check(gpu, LENS, 4, 2, D, rot=rot, interleaved=interleaved, norm=True, m=1.25)


@pytest.mark.parametrize("page", [32, 96, 256])
def test_pages(gpu, page):
    check(gpu, LENS + [(300, 500)], 4, 2, 64, page=page)


@pytest.mark.parametrize("pad", [1, 4, 8])
def test_strides_and_alignments(gpu, pad):
    check(gpu, LENS, 4, 2, 128, pad=pad, norm=True, rot=40)


def test_far_positions(gpu):
    check(gpu, [(3, 500001), (40, 131072)], 2, 1, 64, page=256, base=5e5)


def test_rows_before_position_zero_and_pages_that_are_not_there(gpu):
    check(gpu, [(5, 3), (90, 40), (70, 200)], 4, 2, 64, page=32, break_pages=[(2, 4), (2, 5)])


def test_many_sequences(gpu):
    """More sequences than one workgroup's threads look over at once."""
    check(gpu, [(1, 1 + i % 90) for i in range(700)], 2, 1, 64, page=32)


def test_another_stream(gpu):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    check(gpu, LENS, 4, 2, 64, stream=side)


def test_graph_follows_lengths(gpu):
    from raceline_amd import ops

    s = Sequences([(1, 90), (3, 64)], 64, 1)
    rng = torch.Generator(device=gpu).manual_seed(3)
    x = torch.randn((4, 6 * 64), generator=rng, device=gpu)
    freq = ops.rope_frequencies(64, device=gpu)
    cu, kv, table = s.dev(gpu)
    kc, vc = ops.kv_cache(s.n_pages, 1, 64, 64, F16, gpu)
    args = (x[:, :256], x[:, 256:320], x[:, 320:], kc, vc, cu, kv, table, freq)
    ops.rope_append(*args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.rope_append(*args)
    for back in (0, 5, 17):
        kv.copy_(torch.from_numpy(s.kv - back))
        kc.zero_(), vc.zero_()
        eager = ops.rope_append(*args)
        want = kc.clone(), vc.clone()
        kc.zero_(), vc.zero_(), out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_no_pages_no_table_and_no_rows(gpu):
    """Without pages the queries are turned and nothing is stored."""
    from raceline_amd import ops

    s = Sequences([(2, 50), (40, 90)], 64)
    cu, kv, table = s.dev(gpu)
    x = torch.randn((42, 6 * 64), device=gpu)
    kc, vc = ops.kv_cache(s.n_pages, 1, 64, 64, F16, gpu)
    freq = ops.rope_frequencies(64, device=gpu)
    parts = x[:, :256], x[:, 256:320], x[:, 320:]
    want = ops.rope_append(*parts, kc, vc, cu, kv, table, freq)
    kc.fill_(3), vc.fill_(5)
    for k, v, t in ((kc, vc, table[:, :0]), (kc[:0], vc[:0], table)):
        assert torch.equal(ops.rope_append(*parts, k, v, cu, kv, t, freq), want)
    assert (kc == 3).all() and (vc == 5).all()
    empty = torch.zeros(1, dtype=torch.int32, device=gpu)
    none = [p[:0] for p in parts]
    assert ops.rope_append(*none, kc, vc, empty, empty[:0], table[:0], freq).shape == (0, 256)


@pytest.mark.parametrize("H,KV", [(1, 1), (40, 1), (7, 7)])
def test_heads(gpu, H, KV):
    check(gpu, [(1, 33), (40, 40)], H, KV, 64, norm=True)


def test_infinities_and_nan_stay_in_their_head(gpu):
    from raceline_amd import ops

    s = Sequences([(3, 3)], 32)
    x = torch.randn((3, 4 * 64), device=gpu)
    x[1, 5], x[2, 64 + 7] = float("inf"), float("nan")
    kc, vc = ops.kv_cache(s.n_pages, 1, 64, 32, F16, gpu)
    q = ops.rope_append(x[:, :128], x[:, 128:192], x[:, 192:], kc, vc, *s.dev(gpu), ops.rope_frequencies(32, device=gpu))
    bad = (~q.isfinite()).cpu().numpy()
    assert set(zip(*np.nonzero(bad))) == {(1, 5), (1, 21), (2, 64 + 7), (2, 64 + 23)}


def test_offsets_past_32_bits(gpu):
    """The same rows into pages at the end of a cache of 4.6e9 elements (9.2 GB) an array."""
    from raceline_amd import ops

    s = Sequences([(1, 130), (40, 70)], 64)
    cu, kv, table = s.dev(gpu)
    x = torch.randn((41, 12 * 256), device=gpu)
    parts = x[:, :1024], x[:, 1024:2048], x[:, 2048:]
    freq = ops.rope_frequencies(64, device=gpu)
    small = [c.fill_(3) for c in ops.kv_cache(s.n_pages, 4, 256, 64, F16, gpu)]
    n = 70000
    large = ops.kv_cache(n, 4, 256, 64, F16, gpu)
    for c in large:
        c[n - s.n_pages:] = 3
    q = ops.rope_append(*parts, *small, cu, kv, table, freq)
    q2 = ops.rope_append(*parts, *large, cu, kv, table + (n - s.n_pages), freq)
    assert torch.equal(q, q2)
    for a, b in zip(small, large):
        assert torch.equal(a, b[n - s.n_pages:])
