"""Attention over the paged cache against the same in 64 bits (tests/paged.py), where it can go
wrong: one token to chunks, lengths around a block's 32 and a page's positions, shared heads of every
count, rows that see nothing, windows, caps, pages that are not there, infinities and NaN in masked
places, strides, long offsets, streams and graphs."""

import numpy as np
import pytest
import torch

from tests.paged import Sequences, attend, attention_tolerance, pack_keys, pack_values

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(gpu, lens, H, KV, D, page=64, dtype=F16, seed=0, q_scale=1.5):
    """A cache whose unwritten places hold NaN, and the queries, all of them also as float64."""
    rng = np.random.default_rng(seed)
    s = Sequences(lens, page, seed)
    kc = np.full((s.n_pages, KV, page, D), np.nan, np.float32)
    vc = kc.copy()
    keys, values = [], []
    for b, (_, kv) in enumerate(lens):
        k, v = (rng.standard_normal((kv, KV, D)).astype(np.float32) for _ in range(2))
        k, v = (torch.from_numpy(x).to(dtype).float().numpy() for x in (k, v))
        for p in range(kv):
            at = s.table[b, p // page]
            if at >= 0:
                kc[at, :, p % page], vc[at, :, p % page] = k[p], v[p]
        keys.append(k)
        values.append(v)
    q = torch.from_numpy((rng.standard_normal((s.T, H * D)) * q_scale).astype(np.float32)).to(dtype)
    s.q = q.float().numpy().reshape(s.T, H, D).astype(np.float64)
    s.keys, s.values = keys, values
    s.dq = q.to(gpu)
    s.kc = torch.from_numpy(pack_keys(kc)).to(gpu).to(dtype)
    s.vc = torch.from_numpy(pack_values(vc)).to(gpu).to(dtype)
    s.dtype, s.D = dtype, D
    return s


def check(s, out, scale=None, window=0, cap=0.0, hidden=None, rows=None):
    scale = s.D ** -0.5 if scale is None else scale
    got = out.float().cpu().numpy().astype(np.float64).reshape(s.T, -1, s.D)
    for b, (n, kv) in enumerate(s.lens):
        if not n:
            continue
        r = slice(s.cu[b], s.cu[b] + n)
        ref, size = attend(s.q[r], s.keys[b], s.values[b], kv, scale, window, cap, hidden[b] if hidden else ())
        tol = attention_tolerance(ref, size, s.q[r], s.keys[b], max(kv, 1), scale, cap, s.dtype, out.dtype)
        err = np.abs(got[r] - ref)
        assert np.isfinite(got[r]).all(), f"sequence {b}: not finite"
        assert (err <= tol).all(), f"sequence {b} ({n}, {kv}): off by {(err / tol).max():.2f} of its tolerance"


def run(s, gpu, **kw):
    from raceline_amd import ops

    cu, kv, table = s.dev(gpu)
    out = ops.attention(kw.pop("q", s.dq), s.kc, s.vc, cu, kv, table, kw.pop("max_q", s.max_q),
                        kw.pop("max_kv", s.max_kv), **kw)
    torch.cuda.synchronize()
    return out


TYPES = [(F16, F16), (BF16, F16), (BF16, BF16), (F16, BF16)]


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=["f16", "bf16-f16", "bf16", "f16-bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_single_tokens_of_all_lengths(gpu, D, dtype, out_dtype):
    lens = [(1, kv) for kv in (1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 300)]
    s = make(gpu, lens, 8, 2, D, dtype=dtype)
    check(s, run(s, gpu, out_dtype=out_dtype))


@pytest.mark.parametrize("H,KV", [(1, 1), (3, 3), (5, 1), (8, 1), (16, 1), (17, 1), (33, 1), (40, 8), (64, 2)])
def test_shared_heads_of_every_count(gpu, H, KV):
    s = make(gpu, [(1, 70), (2, 40), (1, 200)], H, KV, 64)
    check(s, run(s, gpu))


@pytest.mark.parametrize("dtype,out_dtype", TYPES, ids=["f16", "bf16-f16", "bf16", "f16-bf16"])
@pytest.mark.parametrize("D,H,KV,page", [(64, 4, 4, 32), (128, 8, 2, 96), (256, 5, 1, 64)])
def test_chunks_and_prompts(gpu, D, H, KV, page, dtype, out_dtype):
    lens = [(70, 70), (129, 131), (33, 260), (1, 1), (64, 64)]
    s = make(gpu, lens, H, KV, D, page=page, dtype=dtype)
    check(s, run(s, gpu, out_dtype=out_dtype))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_drafts_chunks_tokens_and_empty_sequences_together(gpu, D):
    lens = [(1, 900), (0, 50), (140, 140), (5, 77), (0, 0), (8, 8), (1, 1), (60, 333)]
    s = make(gpu, lens, 8, 2, D)
    check(s, run(s, gpu))


@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (4096, 1), (1, 100000), (4096, 100000), (0, 0)])
def test_wrong_bounds_choose_another_kernel_only(gpu, max_q, max_kv):
    s = make(gpu, [(1, 700), (90, 400), (3, 30)], 8, 2, 128)
    check(s, run(s, gpu, max_q=max_q, max_kv=max_kv))


@pytest.mark.parametrize("lens", [[(1, 9000)], [(5, 4097), (1, 3)], [(100, 6000)], [(100, 6000), (1, 5000)]],
                         ids=["token", "draft", "chunk", "both"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_keys_split_over_workgroups(gpu, D, lens):
    s = make(gpu, lens, 4, 1, D)
    out = run(s, gpu)
    check(s, out)
    assert torch.equal(out, run(s, gpu))


@pytest.mark.parametrize("lens", [[(1, 200), (1, 5), (4, 130)], [(150, 300), (40, 40)]], ids=["few", "many"])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000, 2**31 - 1])
def test_windows(gpu, window, lens):
    s = make(gpu, lens, 4, 2, 64)
    check(s, run(s, gpu, window=window), window=window if window < 2**31 - 1 else 0)


@pytest.mark.parametrize("lens", [[(1, 6000)], [(60, 6000)]], ids=["few", "many"])
def test_window_over_a_long_context_with_pages_given_back(gpu, lens):
    s = make(gpu, lens, 8, 2, 128)
    n, kv = lens[0]
    s.table[0, :(kv - n + 1 - 2500) // 64] = -1
    check(s, run(s, gpu, window=2500), window=2500)


@pytest.mark.parametrize("cap", [1.0, 30.0, 1e4])
@pytest.mark.parametrize("lens", [[(1, 200), (3, 50)], [(100, 150)]], ids=["few", "many"])
def test_capped_scores(gpu, lens, cap):
    s = make(gpu, lens, 4, 2, 128, q_scale=8.0)
    check(s, run(s, gpu, softcap=cap), cap=cap)


@pytest.mark.parametrize("lens", [[(1, 100), (3, 50)], [(100, 150)]], ids=["few", "many"])
@pytest.mark.parametrize("scale", [1e-3, 0.5])
def test_scale(gpu, lens, scale):
    s = make(gpu, lens, 4, 2, 64)
    check(s, run(s, gpu, scale=scale), scale=scale)


@pytest.mark.parametrize("D,H,KV", [(64, 4, 2), (128, 8, 2), (256, 4, 4)])
def test_rows_that_see_no_key_are_zero(gpu, D, H, KV):
    """More new rows than tokens: the first rows lie before position 0."""
    lens = [(5, 3), (90, 40), (3, 0)]
    s = make(gpu, lens, H, KV, D)
    out = run(s, gpu)
    check(s, out)
    assert (out[:2] == 0).all() and (out[5:55] == 0).all() and (out[95:] == 0).all()


@pytest.mark.parametrize("lens", [[(2, 300), (1, 100)], [(120, 300), (1, 100)]], ids=["few", "many"])
def test_pages_that_are_not_there_are_not_seen(gpu, lens):
    s = make(gpu, lens, 4, 2, 128, page=32)
    s.table[0, 2], s.table[0, 5], s.table[0, 9] = -1, s.n_pages, 2**31 - 1
    s.table[1, :] = -7                                       # a sequence without any
    hidden = [[p for c in (2, 5, 9) for p in range(32 * c, min(32 * c + 32, 300))], list(range(100))]
    out = run(s, gpu)
    check(s, out, hidden=hidden)
    assert (out[s.cu[1]:] == 0).all()


def test_positions_past_the_table_are_not_seen(gpu):
    s = make(gpu, [(1, 200), (40, 128)], 4, 2, 64)
    s.table = s.table[:, :1].copy()
    check(s, run(s, gpu), hidden=[range(64, 200), range(64, 128)])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(4, 100)], [(100, 130)], [(60, 4000)]], ids=["few", "many", "split"])
@pytest.mark.parametrize("odd", [float("inf"), float("-inf"), float("nan")])
def test_infinities_and_nan_reach_only_the_rows_that_see_them(gpu, lens, odd, D):
    s = make(gpu, lens, 4, 2, D, page=64)
    n, kv = lens[0]
    at, dim = kv - 2, 3                                      # seen by the last two rows alone
    place = s.table[0, at // 64], slice(None), at % 64
    for c, pack in ((s.vc, pack_values), (s.kc, pack_keys)):
        mark = np.zeros((1, 1, 64, D), np.float32)
        mark[0, 0, at % 64, dim] = 1
        m = torch.from_numpy(pack(mark)).to(gpu)[0, 0].bool()
        c[int(place[0])][:, m] = odd
        out = run(s, gpu).float().cpu().numpy().reshape(n, 4, D)
        ref, size = attend(s.q, s.keys[0], s.values[0], kv, D ** -0.5)
        tol = attention_tolerance(ref, size, s.q, s.keys[0], kv, D ** -0.5, 0.0, F16, F16)
        assert (np.abs(out[:n - 2] - ref[:n - 2]) <= tol[:n - 2]).all()
        if c is s.vc:
            assert np.array_equal(out[n - 2:, :, dim], np.full((2, 4), odd, np.float32), equal_nan=True)
            rest = np.delete(np.arange(D), dim)
            assert (np.abs(out[n - 2:][..., rest] - ref[n - 2:][..., rest]) <= tol[n - 2:][..., rest]).all()
        c[int(place[0])][:, m] = 0.5


@pytest.mark.parametrize("lens", [[(1, 100), (3, 50)], [(100, 150)]], ids=["few", "many"])
@pytest.mark.parametrize("pad", [1, 4, 8])
def test_strides_and_alignments(gpu, lens, pad):
    s = make(gpu, lens, 4, 2, 64)
    big = torch.full((s.T, 256 + 2 * pad), 7.0, dtype=F16, device=gpu)
    q = big[:, pad:pad + 256]
    q.copy_(s.dq)
    room = torch.full((s.T + 3, 256 + 2 * pad), 7.0, dtype=F16, device=gpu)
    out = run(s, gpu, q=q, out=room[:s.T, pad:pad + 256])
    check(s, out)
    assert (room[:, :pad] == 7).all() and (room[:, pad + 256:] == 7).all() and (room[s.T:] == 7).all()


def test_rows_behind_the_last_sequence_are_left_as_they_were(gpu):
    for lens in ([(1, 50), (2, 60)], [(70, 90), (2, 3)], [(1, 5000), (40, 5000)]):
        s = make(gpu, lens, 4, 2, 64)
        q = torch.full((s.T + 37, 256), float("nan"), dtype=F16, device=gpu)
        q[:s.T] = s.dq
        out = torch.full((s.T + 37, 256), 7.0, dtype=F16, device=gpu)
        run(s, gpu, q=q, out=out)
        check(s, out[:s.T])
        assert (out[s.T:] == 7).all()


def test_offsets_past_32_bits(gpu):
    """Pages at the end of a cache of 4.6e9 elements (9.2 GB) an array."""
    from raceline_amd import ops

    s = make(gpu, [(1, 130), (40, 70)], 4, 4, 256, page=64)
    n = 70000
    kc, vc = ops.kv_cache(n, 4, 256, 64, F16, gpu)
    kc[n - s.n_pages:], vc[n - s.n_pages:] = s.kc, s.vc
    s.table += n - s.n_pages
    s.kc, s.vc = kc, vc
    check(s, run(s, gpu))


def test_another_stream_and_a_kept_workspace(gpu):
    from raceline_amd import ops

    s = make(gpu, [(1, 6000), (50, 5000)], 4, 1, 128)
    cu, kv, table = s.dev(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ws = torch.full((ops.attention_workspace_bytes(s.T, 4, 1, 128, 2, s.max_q, s.max_kv),), 255, dtype=torch.uint8,
                    device=gpu)
    assert ws.numel() > 0
    out = ops.attention(s.dq, s.kc, s.vc, cu, kv, table, s.max_q, s.max_kv, stream=side)
    out2 = ops.attention(s.dq, s.kc, s.vc, cu, kv, table, s.max_q, s.max_kv, workspace=ws, stream=side)
    side.synchronize()
    check(s, out)
    assert torch.equal(out, out2)


@pytest.mark.parametrize("lens", [[(1, 6000), (1, 40)], [(60, 5000)]], ids=["few", "many"])
def test_graph_follows_lengths_and_pages(gpu, lens):
    from raceline_amd import ops

    s = make(gpu, lens, 8, 2, 128)
    cu, kv, table = s.dev(gpu)
    args = (s.dq, s.kc, s.vc, cu, kv, table, s.max_q, s.max_kv)
    ops.attention(*args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.attention(*args)
    for shorten in (0, 33, 1000, 0):
        new = (s.kv - shorten).clip(min=s.max_q).astype(np.int32)
        kv.copy_(torch.from_numpy(new))
        eager = ops.attention(*args)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"shortened by {shorten}"
        if not shorten:
            check(s, out)


@pytest.mark.parametrize("lens", [[(1, 1 + 7 * i % 400) for i in range(100)],
                                  [(1 + 11 * i % 60, 100 + 11 * i % 60) for i in range(70)],
                                  [(1 + 11 * i % 60, 100 + 37 * i % 3000) for i in range(70)],
                                  [(1 + i, 1 + i) for i in range(63)]], ids=["few", "many", "both", "63"])
def test_many_sequences(gpu, lens):
    """More sequences than a wave's lanes, and as many as it has."""
    s = make(gpu, lens, 4, 2, 64, page=32)
    check(s, run(s, gpu))


def test_more_shared_heads_than_a_tile_has_rows(gpu):
    s = make(gpu, [(3, 40), (2, 90)], 160, 1, 64)
    check(s, run(s, gpu))


def test_sequences_that_share_pages(gpu):
    """Two sequences with one prompt's pages, and their own after it."""
    s = make(gpu, [(1, 192), (40, 192)], 4, 2, 128)
    s.table[1, :2] = s.table[0, :2]
    for b in (0, 1):
        s.keys[b][:128], s.values[b][:128] = s.keys[0][:128], s.values[0][:128]
    check(s, run(s, gpu))


def test_no_pages_and_no_table(gpu):
    from raceline_amd import ops

    s = make(gpu, [(2, 50), (40, 90)], 4, 2, 64)
    cu, kv, table = s.dev(gpu)
    for k, v, t in ((s.kc, s.vc, table[:, :0]), (s.kc[:0], s.vc[:0], table), (s.kc[:0], s.vc[:0], table[:, :0])):
        out = ops.attention(s.dq, k, v, cu, kv, t, s.max_q, s.max_kv)
        assert (out == 0).all()
    empty = torch.zeros(1, dtype=torch.int32, device=gpu)
    out = ops.attention(s.dq[:0], s.kc, s.vc, empty, empty[:0], table[:0], 0, 0)
    assert out.shape == (0, 256)
    seven = torch.full_like(s.dq, 7.0)
    ops.attention(s.dq, s.kc, s.vc, empty, empty[:0], table[:0], 1, 1, out=seven)
    assert (seven == 7).all()


def test_the_rows_may_take_the_queries_place(gpu):
    for lens in ([(1, 50), (3, 600)], [(70, 300)], [(1, 6000)], [(50, 6000)]):
        s = make(gpu, lens, 4, 2, 64)
        q = s.dq.clone()
        assert run(s, gpu, q=q, out=q) is q
        check(s, q)


def test_two_streams_at_once(gpu):
    from raceline_amd import ops

    work = [make(gpu, lens, 4, 1, 128, seed=i) for i, lens in enumerate([[(1, 9000)], [(60, 5000)]])]
    args = [(s.dq, s.kc, s.vc, *s.dev(gpu), s.max_q, s.max_kv) for s in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(ops.attention(*args[i]))
    torch.cuda.synchronize()
    for s, os in zip(work, outs):
        for o in os:
            check(s, o)


def test_two_graphs_at_once(gpu):
    """Each graph keeps its own scratch."""
    from raceline_amd import ops

    work = [make(gpu, [(1, 9000 - 500 * i)], 4, 1, 128, seed=i) for i in range(2)]
    args = [(s.dq, s.kc, s.vc, *s.dev(gpu), s.max_q, s.max_kv) for s in work]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in work], []
    for g, a in zip(graphs, args):
        ops.attention(*a)
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(ops.attention(*a))
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, o in zip(work, outs):
            check(s, o)


def test_windows_past_32_bits_are_none(gpu):
    s = make(gpu, [(1, 200), (40, 128)], 4, 2, 64)
    check(s, run(s, gpu, window=2**32 + 5, max_kv=2**40))
