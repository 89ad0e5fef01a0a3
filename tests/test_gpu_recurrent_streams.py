"""causal_conv, gated_delta and sample on other streams than the current one and in captured graphs: outputs and
scratch are not memory that other work still writes, replays follow what changes in place, and graphs may share
scratch in turn."""

import pytest
import torch

from tests import recurrent as R

pytestmark = pytest.mark.gpu

WAIT = 5_000_000    # clock cycles: some milliseconds, longer than the calls below


def conv(gpu, lens=((70, 300), (1, 40))):
    from raceline_amd import ops

    s = R.Sequences(list(lens))
    x, w = torch.randn((s.T, 256), device=gpu), torch.randn((256, 4), device=gpu)
    state, seqs = torch.randn((s.n_slots, 3, 256), device=gpu), s.dev(gpu)
    call = lambda stream=None, **kw: ops.causal_conv(x, w, call.state, *seqs, stream=stream, **kw)         # noqa: E731
    call.state, call.seqs, call.scratch = state, seqs, 0
    return call


def delta(gpu, lens):
    from raceline_amd import ops

    s = R.Sequences(lens)
    Hk, Hv, D = 2, 4, 64
    q, k, v = (torch.randn((s.T, h * D), device=gpu).half() for h in (Hk, Hk, Hv))
    a, b, z = (torch.randn((s.T, n), device=gpu) for n in (Hv, Hv, Hv * D))
    a_log, dt, norm = torch.randn(Hv, device=gpu) - 1, torch.randn(Hv, device=gpu) - 2, torch.randn(D, device=gpu)
    state, seqs = torch.randn((s.n_slots, Hv, D, D), device=gpu), s.dev(gpu)
    call = lambda stream=None, **kw: ops.gated_delta(q, k, v, a, b, a_log, dt, call.state, *seqs, max_q=s.max_q, z=z,   # noqa: E731
                                                     norm=norm, stream=stream, **kw)
    call.state, call.seqs = state, seqs
    call.scratch = ops.gated_delta_workspace_bytes(s.T, Hk, Hv, D, D, s.B, s.max_q)
    return call


def sample(gpu, rows=3, V=50000):
    from raceline_amd import ops

    x, u = torch.randn((rows, V), device=gpu) * 3, torch.rand(rows, device=gpu, dtype=torch.float64)
    k, p = torch.full((rows,), 300, dtype=torch.int32, device=gpu), torch.full((rows,), 0.9, device=gpu)
    call = lambda stream=None, **kw: ops.sample(x, u, top_k=k, top_p=p, stream=stream, **kw)               # noqa: E731
    call.state, call.scratch, call.logits, call.u, call.p = None, ops.sample_workspace_bytes(rows, V), x, u, p
    return call


CALLS = {"causal_conv": conv, "gated_delta-tokens": lambda gpu: delta(gpu, [(3, 300), (1, 40)]),
         "gated_delta-chunks": lambda gpu: delta(gpu, [(150, 300), (1, 40), (64, 64)]), "sample": sample}


def fresh(call, start, stream=None, **kw):
    """The call on a state of its own -> output and state."""
    if start is not None:
        call.state = start.clone()
        torch.cuda.synchronize()
    out = call(stream, **kw)
    return out, call.state


def same(a, b):
    return torch.equal(a[0], b[0]) and (a[1] is None or torch.equal(a[1], b[1]))


@pytest.mark.parametrize("name", CALLS)
def test_new_tensors_are_not_memory_still_to_be_written(gpu, name):
    call = CALLS[name](gpu)
    start = call.state
    want = fresh(call, start)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    if start is not None:
        call.state = start.clone()
        torch.cuda.synchronize()
    sizes = [want[0].numel() * want[0].element_size()] + ([call.scratch] if call.scratch else [])
    late = [torch.empty(n, dtype=torch.uint8, device=gpu) for n in sizes]
    torch.cuda._sleep(WAIT)
    for t in late:
        t.fill_(0x7F)
    del late, t                                              # free for the current stream, and still to be written
    got = call(side)
    side.synchronize()
    first = got.cpu()
    torch.cuda.synchronize()
    assert torch.equal(first, want[0].cpu()) and same((got, call.state), want)


@pytest.mark.parametrize("name", CALLS)
def test_an_output_outlives_what_the_current_stream_reads_of_it(gpu, name):
    call = CALLS[name](gpu)
    start = call.state
    want = fresh(call, start)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got, _ = fresh(call, start, side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(WAIT)
    copy = got.clone()
    del got
    with torch.cuda.stream(side):
        for _ in range(4):
            torch.empty_like(want[0]).fill_(7)               # would take the freed output's place
    torch.cuda.synchronize()
    assert torch.equal(copy, want[0])


@pytest.mark.parametrize("name", [n for n in CALLS if n != "sample"])
def test_replays_follow_lengths_and_slots(gpu, name):
    """A padded batch is captured once; replays see what changed in place, and go on from the state they left."""
    call = CALLS[name](gpu)
    cu, kv, slots = call.seqs
    keep = torch.full_like(slots, 1000)
    start = call.state
    fresh(call, start, keep=keep)
    state = call.state = start.clone()
    out = torch.zeros_like(call(keep=keep))
    state.copy_(start)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(keep=keep, out=out)
    first = [x.clone() for x in (cu, kv, slots)]
    mirror = start.clone()
    for step in range(5):
        cu.copy_(first[0]), kv.copy_(first[1]), slots.copy_(first[2]), keep.fill_(1000)
        if step == 1:
            cu[1:] -= 1                                      # one row less, another behind the last sequence
        if step == 2:
            slots[0] = -1
        if step == 3:
            keep[0] = 1
            kv.copy_(cu[1:] - cu[:-1])                       # all begin from zeros
        out.fill_(3)
        g.replay()
        torch.cuda.synchronize()
        call.state = mirror
        want = call(keep=keep, out=torch.full_like(out, 3))
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, mirror), f"replay {step}"


def test_replays_of_sample_follow_the_logits(gpu):
    call = sample(gpu)
    out = torch.zeros(3, dtype=torch.int32, device=gpu)
    call(out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out=out)
    for step in range(6):
        call.logits.normal_().mul_(3)
        call.u.uniform_()
        call.p.fill_([0.9, 0.2, 1.0, 0.5, 0.99, 0.0][step])
        if step == 3:
            call.logits[1] = -float("inf")
        out.fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), f"replay {step}"


def test_graphs_that_share_scratch_in_turn(gpu):
    """Two captured calls with one workspace, replayed one after the other with eager calls between them."""
    calls = [delta(gpu, [(150, 300), (1, 40), (64, 64)]), delta(gpu, [(90, 90), (200, 300)]), sample(gpu, 2, 9000), sample(gpu, 5, 30000)]
    ws = torch.empty(max(c.scratch for c in calls), dtype=torch.uint8, device=gpu)
    starts = [c.state for c in calls]
    wants = [fresh(c, s) for c, s in zip(calls, starts)]
    graphs = []
    for c, s, w in zip(calls, starts, wants):
        if s is not None:
            c.state = s.clone()
        c.out = torch.zeros_like(w[0])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c(out=c.out, workspace=ws)
        graphs.append(g)
    for turn in range(4):
        for c, s, w, g in zip(calls, starts, wants, graphs):
            if s is not None:
                c.state.copy_(s)
            c.out.zero_()
            ws.fill_(0xFF if turn % 2 else 0x7B)
            g.replay()
            torch.cuda.synchronize()
            assert same((c.out, c.state), w)
            kept = None if s is None else c.state
            assert same(fresh(c, s, workspace=ws), w)
            c.state = kept
