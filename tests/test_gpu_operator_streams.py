"""The operators on a stream beside the current one: outputs and scratch are not memory that work queued
on the current stream has still to write, and an output outlives what the current stream still reads of it."""

import pytest
import torch

from tests.paged import Sequences

pytestmark = pytest.mark.gpu

WAIT = 5_000_000    # clock cycles: some milliseconds, longer than the calls below


def rope(gpu):
    from raceline_amd import ops

    s = Sequences([(70, 300), (1, 40)], 64)
    x = torch.randn((s.T, 6 * 64), device=gpu)
    kc, vc = ops.kv_cache(s.n_pages, 1, 64, 64, torch.float16, gpu)
    freq = ops.rope_frequencies(64, device=gpu)
    seqs = s.dev(gpu)
    return lambda stream: ops.rope_append(x[:, :256], x[:, 256:320], x[:, 320:], kc, vc, *seqs, freq, stream=stream)


def attn(gpu, lens):
    from raceline_amd import ops

    s = Sequences(lens, 64)
    kc, vc = (torch.randn((s.n_pages, 1, 64, 128), device=gpu).half() for _ in range(2))
    q = torch.randn((s.T, 4 * 128), device=gpu).half()
    seqs = s.dev(gpu)
    size = ops.attention_workspace_bytes(s.T, 4, 1, 128, len(lens), s.max_q, s.max_kv)
    call = lambda stream: ops.attention(q, kc, vc, *seqs, s.max_q, s.max_kv, stream=stream)    # noqa: E731
    call.scratch = size
    return call


def logits(gpu):
    from raceline_amd import ops

    x = torch.randn((3, 50000), device=gpu)
    allowed = torch.randint(-2**31, 2**31, (3, 1563), device=gpu).int()
    return lambda stream: ops.adjust_logits(x, allowed=allowed, stream=stream)


CALLS = {"rope_append": rope, "attention": lambda gpu: attn(gpu, [(70, 300), (1, 40)]),
         "attention-few-split": lambda gpu: attn(gpu, [(2, 6000)]),
         "attention-many-split": lambda gpu: attn(gpu, [(60, 5000)]), "adjust_logits": logits}


@pytest.mark.parametrize("name", CALLS)
def test_new_tensors_are_not_memory_still_to_be_written(gpu, name):
    call = CALLS[name](gpu)
    want = call(None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    sizes = [want.numel() * want.element_size()] + ([call.scratch] if getattr(call, "scratch", 0) else [])
    late = [torch.empty(n, dtype=torch.uint8, device=gpu) for n in sizes]
    torch.cuda._sleep(WAIT)
    for t in late:
        t.fill_(0x7F)
    del late, t                                              # free for the current stream, and still to be written
    got = call(side)
    side.synchronize()
    first = got.cpu()
    torch.cuda.synchronize()
    assert torch.equal(first, want.cpu()) and torch.equal(got, want)


@pytest.mark.parametrize("name", CALLS)
def test_an_output_outlives_what_the_current_stream_reads_of_it(gpu, name):
    call = CALLS[name](gpu)
    want = call(None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = call(side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(WAIT)
    copy = got.clone()
    del got
    with torch.cuda.stream(side):
        for _ in range(4):
            torch.empty_like(want).fill_(7)                  # would take the freed output's place
    torch.cuda.synchronize()
    assert torch.equal(copy, want)


def test_a_capture_on_a_stream_given_by_name(gpu):
    """The captured stream passed as `stream`: the graph owns what the call allocates."""
    call = attn(gpu, [(2, 6000)])
    want = call(None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = call(side)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
