"""What rope_append, attention and adjust_logits refuse, without a GPU: the C functions before any
device work (pointers are placeholders), the Python layer before it calls them. And the rotary
frequencies, which are formed on the host."""

import contextlib
import math

import numpy as np
import pytest
import torch

from raceline_amd import lib, ops

ROPE = dict(q=16, q_stride=256, k=16, k_stride=128, v=16, v_stride=128, T=4, freq=16, rot=64, interleaved=0, mscale=1.0,
            q_norm=None, k_norm=None, eps=1e-6, heads=4, kv_heads=2, D=64, dtype=0, q_out=16, q_out_stride=256,
            k_cache=16, v_cache=16, n_pages=4, page_size=64, cu_q=16, kv_len=16, table=16, table_stride=2, table_width=2,
            B=1, stream=None)
ATTN = dict(q=16, q_stride=256, T=4, heads=4, kv_heads=2, D=64, dtype=0, k_cache=16, v_cache=16, n_pages=4, page_size=64,
            cu_q=16, kv_len=16, table=16, table_stride=2, table_width=2, B=1, max_q=4, max_kv=100, scale=0.125, window=0,
            softcap=0.0, out=16, out_stride=256, out_dtype=0, workspace=None, workspace_bytes=0, stream=None)
LOGITS = dict(logits=16, stride=1000, rows=2, vocab=1000, tokens=16, token_stride=10, max_tokens=10, n_tokens=None,
              n_prompt=None, repetition=None, presence=None, frequency=None, bias_ids=16, bias=16, n_bias=3,
              bias_stride=3, allowed=16, allowed_stride=32, out=16, out_stride=1000, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(D=96), "head size 96"), (dict(dtype=2), "unknown dtype"), (dict(heads=5), "evenly"), (dict(heads=1), "evenly"),
    (dict(kv_heads=0), "evenly"), (dict(rot=63), "rot=63"), (dict(rot=66), "rot=66"), (dict(rot=-2), "rot=-2"),
    (dict(page_size=48), "page_size=48"), (dict(page_size=0), "page_size=0"), (dict(table_stride=1), "table_stride=1"),
    (dict(table_width=1 << 24, table_stride=1 << 24), "2.29 positions"), (dict(q=None), "null pointer"),
    (dict(n_pages=1 << 30, page_size=128), "2.31 blocks"),
    (dict(freq=None), "null pointer"), (dict(kv_len=None), "null pointer"), (dict(k_cache=None), "null cache"),
    (dict(table=None), "null table"), (dict(q_stride=255), "stride"), (dict(v_stride=127), "stride"),
    (dict(q_out_stride=0), "stride"), (dict(k_cache=24), "16-byte aligned"), (dict(T=-1), "T=-1"), (dict(B=-1), "B=-1"),
    (dict(T=1 << 27), "too large")])
def test_rope_append_refuses(change, message):
    with pytest.raises(lib.RlqError, match=message):
        lib.call("rlq_rope_append", *{**ROPE, **change}.values())


@pytest.mark.parametrize("change,message", [
    (dict(D=80), "head size 80"), (dict(dtype=3), "unknown dtype"), (dict(out_dtype=2), "unknown output dtype"),
    (dict(heads=3), "evenly"), (dict(page_size=16), "page_size=16"), (dict(table_width=3), "table_width=3"),
    (dict(table_width=1 << 24, table_stride=1 << 24), "2.29 positions"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
    (dict(softcap=-1.0), "softcap"), (dict(softcap=math.nan), "softcap"), (dict(softcap=1e-40), "passes fp32"),
    (dict(n_pages=1 << 30, page_size=128), "2.31 blocks"), (dict(window=-1), "window=-1"),
    (dict(max_q=-1), "max_q=-1"), (dict(max_kv=-1), "max_kv=-1"), (dict(T=-4), "T=-4"), (dict(q=None), "null pointer"),
    (dict(out=None), "null pointer"), (dict(v_cache=None), "null cache"), (dict(table=None), "null table"),
    (dict(q_stride=128), "stride"), (dict(out_stride=128), "stride"), (dict(v_cache=8), "16-byte aligned"),
    (dict(max_kv=9000), "bytes of 16-byte aligned workspace"),
    (dict(max_kv=9000, workspace=8, workspace_bytes=1 << 30), "bytes of 16-byte aligned workspace")])
def test_attention_refuses(change, message):
    with pytest.raises(lib.RlqError, match=message):
        lib.call("rlq_attention", *{**ATTN, **change}.values())


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows=-1"), (dict(rows=70000), "rows=70000"), (dict(vocab=-5), "vocab=-5"), (dict(n_bias=1025), "n_bias"),
    (dict(n_bias=-1), "n_bias"), (dict(logits=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(stride=999), "strides"), (dict(out_stride=999), "strides"), (dict(tokens=None), "null tokens"),
    (dict(bias=None), "null biases"), (dict(bias_ids=None), "null biases"), (dict(allowed_stride=31), "mask row"),
    (dict(max_tokens=-1), "max_tokens=-1")])
def test_adjust_logits_refuses(change, message):
    with pytest.raises(lib.RlqError, match=message):
        lib.call("rlq_adjust_logits", *{**LOGITS, **change}.values())


def test_calls_without_rows_do_nothing():
    for name, args in (("rlq_rope_append", ROPE), ("rlq_attention", ATTN)):
        assert lib.call(name, *{**args, "T": 0, "q": None}.values()) == 0
        assert lib.call(name, *{**args, "B": 0, "cu_q": None}.values()) == 0
    assert lib.call("rlq_adjust_logits", *{**LOGITS, "rows": 0, "logits": None}.values()) == 0


def test_attention_workspace_query():
    assert ops.attention_workspace_bytes(1, 16, 4, 256, 1, 1, 100) == 0            # one run of keys: nothing to join
    assert ops.attention_workspace_bytes(1, 16, 4, 256, 1, 1, 100000) > 0
    assert ops.attention_workspace_bytes(1, 16, 4, 256, 1, 1, 100000, window=64) == 0
    assert ops.attention_workspace_bytes(1, 16, 4, 250, 1, 1, 100000) == 0         # no such head size


def paged(B=2, KV=2, D=64, page=64, dtype=torch.float16):
    k = torch.zeros((3, KV, page, D), dtype=dtype)
    return [k, k.clone(), torch.zeros(B + 1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32),
            torch.zeros((B, 2), dtype=torch.int32)]


@contextlib.contextmanager
def refused():
    """A refusal of the arguments, not of where they are."""
    with pytest.raises((ValueError, TypeError, lib.RlqError)) as e:
        yield
    assert "on the GPU" not in str(e.value)


def change(args, at, value):
    args = list(args)
    args[at] = value
    return args


def test_python_layer_refuses_caches_and_sequences():
    q, args = torch.zeros((4, 256), dtype=torch.float16), paged()
    bad = [(0, args[0][:2]), (0, args[0].bfloat16()), (1, args[1].transpose(2, 3)), (0, args[0].float()), (0, args[0][0]),
           (2, args[2].long()), (3, args[3].long()), (4, args[4].long()), (2, args[2][:2]), (3, torch.zeros((2, 1), dtype=torch.int32)),
           (4, args[4][:1]), (4, args[4][:1].expand(2, 2)), (4, args[4][0]), (4, torch.zeros((2, 4), dtype=torch.int32)[:, ::2])]
    for at, value in bad:
        with refused():
            ops.attention(q, *change(args, at, value), max_q=4, max_kv=10)
        with refused():
            ops.rope_append(torch.zeros((4, 256)), torch.zeros((4, 128)), torch.zeros((4, 128)),
                            *change(args, at, value), None)


def test_python_layer_refuses_rows():
    args = paged()
    q = torch.zeros((4, 256), dtype=torch.float16)
    for bad in (q.float(), q.bfloat16(), q[:, :200], q[:, :0], q[:, ::2], q[0], q.t()):
        with refused():
            ops.attention(bad, *args, max_q=4, max_kv=10)
    for out in (q[:3], torch.zeros((4, 512), dtype=torch.float16)[:, ::2], q.float()):
        with refused():
            ops.attention(q, *args, max_q=4, max_kv=10, out=out)
    q, k = torch.zeros((4, 256)), torch.zeros((4, 128))
    freq = torch.zeros(32, dtype=torch.float64)
    ok = dict(q=q, k=k, v=k, freq=freq)
    for bad in (dict(q=q.half()), dict(q=q[:, :64]), dict(k=k[:3]), dict(v=k[:, :64]), dict(k=q[:, ::2]),
                dict(freq=freq.float()), dict(freq=torch.zeros(64, dtype=torch.float64)[::2]), dict(q_norm=torch.zeros(63)),
                dict(k_norm=torch.zeros(64, dtype=torch.float64)), dict(out=torch.zeros((4, 256)))):
        a = {**ok, **bad}
        with refused():
            ops.rope_append(a.pop("q"), a.pop("k"), a.pop("v"), *args, a.pop("freq"), **a)


def test_python_layer_refuses_logits():
    x, i = torch.zeros((2, 100)), dict(dtype=torch.int32)
    for bad in (dict(tokens=torch.zeros((2, 5))), dict(tokens=torch.zeros((3, 5), **i)), dict(n_tokens=torch.zeros(3, **i)),
                dict(repetition=torch.zeros(2, dtype=torch.float64)), dict(presence=torch.zeros((2, 1))),
                dict(bias=torch.zeros((2, 3))), dict(bias_ids=torch.zeros((2, 3), **i)),
                dict(bias=torch.zeros((2, 3)), bias_ids=torch.zeros((2, 4), **i)),
                dict(bias=torch.zeros((2, 3)), bias_ids=torch.zeros((1, 3), **i)), dict(allowed=torch.zeros((2, 3), **i)),
                dict(allowed=torch.zeros((2, 4))), dict(out=torch.zeros((2, 99))), dict(out=x.double())):
        with refused():
            ops.adjust_logits(x, **bad)
    with refused():
        ops.adjust_logits(x.half())


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(ValueError, match="on the GPU"):
        ops.attention(torch.zeros((4, 256), dtype=torch.float16), *paged(), max_q=4, max_kv=10)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.rope_append(torch.zeros((4, 256)), torch.zeros((4, 128)), torch.zeros((4, 128)), *paged(), None)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.adjust_logits(torch.zeros((2, 100)))


def test_kv_cache_refuses():
    for bad in (dict(page_size=48), dict(head_dim=96), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            ops.kv_cache(**{**dict(n_pages=1, kv_heads=1, head_dim=64, device="cpu"), **bad})
    k, v = ops.kv_cache(3, 2, 64, 32, torch.bfloat16, device="cpu")
    assert k.shape == v.shape == (3, 2, 32, 64) and k.dtype == torch.bfloat16


def test_rope_frequencies():
    """The formulas of include/rlq.h in 64 bits: each is a few roundings of 2^-53."""
    rot, base, i = 64, 1e4, np.arange(32)
    plain = base ** (-2.0 * i / rot)

    def got(**kw):
        return ops.rope_frequencies(rot, base, device="cpu", **kw).numpy()

    close = dict(rtol=64 * 2.0 ** -53, atol=0)      # the exponent's rounding times ln(base) in the power
    np.testing.assert_allclose(got(), plain, **close)
    np.testing.assert_allclose(got(scaling="linear", factor=8), plain / 8, **close)
    ntk = got(scaling="ntk", factor=8)
    assert ntk[0] == 1
    np.testing.assert_allclose(ntk[-1], plain[-1] / 8, **close)
    parts = got(scaling="parts", factor=8, low=1, high=4, original=8192)
    turns = 8192 * plain / (2 * math.pi)
    assert (parts[turns >= 4] == got()[turns >= 4]).all()
    np.testing.assert_allclose(parts[turns <= 1], plain[turns <= 1] / 8, **close)
    mid = (turns > 1) & (turns < 4)
    keep = (turns[mid] - 1) / 3
    np.testing.assert_allclose(parts[mid], plain[mid] * (keep + (1 - keep) / 8), rtol=1e-13)
    assert ops.rope_frequencies(0, device="cpu").numel() == 0


@pytest.mark.parametrize("kw", [dict(rot=63), dict(rot=-2), dict(base=1.0), dict(base=math.inf), dict(scaling="other"),
                                dict(scaling="linear", factor=0.5), dict(scaling="ntk", factor=math.nan),
                                dict(scaling="ntk", factor=2, rot=2), dict(scaling="parts", factor=2, low=4, high=4, original=10),
                                dict(scaling="parts", factor=2, original=0), dict(scaling="parts", factor=2, low=-1, original=9)])
def test_rope_frequencies_refuse(kw):
    with pytest.raises((ValueError, lib.RlqError)):
        ops.rope_frequencies(**{**dict(rot=64, device="cpu"), **kw})


def test_fatal_mode_reports_before_device_work():
    """The default mode prints and exits (tests/test_capi.py has it for the linears)."""
    import subprocess
    import sys

    code = ("import ctypes; from raceline_amd import lib; L = lib.load(); "
            "L.rlq_adjust_logits(None, 0, -1, 0, None, 0, 0, None, None, None, None, None, None, None, 0, 0, None, 0, None, 0, None)")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 1 and "raceline: fatal: rlq_adjust_logits" in r.stderr
