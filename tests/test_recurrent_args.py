"""What causal_conv, gated_delta and sample refuse, without a GPU: the C functions before any device work (pointers
are placeholders), the Python layer before it calls them."""

import math

import pytest
import torch

from raceline_amd import lib, ops

CONV = dict(x=16, x_stride=64, T=4, channels=64, taps=4, w=16, bias=None, silu=1, state=16, n_slots=2, cu_q=16, kv_len=16,
            slots=16, keep=None, B=1, out=16, out_stride=64, out_dtype=0, stream=None)
DELTA = dict(q=16, q_stride=128, k=16, k_stride=128, v=16, v_stride=256, T=4, k_heads=2, v_heads=4, Dk=64, Dv=64, dtype=0,
             a=16, a_stride=4, b=16, b_stride=4, a_log=16, dt_bias=16, eps=1e-6, scale=0.125, z=16, z_stride=256, norm=16,
             norm_eps=1e-6, state=16, n_slots=2, cu_q=16, kv_len=16, slots=16, keep=None, B=1, max_q=4, out=16,
             out_stride=256, out_dtype=0, workspace=None, workspace_bytes=0, stream=None)
SAMPLE = dict(logits=16, stride=1000, rows=2, vocab=1000, uniform=16, temperature=None, top_k=None, top_p=None, min_p=None,
              tokens=16, probs=None, workspace=16, workspace_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(T=-1), "T=-1"), (dict(B=-1), "B=-1"), (dict(T=1 << 27), "too large"), (dict(B=1 << 21), "too large"),
    (dict(channels=0), "channels=0"), (dict(taps=1), "taps=1"), (dict(taps=5), "taps=5"), (dict(out_dtype=2), "output dtype"),
    (dict(n_slots=-1), "n_slots=-1"), (dict(x=None), "null pointer"), (dict(w=None), "null pointer"),
    (dict(cu_q=None), "null pointer"), (dict(slots=None), "null pointer"), (dict(state=None), "null state"),
    (dict(x_stride=63), "stride"), (dict(out_stride=63), "stride"),
    (dict(channels=1 << 30, x_stride=1 << 30, out_stride=1 << 30), "too many")])
def test_causal_conv_refuses(change, message):
    with pytest.raises(lib.RlqError, match=message):
        lib.call("rlq_causal_conv", *{**CONV, **change}.values())


@pytest.mark.parametrize("change,message", [
    (dict(T=-1), "T=-1"), (dict(B=-1), "B=-1"), (dict(T=1 << 27), "too large"), (dict(Dk=96), "key size 96"),
    (dict(Dk=256), "key size 256"), (dict(Dv=32), "value size 32"), (dict(dtype=2), "unknown dtype"),
    (dict(out_dtype=2), "output dtype"), (dict(v_heads=3), "evenly"), (dict(v_heads=1), "evenly"), (dict(k_heads=0), "evenly"),
    (dict(eps=0.0), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(scale=math.nan), "scale"),
    (dict(z=None), "together"), (dict(norm=None), "together"), (dict(norm_eps=0.0), "norm_eps"),
    (dict(norm_eps=math.inf), "norm_eps"), (dict(n_slots=-1), "n_slots=-1"), (dict(max_q=-1), "max_q=-1"),
    (dict(q=None), "null pointer"), (dict(a_log=None), "null pointer"), (dict(slots=None), "null pointer"),
    (dict(state=None), "16-byte aligned"), (dict(state=20), "16-byte aligned"), (dict(q_stride=127), "stride"),
    (dict(v_stride=255), "stride"), (dict(a_stride=3), "stride"), (dict(b_stride=3), "stride"), (dict(z_stride=255), "stride"),
    (dict(out_stride=255), "stride"), (dict(B=1 << 20, v_heads=4096, v_stride=1 << 18, a_stride=4096, b_stride=4096,
                                            z_stride=1 << 18, out_stride=1 << 18), "too many"),
    (dict(B=1 << 20, v_heads=64, v_stride=4096, a_stride=64, b_stride=64, z_stride=4096, out_stride=4096), "too many"),
    (dict(B=1 << 20, v_heads=16, v_stride=1024, a_stride=16, b_stride=16, z_stride=1024, out_stride=1024, max_q=1 << 24,
          workspace=16, workspace_bytes=1 << 40), "too many")])
def test_gated_delta_refuses(change, message):
    with pytest.raises(lib.RlqError, match=message):
        lib.call("rlq_gated_delta", *{**DELTA, **change}.values())


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows=-1"), (dict(rows=70000), "rows=70000"), (dict(vocab=0), "vocab=0"),
    (dict(vocab=(1 << 22) + 1, stride=1 << 23), "vocab="), (dict(logits=None), "null pointer"),
    (dict(uniform=None), "null pointer"), (dict(tokens=None), "null pointer"), (dict(stride=999), "stride"),
    (dict(workspace=None), "16-byte aligned workspace"), (dict(workspace=24), "16-byte aligned workspace"),
    (dict(workspace_bytes=100), "16-byte aligned workspace")])
def test_sample_refuses(change, message):
    with pytest.raises(lib.RlqError, match=message):
        lib.call("rlq_sample", *{**SAMPLE, **change}.values())


@pytest.mark.parametrize("change", [dict(workspace=None, workspace_bytes=1 << 40), dict(workspace=24, workspace_bytes=1 << 40),
                                    dict(workspace=16, workspace_bytes=1000)])
def test_gated_delta_in_chunks_refuses_other_scratch(change):
    with pytest.raises(lib.RlqError, match="16-byte aligned workspace"):
        lib.call("rlq_gated_delta", *{**DELTA, "max_q": 1000, **change}.values())


def test_workspace_queries():
    assert ops.gated_delta_workspace_bytes(1, 16, 32, 128, 128, 1, 1) == 0                # token by token
    one, two, long = (ops.gated_delta_workspace_bytes(T, 16, 32, 128, 128, 1, T) for T in (1000, 2000, 1 << 20))
    assert 0 < one < two < long < 400 << 20                                               # bounded, however long
    assert ops.gated_delta_workspace_bytes(0, 16, 32, 128, 128, 1, 100) == 0
    assert ops.gated_delta_workspace_bytes(100, 16, 8, 128, 128, 1, 100) == 0             # no such heads
    assert ops.sample_workspace_bytes(3, 1000) == 3 * ops.sample_workspace_bytes(1, 1000) > 0
    assert ops.sample_workspace_bytes(1, 1 << 23) == ops.sample_workspace_bytes(-1, 100) == 0


def test_calls_without_rows_do_nothing():
    for name, args, none in (("rlq_causal_conv", CONV, "x"), ("rlq_gated_delta", DELTA, "q")):
        assert lib.call(name, *{**args, "T": 0, none: None}.values()) == 0
        assert lib.call(name, *{**args, "B": 0, "cu_q": None}.values()) == 0
    assert lib.call("rlq_sample", *{**SAMPLE, "rows": 0, "logits": None}.values()) == 0


f32, f16, i32, f64 = torch.float32, torch.float16, torch.int32, torch.float64


def conv_args(**change):
    a = dict(x=torch.zeros(4, 64), weight=torch.zeros(64, 4), state=torch.zeros(3, 3, 64), cu_q=torch.zeros(2, dtype=i32),
             kv_len=torch.zeros(1, dtype=i32), slots=torch.zeros(1, dtype=i32))
    return {**a, **change}


@pytest.mark.parametrize("change,error", [
    (dict(x=torch.zeros(4, 64).half()), ValueError), (dict(x=torch.zeros(64, 4).t()), ValueError),
    (dict(weight=torch.zeros(63, 4)), ValueError), (dict(weight=torch.zeros(4, 64).t()), ValueError),
    (dict(weight=torch.zeros(64, 4).half()), ValueError), (dict(state=torch.zeros(3, 2, 64)), ValueError),
    (dict(state=torch.zeros(3, 3, 64).half()), ValueError), (dict(state=torch.zeros(3, 64, 3).transpose(1, 2)), ValueError),
    (dict(bias=torch.zeros(63)), ValueError), (dict(slots=torch.zeros(1, dtype=torch.int64)), TypeError),
    (dict(slots=torch.zeros(2, dtype=i32)), ValueError), (dict(cu_q=torch.zeros(1, dtype=i32)), ValueError),
    (dict(keep=torch.zeros(2, dtype=i32)), ValueError), (dict(keep=torch.zeros(1)), TypeError),
    (dict(out=torch.zeros(4, 63).half()), ValueError), (dict(out=torch.zeros(4, 64)), ValueError),
    (dict(out_dtype=f32), ValueError), ({}, ValueError)])     # the last: nothing is on a GPU
def test_causal_conv_checks_its_tensors(change, error):
    with pytest.raises(error):
        ops.causal_conv(**conv_args(**change))


def delta_args(**change):
    a = dict(q=torch.zeros(4, 128, dtype=f16), k=torch.zeros(4, 128, dtype=f16), v=torch.zeros(4, 256, dtype=f16),
             a=torch.zeros(4, 4), b=torch.zeros(4, 4), a_log=torch.zeros(4), dt_bias=torch.zeros(4),
             state=torch.zeros(3, 4, 64, 64), cu_q=torch.zeros(2, dtype=i32), kv_len=torch.zeros(1, dtype=i32),
             slots=torch.zeros(1, dtype=i32), max_q=4)
    return {**a, **change}


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(4, 128)), ValueError), (dict(k=torch.zeros(4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(4, 64, dtype=f16)), ValueError), (dict(q=torch.zeros(4, 100, dtype=f16)), ValueError),
    (dict(v=torch.zeros(5, 256, dtype=f16)), ValueError), (dict(v=torch.zeros(4, 128, dtype=f16)), ValueError),
    (dict(a=torch.zeros(4, 3)), ValueError), (dict(b=torch.zeros(4, 4).half()), ValueError),
    (dict(a_log=torch.zeros(3)), ValueError), (dict(dt_bias=torch.zeros(4, dtype=f64)), ValueError),
    (dict(state=torch.zeros(3, 4, 64, 64).half()), ValueError), (dict(state=torch.zeros(3, 4, 64, 64).transpose(2, 3)), ValueError),
    (dict(z=torch.zeros(4, 256)), ValueError), (dict(norm=torch.zeros(64)), ValueError),
    (dict(z=torch.zeros(4, 255), norm=torch.zeros(64)), ValueError), (dict(z=torch.zeros(4, 256), norm=torch.zeros(63)), ValueError),
    (dict(keep=torch.zeros(1)), TypeError), (dict(out=torch.zeros(4, 255).half()), ValueError),
    (dict(out_dtype=f32), ValueError), (dict(workspace=torch.zeros(4, 4).t()), ValueError), ({}, ValueError)])
def test_gated_delta_checks_its_tensors(change, error):
    with pytest.raises(error):
        ops.gated_delta(**delta_args(**change))


def sample_args(**change):
    return {**dict(logits=torch.zeros(2, 1000), uniform=torch.zeros(2, dtype=f64)), **change}


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(2, 1000).half()), dict(logits=torch.zeros(1000, 2).t()), dict(uniform=torch.zeros(2)),
    dict(uniform=torch.zeros(3, dtype=f64)), dict(temperature=torch.zeros(1)), dict(top_k=torch.zeros(2)),
    dict(top_p=torch.zeros(2, dtype=f64)), dict(min_p=torch.zeros(2, 1)), dict(out=torch.zeros(2, dtype=torch.int64)),
    dict(probs=torch.zeros(3)), dict(workspace=torch.zeros(4, 4).t()), {}])
def test_sample_checks_its_tensors(change):
    with pytest.raises(ValueError):
        ops.sample(**sample_args(**change))


def test_gated_delta_goes_token_by_token_where_chunks_have_no_room():
    """32768 sequences of 32 heads of 128 and more: whatever max_q is, and without scratch. Below, max_q chooses."""
    for heads, dv, border in ((32, 128, 1 << 15), (16, 256, 1 << 15), (8, 64, 1 << 18)):
        assert ops.gated_delta_workspace_bytes(1 << 20, 1, heads, 64, dv, border - 1, 1 << 20) > 0
        assert ops.gated_delta_workspace_bytes(1 << 20, 1, heads, 64, dv, border, 1 << 20) == 0
