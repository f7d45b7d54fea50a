"""CPU checks of the operators' host side: structure mirrors, bucket borders, rotation fractions, and the C entries'
refusals (each returns its error before anything is enqueued, so no GPU is needed)."""

import ctypes as C
import math
from fractions import Fraction

import pytest
import torch

from multigpubeamsearch_b200 import _lib, operators as ops

ERR_ARG, ERR_UNSUPPORTED, ERR_TOO_LARGE = -1, -2, -5
SOME = 1 << 20  # an address that is aligned and never read: every call below is refused


def test_structures_match():
    lib = ops._load()
    assert lib.mgbs_sizeof_qk_norm_args() == C.sizeof(ops.MgbsQkNormArgs)
    assert lib.mgbs_sizeof_rel_attention_args() == C.sizeof(ops.MgbsRelAttentionArgs)
    assert lib.mgbs_sizeof_distill_args() == C.sizeof(ops.MgbsDistillArgs)


@pytest.mark.parametrize("num_buckets,max_distance,causal", [(32, 128, False), (32, 128, True), (4, 2, False), (2, 2, True), (64, 1024, False), (10, 100, False), (7, 30, True)])
def test_buckets_follow_the_definition_in_exact_fractions(num_buckets, max_distance, causal):
    plan = ops.RelativeBuckets(num_buckets, max_distance, causal, device="cpu")
    side = num_buckets if causal else num_buckets // 2
    exact = side // 2
    got = plan.map.tolist()
    assert len(got) == 2 * max_distance + 1 and 0 <= min(got) and max(got) < num_buckets
    for off in range(-max_distance, max_distance + 1):
        n = max(-off, 0) if causal else abs(off)
        if n >= exact:
            # floor(log(n / exact) / log(max / exact) * steps), decided by powers: (n/exact)^steps >= (max/exact)^s
            steps = side - exact
            s = max(s for s in range(steps + 1) if Fraction(n, exact) ** steps >= Fraction(max_distance, exact) ** s)
            n = exact + min(s, steps - 1)
        assert got[off + max_distance] == n + (side if not causal and off > 0 else 0), off
    order, start = plan.order.tolist(), plan.start.tolist()
    assert sorted(order) == list(range(2 * max_distance + 1)) and start[0] == 0 and start[-1] == len(order)
    for b in range(num_buckets):
        assert all(got[i] == b for i in order[start[b]:start[b + 1]])


@pytest.mark.parametrize("args", [dict(num_buckets=3), dict(num_buckets=2), dict(num_buckets=514), dict(num_buckets=1, causal=True), dict(max_distance=8), dict(max_distance=1025)])
def test_buckets_refuse(args):
    with pytest.raises(RuntimeError):
        ops.RelativeBuckets(**args, device="cpu")


def test_rotation_fractions():
    plan = ops.RotaryFrequencies(64, base=10000.0, device="cpu")
    for i, t in enumerate(plan.phase.tolist()):
        turn = (t % (1 << 64)) / 2.0 ** 64
        assert abs(turn - 10000.0 ** (-2 * i / 64) / (2 * math.pi)) < 2.0 ** -52
    own = ops.RotaryFrequencies(4, inv_freq=[1.0, -0.5], device="cpu")
    assert own.phase[1].item() < 0
    for bad in (dict(head_dim=3), dict(head_dim=4, inv_freq=[1.0]), dict(head_dim=2, inv_freq=[math.inf]), dict(head_dim=2, base=0.0)):
        with pytest.raises(RuntimeError):
            ops.RotaryFrequencies(**bad, device="cpu")


def test_functions_refuse_cpu_tensors():
    q = torch.zeros(1, 2, 1, 32, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.relative_attention(q, q, q, torch.zeros(32, 1, dtype=torch.bfloat16), ops.RelativeBuckets(device="cpu"))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qk_norm_rope(q, q, torch.ones(32), torch.ones(32), ops.RotaryFrequencies(32, device="cpu"))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.distill_top_logits(torch.zeros(2, 4), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64))


def qk_args(**more):
    a = ops.MgbsQkNormArgs(dtype=0, head_dim=32, heads_q=2, heads_k=1, batch=2, tokens=3, eps=1e-6)
    for n in ("q", "k", "q_out", "k_out", "q_gain", "k_gain", "phase", "dq_out", "dk_out", "dq_gain", "dk_gain", "workspace"):
        setattr(a, n, SOME)
    for n, v in more.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("more,code", [
    (dict(dtype=3), ERR_UNSUPPORTED), (dict(dtype=-1), ERR_UNSUPPORTED), (dict(head_dim=33), ERR_UNSUPPORTED), (dict(head_dim=0), ERR_UNSUPPORTED),
    (dict(head_dim=258), ERR_UNSUPPORTED), (dict(heads_q=0), ERR_ARG), (dict(heads_k=0), ERR_ARG), (dict(batch=-1), ERR_ARG),
    (dict(batch=1 << 20, tokens=1 << 12), ERR_TOO_LARGE), (dict(eps=-1.0), ERR_ARG), (dict(eps=math.nan), ERR_ARG), (dict(q=None), ERR_ARG),
    (dict(k_out=None), ERR_ARG), (dict(q_gain=None), ERR_ARG), (dict(phase=None), ERR_ARG), (dict(position_bits=16), ERR_ARG),
    (dict(position_bits=32), ERR_ARG)])
def test_qk_norm_rope_refuses(more, code):
    lib = ops._load()
    assert lib.mgbs_qk_norm_rope(C.byref(qk_args(**more)), None) == code
    assert lib.mgbs_qk_norm_rope_backward(C.byref(qk_args(**more)), None) == code


@pytest.mark.parametrize("name", ["dq_out", "dk_out", "dq_gain", "dk_gain", "workspace"])
def test_qk_norm_rope_backward_refuses(name):
    assert ops._load().mgbs_qk_norm_rope_backward(C.byref(qk_args(**{name: None})), None) == ERR_ARG


def rel_args(**more):
    a = ops.MgbsRelAttentionArgs(dtype=0, head_dim=32, heads=2, heads_kv=1, batch=2, tokens=80, num_buckets=32, max_distance=128, scale=0.2)
    for n in ("q", "k", "v", "table", "bucket_map", "bucket_order", "bucket_start", "out", "stats", "dout", "dq", "dk", "dv", "dtable", "workspace"):
        setattr(a, n, SOME)
    for n in ("q_stride", "k_stride", "v_stride", "dout_stride"):
        getattr(a, n)[:] = (80 * 64, 64, 32)
    for n, v in more.items():
        if n.endswith("stride"):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


@pytest.mark.parametrize("more,code", [
    (dict(dtype=2), ERR_UNSUPPORTED), (dict(head_dim=48), ERR_UNSUPPORTED), (dict(head_dim=128), ERR_UNSUPPORTED), (dict(heads=3, heads_kv=2), ERR_ARG),
    (dict(heads=0), ERR_ARG), (dict(heads_kv=0), ERR_ARG), (dict(heads=1026, heads_kv=1), ERR_TOO_LARGE), (dict(tokens=(1 << 20) + 1), ERR_TOO_LARGE),
    (dict(batch=-1), ERR_ARG), (dict(tokens=-1), ERR_ARG), (dict(num_buckets=0), ERR_ARG), (dict(num_buckets=513), ERR_ARG), (dict(max_distance=0), ERR_ARG),
    (dict(max_distance=1025), ERR_ARG), (dict(scale=0.0), ERR_ARG), (dict(scale=-1.0), ERR_ARG), (dict(scale=math.nan), ERR_ARG), (dict(scale=math.inf), ERR_ARG),
    (dict(q=None), ERR_ARG), (dict(out=None), ERR_ARG), (dict(table=None), ERR_ARG), (dict(bucket_map=None), ERR_ARG), (dict(bucket_start=None), ERR_ARG),
    (dict(q=SOME + 2), ERR_UNSUPPORTED), (dict(k_stride=(80 * 64, 60, 32)), ERR_UNSUPPORTED), (dict(out=SOME + 8), ERR_UNSUPPORTED)])
def test_relative_attention_refuses(more, code):
    lib = ops._load()
    assert lib.mgbs_rel_attention(C.byref(rel_args(**more)), None) == code
    assert lib.mgbs_rel_attention_backward(C.byref(rel_args(**more)), None) == code


@pytest.mark.parametrize("more,code", [(dict(dout=None), ERR_ARG), (dict(dq=None), ERR_ARG), (dict(dtable=None), ERR_ARG), (dict(workspace=None), ERR_ARG),
                                       (dict(stats=None), ERR_ARG), (dict(dout_stride=(80 * 64, 64, 31)), ERR_UNSUPPORTED), (dict(dv=SOME + 4), ERR_UNSUPPORTED)])
def test_relative_attention_backward_refuses(more, code):
    assert ops._load().mgbs_rel_attention_backward(C.byref(rel_args(**more)), None) == code


def distill_args(**more):
    a = ops.MgbsDistillArgs(dtype=0, entries=3, rows=4, width=12, index_bits=64, row_stride=12, grad_stride=12, teacher_stride=3, index_stride=3, temperature=1.0)
    a.logits, a.teacher, a.index, a.loss, a.grad = SOME, 2 * SOME, 3 * SOME, 4 * SOME, 5 * SOME
    for n, v in more.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("more,code", [
    (dict(dtype=5), ERR_UNSUPPORTED), (dict(entries=0), ERR_ARG), (dict(entries=1025), ERR_TOO_LARGE), (dict(rows=-1), ERR_ARG), (dict(width=0), ERR_ARG),
    (dict(index_bits=16), ERR_ARG), (dict(temperature=0.0), ERR_ARG), (dict(temperature=-1.0), ERR_ARG), (dict(temperature=math.nan), ERR_ARG),
    (dict(temperature=1e-39), ERR_ARG), (dict(logits=None), ERR_ARG), (dict(teacher=None), ERR_ARG), (dict(index=None), ERR_ARG), (dict(loss=None), ERR_ARG),
    (dict(grad=SOME), ERR_ARG), (dict(logits=SOME + 1), ERR_ARG)])
def test_distill_refuses(more, code):
    assert ops._load().mgbs_distill_top_logits(C.byref(distill_args(**more)), None) == code


def test_empty_calls_do_nothing():
    lib = ops._load()
    assert lib.mgbs_qk_norm_rope(C.byref(qk_args(batch=0)), None) == 0
    assert lib.mgbs_rel_attention(C.byref(rel_args(batch=0)), None) == 0
    assert lib.mgbs_distill_top_logits(C.byref(distill_args(rows=0)), None) == 0


def test_error_names():
    with pytest.raises(RuntimeError, match="too large"):
        _lib.check(ERR_TOO_LARGE, "relative_attention")


def test_transformer_config_mirrors():
    from multigpubeamsearch_b200 import scorers

    lib = ops._load()
    lib.mgbs_sizeof_tf_config.restype = C.c_int
    assert lib.mgbs_sizeof_tf_config() == C.sizeof(scorers.MgbsTfConfig)
