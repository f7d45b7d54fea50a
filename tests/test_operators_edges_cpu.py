"""CPU checks of the operators' edges: what the C entries let through and refuse, and what the functions refuse before they
look at a tensor's device."""

import ctypes as C
import re
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from multigpubeamsearch_b200 import operators as ops, scorers

ERR_ARG, ERR_UNSUPPORTED = -1, -2
SOME = 1 << 20  # an address that is aligned and never read: no call below enqueues anything


@pytest.mark.parametrize("batch,tokens", [(0, 5), (3, 0), (0, 0)])
@pytest.mark.parametrize("bits", [32, 64])
def test_no_tokens_need_no_positions(batch, tokens, bits):
    a = ops.MgbsQkNormArgs(dtype=0, head_dim=32, heads_q=2, heads_k=1, batch=batch, tokens=tokens, eps=1e-6, position_bits=bits,
                           q_gain=SOME, k_gain=SOME, phase=SOME)
    assert ops._load().mgbs_qk_norm_rope(C.byref(a), None) == 0
    a.batch, a.tokens, a.q, a.k, a.q_out, a.k_out = 1, 1, SOME, SOME, SOME, SOME
    assert ops._load().mgbs_qk_norm_rope(C.byref(a), None) == ERR_ARG


# how wide the kernels access arrays in shared memory through another type or by vector instructions
WIDE_ACCESS = {
    "mgbs_distill.cu": {"held": 16, "s_seen": 16},
    "mgbs_qk_norm.cu": {"angles": 16},
    "mgbs_rel_attention.cu": {"rel_smem": 16, "row_stat": 16, "row_delta": 8},
    "mgbs_rel_attention_tc.cu": {"tc_smem": 1024, "bars": 8},
    "mgbs_rel_attention_tc_bwd.cu": {"tc_smem": 1024, "bars": 8, "stat": 16},
}


@pytest.mark.parametrize("name", WIDE_ACCESS)
def test_shared_arrays_declare_their_alignment(name):
    """An array that is read or written wider than its elements says so, instead of resting on the compiler's layout."""
    text = (Path(ops.__file__).parent / "csrc" / name).read_text()
    for array, width in WIDE_ACCESS[name].items():
        found = re.findall(r"__shared__\s+(?:__align__\((\d+)\)\s+)?[\w:]+\s+(?:\w+(?:\[[^;]*?\])+,\s*)*" + array + r"\[", text)
        assert found and all(a and int(a) >= width for a in found), (array, found)
    # every other one is accessed by its own elements only
    for array in re.findall(r"__shared__(?:\s+__align__\(\d+\))?\s+[\w:]+\s+(\w+)\[", text):
        if array not in WIDE_ACCESS[name]:
            assert not re.search(r"reinterpret_cast<(?:const )?(?:uint4|float4|float2|int4|uint2)\*>\(&?" + array + r"\b", text), array


def test_sums_sent_between_blocks_are_aligned():
    text = (Path(ops.__file__).parent / "csrc" / "mgbs_distill.cu").read_text()
    assert "st.shared::cluster.v2.b32" in text and "struct __align__(8) Sum" in text


def calls():
    """Each function on CPU tensors, as (call, its differentiable arguments): refused for a reason that comes before the device's."""
    q = torch.zeros(1, 2, 1, 32, dtype=torch.bfloat16)
    gain, table = torch.ones(32), torch.zeros(32, 1, dtype=torch.bfloat16)
    logits, teacher, index = torch.zeros(2, 4), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64)
    rotary, plan = ops.RotaryFrequencies(32, device="cpu"), ops.RelativeBuckets(device="cpu")
    return {
        "qk_norm_rope": (lambda q, k, g, h: ops.qk_norm_rope(q, k, g, h, rotary), (q, q, gain, gain)),
        "relative_attention": (lambda q, k, v, t: ops.relative_attention(q, k, v, t, plan), (q, q, q, table)),
        "distill_top_logits": (lambda z: ops.distill_top_logits(z, teacher, index), (logits,)),
        "distill_top_logits_step": (lambda z: ops.distill_top_logits_step(z, teacher, index), (logits,)),
    }


@pytest.mark.parametrize("name", calls())
def test_forward_mode_is_refused(name):
    call, leaves = calls()[name]
    for n in range(len(leaves)):
        with forward_ad.dual_level():
            args = [x.clone() for x in leaves]
            args[n] = forward_ad.make_dual(args[n], torch.ones_like(args[n]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*args)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="CUDA"):  # a level without a tangent is none of its business
        call(*leaves)


@pytest.mark.parametrize("name", calls())
def test_tracing_is_refused(name):
    call, leaves = calls()[name]
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(call, leaves, check_trace=False)
    with pytest.raises(RuntimeError, match="recorded"):
        make_fx(call)(*leaves)


@pytest.mark.parametrize("function,count", [(ops._QkNormRope, 2), (ops._RelativeAttention, 1), (ops._DistillTopLogits, 1)])
def test_forward_mode_over_a_backward_is_refused(function, count):
    with forward_ad.dual_level():
        grads = [forward_ad.make_dual(torch.zeros(3), torch.ones(3)) for _ in range(count)]
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            function.backward(None, *grads)


def encoder_config(**more):
    """A transformer scorer's configuration with relative positions in layer 1, its pointers never read."""
    c = scorers.MgbsTfConfig(state_len=54, state_stride=64, num_values=6, d_model=256, heads=8, ffn=1024, layers=2, encoders=1, max_states=8,
                             micro_batch=8, qk_eps=1e-6, rel_buckets=32, rel_distance=128)
    for n in ("x", "y", "qkv", "att", "hid", "q", "err", "rel_map", "rel_order", "rel_start"):
        setattr(c, n, SOME)
    c.rotary_phase[0] = SOME
    for n in ("q_gain", "k_gain", "rel_table"):
        setattr(c.layer[0][1], n, SOME)
    for n, v in more.items():
        if n in ("q_gain", "k_gain", "rel_table"):
            setattr(c.layer[0][1], n, v)
        elif n == "rotary_phase":
            c.rotary_phase[0] = v
        else:
            setattr(c, n, v)
    return c


@pytest.mark.parametrize("bad,code", [(dict(rel_buckets=0), ERR_ARG), (dict(rel_buckets=513), ERR_ARG), (dict(rel_distance=0), ERR_ARG),
                                      (dict(rel_distance=1025), ERR_ARG), (dict(qk_eps=-1.0), ERR_ARG), (dict(qk_eps=float("nan")), ERR_ARG),
                                      (dict(qk_eps=float("inf")), ERR_ARG), (dict(q_gain=None), ERR_ARG), (dict(rotary_phase=None), ERR_ARG),
                                      (dict(rel_start=None), ERR_ARG), (dict(dtype=1), ERR_UNSUPPORTED)])
def test_transformer_with_relative_positions_is_refused_when_created(bad, code):
    """Not by a call of its own kernels later on: nothing of the rest of this configuration is looked at before."""
    c, handle, made = encoder_config(**bad), C.c_void_p(), False
    lib = ops._load()
    try:
        rc = lib.mgbs_tf_create(C.byref(c), C.byref(handle))
        made = rc == 0
    finally:
        if made:
            lib.mgbs_tf_destroy(handle)
    assert rc == code
