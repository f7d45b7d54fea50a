"""CPU checks of the operators' edges: what the C entries let through and refuse, and what the functions refuse before they
look at a tensor's device."""

import ctypes as C
import re
from pathlib import Path

import pytest

from multigpubeamsearch_b200 import operators as ops

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
