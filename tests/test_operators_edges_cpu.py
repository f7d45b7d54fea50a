"""CPU checks of the operators' edges: what the C entries let through and refuse, and what the functions refuse before they
look at a tensor's device."""

import ctypes as C

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
