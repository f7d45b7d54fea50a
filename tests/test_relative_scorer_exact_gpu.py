"""GPU tests of the transformer scorer's relative positions, bit for bit: what its graph leaves in the activation buffers
against the operators' own calls on the same tensors."""

import numpy as np
import pytest
import torch

from multigpubeamsearch_b200 import operators as ops
from multigpubeamsearch_b200 import puzzles, scorers

pytestmark = pytest.mark.gpu

TOKENS = 54


def states(count, seed):
    rng = np.random.default_rng(seed)
    out = np.zeros((count, 64), np.uint8)
    out[:, :TOKENS] = rng.integers(0, 6, size=(count, TOKENS))
    return torch.from_numpy(out).cuda()


def weights(layers, norm, bias, base, buckets, model):
    rng = np.random.default_rng(51 + model)
    w = puzzles.transformer_weights(TOKENS, 6, layers=layers, model_idx=model)
    w.update(rotary_base=base, rel_buckets=buckets, qk_eps=1e-5)
    for L in w["layers"]:
        gains = [(1 + 0.2 * rng.standard_normal(32)).astype(np.float32) for _ in range(2)]
        table = torch.from_numpy(rng.standard_normal((buckets[0], 8)).astype(np.float32)).bfloat16().float().numpy()
        if norm:
            L["q_gain"], L["k_gain"] = gains
        if bias:
            L["rel_table"] = table
    return w


def run(ws, rows, micro, dtype):
    sc = scorers.TransformerValueScorer(ws, TOKENS, 64, 6, max_rows=len(rows), micro_batch=micro, dtype=dtype)
    sc.score(rows)
    torch.cuda.synchronize()
    assert sc.error_code() == 0
    held = len(rows) - (len(rows) - 1) // micro * micro  # states of the last micro-batch, which the buffers keep
    qkv = sc.qkv[:held * TOKENS].view(held, TOKENS, 3, 8, 32)
    return qkv, sc.att[:held * TOKENS].view(held, TOKENS, 8, 32)


@pytest.mark.parametrize("count,micro", [(300, 32768), (257, 64), (191, 64), (1, 8)])
@pytest.mark.parametrize("base,buckets", [(10000.0, (32, 128)), (None, (16, 20)), (100.0, (64, 60))])
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
def test_queries_and_keys_in_place(count, micro, base, buckets, dtype):
    """One layer: its buffer without the norm, normalised and rotated by the operator, is its buffer with the norm."""
    rows = states(count, seed=count)
    raw, _ = run([weights(1, False, False, base, buckets, i) for i in range(2)], rows, micro, dtype)
    ws = [weights(1, True, dtype == "bf16", base, buckets, i) for i in range(2)]
    got, att = run(ws, rows, micro, dtype)
    freq = {"inv_freq": [0.0] * 16} if base is None else {"base": base}
    gains = [torch.from_numpy(ws[-1]["layers"][0][n]).cuda() for n in ("q_gain", "k_gain")]
    q, k = ops.qk_norm_rope(raw[:, :, 0], raw[:, :, 1], *gains, ops.RotaryFrequencies(32, **freq), eps=1e-5)
    assert torch.equal(got[:, :, 0], q) and torch.equal(got[:, :, 1], k) and torch.equal(got[:, :, 2], raw[:, :, 2])
    assert not torch.equal(got[:, :, 0], raw[:, :, 0])


@pytest.mark.parametrize("count,micro", [(300, 32768), (257, 64), (191, 64), (1, 8)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("buckets", [(32, 128), (16, 20), (64, 60), (4, 2)])
def test_attention_with_the_table(count, micro, norm, buckets):
    """The last layer's attention output is the operator's on the queries, keys and values beside it."""
    ws = [weights(2, norm, True, 10000.0, buckets, i) for i in range(2)]
    qkv, att = run(ws, states(count, seed=count), micro, "bf16")
    table = torch.from_numpy(ws[-1]["layers"][-1]["rel_table"]).cuda().bfloat16()
    want = ops.relative_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], table, ops.RelativeBuckets(*buckets))
    assert torch.equal(att, want)
    # and a bias of another distance would be seen
    other = ops.relative_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], table.roll(1, 0), ops.RelativeBuckets(*buckets))
    assert not torch.equal(att, other)
