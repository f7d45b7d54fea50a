"""GPU tests of the operators at edges of what their documentation allows: values with a common mean, eps of 0, NaN among
masks, huge values behind masks, calls whose results must not depend on earlier ones."""

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from multigpubeamsearch_b200 import operators as ops

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def normal(gen, *shape, dtype=torch.float32, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") + mean).to(dtype)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------------------------------------------
# Query and key norm
# ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("b,t,h,hk,d,dtype", [(1, 1, 1, 1, 32, torch.bfloat16), (1, 1, 3, 1, 96, torch.float32), (3, 11, 5, 2, 48, torch.float16),
                                              (2, 333, 8, 8, 32, torch.bfloat16), (1, 65, 2, 2, 256, torch.float32)])
def test_qk_norm_rope_without_eps(b, t, h, hk, d, dtype):
    """eps = 0 and no zero vector: all results are the definition's, whatever slots of the last block have no token."""
    gen = generator(b * t)
    x = [normal(gen, b, t, n, d, dtype=dtype).requires_grad_(True) for n in (h, hk)]
    gain = [(1 + 0.2 * normal(gen, d)).requires_grad_(True) for _ in range(2)]
    dy = [normal(gen, *y.shape, dtype=dtype) for y in x]
    rotary = ops.RotaryFrequencies(d, inv_freq=[0.0] * (d // 2))  # turns nothing
    out = ops.qk_norm_rope(*x, *gain, rotary, eps=0.0)
    got = torch.autograd.grad(out, [*x, *gain], dy)
    u = torch.finfo(dtype).eps / 2
    for i in range(2):
        xd, gd = x[i].detach().double().requires_grad_(True), gain[i].detach().double().requires_grad_(True)
        y = gd * xd / xd.square().mean(-1, keepdim=True).sqrt()
        dx, dg = torch.autograd.grad(y, (xd, gd), dy[i].double())
        # one rounding of each result, and 2^-18 for the float32 steps (sums of at most 666 terms and of 256 squares)
        assert ((out[i].double() - y).abs() <= (u + 2.0 ** -18) * y.abs()).all()
        assert (got[i].double() - dx).norm() <= (u + 2.0 ** -18) * dx.norm()
        assert (got[2 + i].double() - dg).norm() <= 2.0 ** -18 * dg.norm()


EARLIER_CALLS = """
import hashlib, sys, torch
from multigpubeamsearch_b200 import operators as ops

def call(b, t, h, hk, train):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn((b, t, n, 32), generator=gen, device="cuda").bfloat16().requires_grad_(train) for n in (h, hk)]
    gain = [torch.ones(32, device="cuda", requires_grad=train) for _ in range(2)]
    out = ops.qk_norm_rope(*x, *gain, ops.RotaryFrequencies(32))
    return torch.autograd.grad(out, [*x, *gain], [torch.randn(y.shape, generator=gen, device="cuda").bfloat16() for y in out]) if train else out

if sys.argv[1] == "other":
    call(4, 128, 8, 8, False)
print(hashlib.sha256(b"".join(g.view(torch.uint8).cpu().numpy().tobytes() for g in call(1, 100001, 2, 1, True))).hexdigest())
"""


def test_qk_norm_rope_does_not_depend_on_earlier_calls():
    """A gradient's bits in a process of its own and in one that called a forward of another shape first."""
    root = Path(__file__).resolve().parents[1]
    said = [subprocess.run([sys.executable, "-c", EARLIER_CALLS, first], cwd=root, capture_output=True, text=True, timeout=600, check=True).stdout
            for first in ("nothing", "other")]
    assert said[0] == said[1]


def test_qk_norm_rope_no_tokens_with_positions():
    """Batches without a sequence and sequences without a token, with positions given: empty results, zero gradients."""
    rotary = ops.RotaryFrequencies(32)
    for b, t, shape in ((0, 5, (0, 5)), (3, 0, (3, 0)), (2, 0, (0,)), (0, 5, (5,))):
        for dtype in (torch.int32, torch.int64):
            q = torch.zeros(b, t, 2, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
            gain = torch.ones(32, device="cuda", requires_grad=True)
            out = ops.qk_norm_rope(q, q[:, :, :1], gain, gain, rotary, positions=torch.zeros(shape, device="cuda", dtype=dtype))
            assert out[0].shape == q.shape and out[1].shape == (b, t, 1, 32)
            grads = torch.autograd.grad(out, (q, gain), [torch.zeros_like(y) for y in out])
            assert grads[0].shape == q.shape and not grads[1].any()


# ---------------------------------------------------------------------------------------------------------------
# Distillation: a NaN among closed columns
# ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("width", [1000, 1025, 3001, 50021, 300007])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fill", [-math.inf, -3.0e38, -1.0e7])
def test_distill_nan_among_closed_columns(width, dtype, fill):
    """All columns from 6 on closed but for a NaN somewhere among them: loss and gradient of that row are NaN, others are not."""
    gen = generator(width)
    places = sorted({7, 2064 % width, width // 3, width // 2, width - 130, width - 1})
    logits = normal(gen, len(places) + 1, width, dtype=dtype)
    logits[:, 6:] = fill
    for row, at in enumerate(places):
        logits[row, max(at, 6)] = math.nan
    teacher = normal(gen, len(places) + 1, 3)
    index = torch.tensor([0, 3, 5], device="cuda").expand(len(places) + 1, 3).contiguous()
    alone = ops.distill_top_logits(logits, teacher, index)
    loss, grad = ops.distill_top_logits_step(logits, teacher, index)
    for got in (alone, loss):
        assert got[:-1].isnan().all() and got[-1].isfinite(), (places, got)
    assert grad[:-1].isnan().all() and grad[-1].isfinite().all()


# ---------------------------------------------------------------------------------------------------------------
# Attention: huge values behind masks
# ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("closed", [-math.inf, -3.0e38, -1.0e4])
@pytest.mark.parametrize("tokens,d", [(40, 32), (700, 64), (700, 32)])
def test_relative_attention_huge_values_behind_a_mask(tokens, d, closed):
    """Keys beyond a distance closed by the table hold values near the type's largest: they weigh nothing."""
    gen = generator(tokens + d)
    b, h, dtype, u = 1, 2, torch.bfloat16, 2.0 ** -8
    q, k = normal(gen, b, tokens, h, d, dtype=dtype), normal(gen, b, tokens, h, d, dtype=dtype)
    plan = ops.RelativeBuckets(32, 16 if tokens < 64 else 128)
    table = normal(gen, 32, h, dtype=dtype)
    table[15] = table[31] = closed  # the last bucket of either side
    reach = next(i for i in range(plan.max_distance + 1) if int(plan.map[plan.max_distance + i]) == 31)
    v = normal(gen, b, tokens, h, d, dtype=dtype)
    rows = max(1, tokens // 2 - reach)  # the first rows see none of the last tokens
    v[:, tokens // 2:] = 1.0e38
    out = ops.relative_attention(q, k, v, table, plan)[:, :rows].double()
    off = torch.arange(tokens, device="cuda")[None] - torch.arange(rows, device="cuda")[:, None]
    index = plan.map.long()[off.clamp(-plan.max_distance, plan.max_distance) + plan.max_distance]
    s = torch.einsum("bihd,bjhd->bhij", q[:, :rows].double(), k.double()) * d ** -0.5 + table.double()[index].permute(2, 0, 1)
    p = s.softmax(-1)
    p = torch.where(index == 31, 0.0, p)  # exp(-1e4 + a few) is 0 in any format that holds 1e38 finite
    want, size = torch.einsum("bhij,bjhd->bihd", p, v.double()), torch.einsum("bhij,bjhd->bihd", p, v.double().abs())
    assert ((out - want).abs() <= (2 * u + 2.0 ** -14) * size).all()
