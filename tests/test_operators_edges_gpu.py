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


# ---------------------------------------------------------------------------------------------------------------
# The table's gradient where the values have a common mean
# ---------------------------------------------------------------------------------------------------------------


def definition(q, k, v, table, plan, lengths, dout):
    """Output and gradients in 64 bits, by differentiation."""
    b, t, h, d = q.shape
    off = torch.arange(t, device="cuda")[None] - torch.arange(t, device="cuda")[:, None]
    index = plan.map.long()[off.clamp(-plan.max_distance, plan.max_distance) + plan.max_distance]
    live = torch.ones(b, t, dtype=torch.bool, device="cuda") if lengths is None else torch.arange(t, device="cuda") < lengths[:, None]
    seen = live[:, None, :, None] & live[:, None, None, :]
    if plan.causal:
        seen = seen & (off <= 0)
    leaves = [x.detach().double().requires_grad_(True) for x in (q, k, v, table)]
    share = h // k.shape[2]
    qd, kd, vd = leaves[0].transpose(1, 2), *(x.transpose(1, 2).repeat_interleave(share, 1) for x in leaves[1:3])
    s = qd @ kd.transpose(-1, -2) * d ** -0.5 + leaves[3][index].permute(2, 0, 1)
    s = torch.where(seen, s, -1e300)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e290).detach())  # 0 all along a row without keys
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-290)
    out = (p @ vd).transpose(1, 2)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout.double() * live[:, :, None, None])]


MEAN_CASES = [
    # batch, tokens, heads, key heads, head_dim, type, causal, ragged, buckets, reach, mean of v
    (3, 54, 8, 8, 32, "bf16", False, False, 32, 128, 4.0),
    (2, 65, 4, 4, 64, "bf16", False, False, 32, 128, 4.0),
    (2, 40, 4, 2, 64, "f16", False, False, 32, 128, 4.0),
    (2, 63, 8, 1, 32, "bf16", True, True, 32, 40, 2.0),
    (2, 300, 2, 2, 64, "f16", False, True, 32, 128, 4.0),
    (1, 1001, 2, 2, 64, "bf16", False, False, 32, 128, 4.0),
    (1, 1001, 2, 2, 64, "f16", False, False, 32, 1024, 4.0),
    (1, 1001, 2, 1, 64, "f16", False, False, 4, 2, 4.0),
    (2, 777, 4, 2, 32, "f16", True, True, 32, 128, 1.0),
    (1, 1001, 11, 1, 32, "bf16", False, True, 8, 5, 3.0),
    (1, 1501, 4, 2, 64, "bf16", True, False, 32, 128, 0.0),
    (2, 449, 2, 2, 32, "bf16", False, False, 32, 128, 0.0),
    (1, 640, 2, 2, 32, "bf16", False, True, 32, 128, 0.0),
    (2, 321, 4, 2, 64, "bf16", True, True, 32, 128, 0.0),
    (9, 33, 8, 4, 32, "f16", False, False, 32, 128, 0.0),
    (30, 54, 8, 8, 32, "bf16", False, True, 32, 128, 0.0),
]


def mean_inputs(case, seed, broadcast=False):
    b, t, h, hk, d, dtype, causal, ragged, buckets, reach, mean = case
    gen, dt = generator(seed), TYPES[dtype]
    q, k, v = normal(gen, b, t, h, d, dtype=dt), normal(gen, b, t, hk, d, dtype=dt), normal(gen, b, t, hk, d, dtype=dt, mean=mean)
    plan = ops.RelativeBuckets(buckets, reach, causal=causal)
    lengths = torch.randint(t // 2, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32) if ragged else None
    return q, k, v, normal(gen, buckets, h, dtype=dt), plan, lengths, normal(gen, b, t, h, d, dtype=dt)


def check_gradients(q, k, v, table, plan, lengths, dout):
    u = torch.finfo(q.dtype).eps / 2
    want = definition(q, k, v, table, plan, lengths, dout)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, table)]
    out = ops.relative_attention(*leaves, plan, lengths=lengths)
    got = torch.autograd.grad(out, leaves, dout)
    # The table's gradient is a float32 sum, rounded once: u of each entry.  A pair's P (dP - delta) is off by some 2^-20 of
    # P (|dP| + |delta|), each below 8 (1 + mean) of the spread sqrt(head_dim) that dP - delta has, and pair for pair on its
    # own: 2^-20 * 80 < 2^-13 of what the pairs add up to, in an entry that is not small beside the largest one.
    off, size = (got[3].double() - want[4]).abs(), want[4].abs()
    assert (off <= u * size + 2.0 ** -12 * size.max()).all(), ("dtable", float((off / size.max()).max() / u))
    assert off.norm() <= 2 * u * size.norm(), ("dtable", float(off.norm() / size.norm() / u))
    # dq, dk, dv: P and dS are rounded before their products, each term on its own (u / sqrt(3) of it, in quadrature), and the
    # results once more: 2 u of the 2-norm with room, where the terms of dS k and dS^T q do not cancel.
    for name, g, w in zip(("dq", "dk", "dv"), got, want[1:]):
        error = (g.double() - w).norm() / w.norm()
        assert error <= 2 * u, (name, float(error / u))


@pytest.mark.parametrize("case", MEAN_CASES, ids=str)
def test_relative_attention_gradients_with_a_mean(case):
    check_gradients(*mean_inputs(case, seed=1))


@pytest.mark.parametrize("case", [MEAN_CASES[4], MEAN_CASES[5], MEAN_CASES[9]], ids=str)
def test_relative_attention_gradients_with_a_mean_broadcast(case):
    """One sequence's keys for several (a stride of 0, which the tile form takes)."""
    q, k, v, table, plan, lengths, dout = mean_inputs(case, seed=2)
    gen = generator(3)
    b, t, h, d = q.shape
    q, dout = (normal(gen, 2 * b, t, h, d, dtype=q.dtype) for _ in range(2))
    k, v = (x[:1].expand(2 * b, -1, -1, -1) for x in (k, v))
    check_gradients(q, k, v, table, plan, None if lengths is None else lengths.repeat(2), dout)


# ---------------------------------------------------------------------------------------------------------------
# Transforms
# ---------------------------------------------------------------------------------------------------------------


def small_calls():
    gen, rotary, plan = generator(50), ops.RotaryFrequencies(32), ops.RelativeBuckets()
    q, gain, table = normal(gen, 2, 70, 2, 32, dtype=torch.bfloat16), torch.ones(32, device="cuda"), normal(gen, 32, 2, dtype=torch.bfloat16)
    logits, teacher, index = normal(gen, 3, 2000), normal(gen, 3, 4), torch.randint(0, 2000, (3, 4), generator=gen, device="cuda")
    return {
        "qk_norm_rope": (lambda x: ops.qk_norm_rope(x, x, gain, gain, rotary)[0], q),
        "relative_attention": (lambda x: ops.relative_attention(x, x, x, table, plan), q),
        "distill_top_logits": (lambda x: ops.distill_top_logits(x, teacher, index), logits),
    }


@pytest.mark.parametrize("name", ["qk_norm_rope", "relative_attention", "distill_top_logits"])
def test_transforms_do_not_pass_a_kernel_by(name):
    call, x = small_calls()[name]
    for bad in (lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.vmap(call)(x[None]),
                lambda: torch.func.grad(lambda y: call(y).float().sum())(x), lambda: torch.jit.trace(call, x, check_trace=False)):
        with pytest.raises(RuntimeError):
            bad()
    y = x.clone().requires_grad_(True)
    once, = torch.autograd.grad(call(y).float().square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        torch.autograd.grad(once.float().sum(), y)


@pytest.mark.parametrize("name", ["qk_norm_rope", "relative_attention", "distill_top_logits"])
def test_inside_a_compiled_function(name):
    """Kept out of the compiled graph, a call does there what it does elsewhere."""
    call, x = small_calls()[name]
    apart = torch.compiler.disable(call)
    both = [lambda y: call(y * 0.5) + 1.0, torch.compile(lambda y: apart(y * 0.5) + 1.0, backend="eager")]
    results = []
    for f in both:
        y = x.clone().requires_grad_(True)
        out = f(y)
        results.append((out.detach(), *torch.autograd.grad(out, y, torch.ones_like(out))))
    assert all(torch.equal(a, b) for a, b in zip(*results))
