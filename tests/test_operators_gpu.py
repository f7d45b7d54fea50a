"""GPU tests of the operators against their definitions in 64 bits.

Tolerances are bounds, element by element, from the operators' own arithmetic: one rounding of a result is at most
u = finfo(type).eps / 2 relative; P and dS are rounded to the operands' type once before they enter a product; the rest
is float32 with sums of at most a few hundred dependent terms, covered by SLACK = 2^-14 of the sum of absolute terms
(2^-24 per operation, exponentials of arguments up to 2^8 whose own error is 2^-24 of the argument)."""

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from multigpubeamsearch_b200 import operators as ops

pytestmark = pytest.mark.gpu

SLACK = 2.0 ** -14
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float((off / bound.clamp_min(1e-300))[bad].max()))


# ---------------------------------------------------------------------------------------------------------------
# qk_norm_rope
# ---------------------------------------------------------------------------------------------------------------


def qk_reference(x, gain, angle, eps, interleaved):
    """(y, magnitude of the rotated pair) in 64 bits."""
    x, gain = x.double(), gain.double()
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain
    d = x.shape[-1]
    a, b = (n[..., 0::2], n[..., 1::2]) if interleaved else (n[..., :d // 2], n[..., d // 2:])
    c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    y0, y1, m = a * c - b * s, b * c + a * s, torch.sqrt(a * a + b * b)
    join = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if interleaved else (lambda p, q: torch.cat([p, q], -1))
    return join(y0, y1), join(m, m)


def angles(rotary, positions, batch, tokens):
    pos = torch.arange(tokens, device="cuda") if positions is None else positions
    pos = pos.double().expand(batch, tokens) if pos.dim() == 1 else pos.double()
    return pos[..., None] * torch.tensor(rotary.inv_freq, dtype=torch.float64, device="cuda")


QK_CASES = [
    # batch, tokens, heads, key heads, head_dim, type, interleaved, positions, layout
    (1, 1, 1, 1, 32, "bf16", False, None, "packed"),
    (1, 54, 8, 8, 32, "bf16", False, None, "packed"),
    (3, 54, 8, 2, 64, "f16", True, None, "packed"),
    (2, 17, 4, 4, 128, "f32", False, "far", "packed"),
    (5, 33, 6, 3, 80, "bf16", True, "far", "transposed"),
    (2, 65, 3, 1, 256, "f16", False, "token", "packed"),
    (4, 9, 2, 1, 2, "f32", False, "negative", "packed"),
    (4, 9, 2, 2, 6, "bf16", True, "negative", "packed"),
    (3, 31, 5, 1, 96, "f32", True, "far", "shifted"),
    (2, 40, 16, 4, 48, "f16", False, "far", "shifted"),
    (1, 700, 1, 1, 36, "bf16", False, None, "packed"),
    (700, 3, 2, 2, 32, "f32", False, "token", "broadcast"),
    (2, 5, 40, 40, 64, "bf16", False, None, "packed"),
    (0, 4, 2, 2, 32, "bf16", False, None, "packed"),
]


def qk_inputs(case, seed=0):
    b, t, h, hk, d, dtype, inter, where, layout = case
    gen, dt = generator(seed), TYPES[dtype]
    if layout == "packed":
        x = normal(gen, b, t, h + hk, d, dtype=dt)
        q, k = x[:, :, :h], x[:, :, h:]
    elif layout == "transposed":
        q, k = normal(gen, b, h, t, d, dtype=dt).transpose(1, 2), normal(gen, b, hk, t, d, dtype=dt).transpose(1, 2)
    elif layout == "shifted":  # rows that start one element past a 16-byte boundary
        x = normal(gen, b * t * (h + hk) * d + 1, dtype=dt)[1:].view(b, t, h + hk, d)
        q, k = x[:, :, :h], x[:, :, h:]
    else:
        q, k = normal(gen, 1, t, h, d, dtype=dt).expand(b, t, h, d), normal(gen, b, t, hk, d, dtype=dt)
    qg, kg = 1 + 0.2 * normal(gen, d), 1 + 0.2 * normal(gen, d)
    pos = None
    if where == "far":
        pos = torch.randint(0, 1 << 40, (b, t), generator=gen, device="cuda")
    elif where == "token":
        pos = torch.randint(0, 1 << 20, (t,), generator=gen, device="cuda", dtype=torch.int32)
    elif where == "negative":
        pos = torch.randint(-1000, 1000, (b, t), generator=gen, device="cuda", dtype=torch.int32)
    return q, k, qg, kg, pos


def qk_rotary(d):
    # a largest angle below 2^40 * 2^-13 keeps float64's own angle error (2^-53 relative) under 2^-26
    return ops.RotaryFrequencies(d, inv_freq=[2.0 ** -14 / (1 + i) for i in range(d // 2)])


def qk_bound(dtype, ref, mag):
    # 40 float32 roundings (sum of up to 256 squares by lanes and halves, reciprocal root, two products, the angle's sine
    # and cosine, the rotation) relative to the pair's magnitude, then one rounding of the result
    return half_step(dtype) * ref.abs() + 40 * 2.0 ** -24 * mag + 1e-30


@pytest.mark.parametrize("case", QK_CASES, ids=str)
def test_qk_norm_rope_forward(case):
    b, t, h, hk, d, dtype, inter, where, layout = case
    q, k, qg, kg, pos = qk_inputs(case)
    rotary = qk_rotary(d) if where == "far" else ops.RotaryFrequencies(d)
    got = ops.qk_norm_rope(q, k, qg, kg, rotary, positions=pos, eps=1e-5, interleaved=inter)
    ang = angles(rotary, pos, b, t)
    for y, x, g in zip(got, (q, k), (qg, kg)):
        ref, mag = qk_reference(x, g, ang, 1e-5, inter)
        assert y.dtype == x.dtype and y.is_contiguous()
        if x.numel():
            within(y, ref, qk_bound(y.dtype, ref, mag), "y")


@pytest.mark.parametrize("case", QK_CASES, ids=str)
def test_qk_norm_rope_backward(case):
    b, t, h, hk, d, dtype, inter, where, layout = case
    q, k, qg, kg, pos = qk_inputs(case)
    rotary = qk_rotary(d) if where == "far" else ops.RotaryFrequencies(d)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, qg, kg)]
    got_y = ops.qk_norm_rope(*leaves, rotary, positions=pos, eps=1e-5, interleaved=inter)
    gen = generator(9)
    dy = [normal(gen, *y.shape, dtype=y.dtype) for y in got_y]
    got = torch.autograd.grad(got_y, leaves, dy)
    again = torch.autograd.grad(ops.qk_norm_rope(*leaves, rotary, positions=pos, eps=1e-5, interleaved=inter), leaves, dy)
    for x, y in zip(got, again):
        assert torch.equal(x, y)
    ang = angles(rotary, pos, b, t)
    for i in range(2):
        x, gain = leaves[i].detach().double().requires_grad_(True), leaves[2 + i].detach().double().requires_grad_(True)
        y, _ = qk_reference(x, gain, ang, 1e-5, inter)
        dx, dg = torch.autograd.grad(y, (x, gain), dy[i].double())
        assert got[i].dtype == leaves[i].dtype and got[2 + i].dtype == torch.float32
        if not x.numel():
            assert not got[2 + i].any()
            continue
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
        u, mag = qk_reference(torch.ones_like(x), torch.ones_like(gain), ang, 0.0, inter)
        # |u| of a pair is at most the pair's |dy|; dx = r (w - n mean(w n)): terms bounded by r max|g| (|dy| + |n| mean)
        pair = dy[i].double().abs().amax(-1, keepdim=True) * 2
        top = gain.abs().max()
        terms = r * top * (pair + (x * r).abs() * (pair * (x * r).abs()).mean(-1, keepdim=True))
        within(got[i], dx, half_step(got[i].dtype) * dx.abs() + 40 * 2.0 ** -24 * terms + 1e-30, "dx")
        # n dependent additions per lane at most, then the tree
        count = x.shape[0] * x.shape[1] * x.shape[2]
        additions = min(count, 64 + count // 64)
        spread = (pair * (x * r).abs()).sum((0, 1, 2))
        within(got[2 + i], dg, (40 + additions) * 2.0 ** -24 * spread + 1e-30, "dgain")


@pytest.mark.parametrize("d", [48, 80, 96, 112, 144, 160, 176, 192, 208, 224, 240])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_qk_norm_rope_partly_used_lanes(d, dtype):
    """Head sizes of 16-byte pieces that are no power of two: lanes of a head's group that have none of it."""
    for b, t, h, hk, inter, where in ((65, 1, 7, 6, False, "negative"), (1, 203, 19, 3, True, "far"), (9, 54, 8, 8, False, None)):
        case = (b, t, h, hk, d, dtype, inter, where, "packed")
        test_qk_norm_rope_forward(case)
        test_qk_norm_rope_backward(case)


def test_qk_norm_rope_gradient_against_differences():
    q, k, qg, kg, _ = qk_inputs((2, 11, 3, 1, 32, "f32", False, None, "packed"))
    rotary = ops.RotaryFrequencies(32)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, qg, kg)]
    out = ops.qk_norm_rope(*leaves, rotary, eps=1e-5)
    gen = generator(4)
    dy = [normal(gen, *y.shape) for y in out]
    grads = torch.autograd.grad(out, leaves, dy)
    ang = angles(rotary, None, 2, 11)

    def value(xs):
        return sum((qk_reference(xs[i].double(), xs[2 + i].double(), ang, 1e-5, False)[0] * dy[i].double()).sum() for i in range(2))

    for n, (x, g) in enumerate(zip(leaves, grads)):
        v = normal(gen, *x.shape).double()
        plus, minus = list(leaves), list(leaves)
        plus[n], minus[n] = x.detach().double() + 1e-5 * v, x.detach().double() - 1e-5 * v
        want = (value(plus) - value(minus)) / 2e-5
        got = (g.double() * v).sum()
        # differences: third derivatives times 1e-10; float32 gradients: 2^-20 of the terms' sum
        assert abs(got - want) <= 1e-6 * abs(want) + 2.0 ** -18 * (g.double() * v).abs().sum(), (n, float(got), float(want))


def test_qk_norm_rope_zero_rows_and_one_gradient():
    rotary = ops.RotaryFrequencies(32)
    q = torch.zeros(1, 3, 2, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    k = normal(generator(1), 1, 3, 1, 32, dtype=torch.bfloat16).requires_grad_(True)
    g = torch.ones(32, device="cuda")
    q2, k2 = ops.qk_norm_rope(q, k, g, g, rotary, eps=1e-6)
    assert not q2.any()
    q2.sum().backward()  # nothing flows into k2
    assert torch.isfinite(q.grad).all() and not k.grad.any()
    # zeros: dx = dy turned back, over sqrt(eps)
    within(q.grad[0, 0], torch.full((2, 32), 1e3, device="cuda", dtype=torch.float64), torch.full((2, 32), 1e3 * 2.0 ** -8 * 1.01, device="cuda"), "dx")


def test_qk_norm_rope_refuses():
    rotary = ops.RotaryFrequencies(32)
    q, g = torch.zeros(1, 2, 2, 32, device="cuda", dtype=torch.bfloat16), torch.ones(32, device="cuda")
    for bad in (lambda: ops.qk_norm_rope(q, q.float(), g, g, rotary), lambda: ops.qk_norm_rope(q, q[:, :1], g, g, rotary),
                lambda: ops.qk_norm_rope(q, q, g.bfloat16(), g, rotary), lambda: ops.qk_norm_rope(q, q, g[:16], g, rotary),
                lambda: ops.qk_norm_rope(q, q, g, g, ops.RotaryFrequencies(64)), lambda: ops.qk_norm_rope(q, q, g, g, rotary, eps=-1.0),
                lambda: ops.qk_norm_rope(q, q, g, g, rotary, positions=torch.zeros(3, device="cuda", dtype=torch.int64)),
                lambda: ops.qk_norm_rope(q, q, g, g, rotary, positions=torch.zeros(2, device="cuda")),
                lambda: ops.qk_norm_rope(q, q, g, g, rotary, positions=torch.zeros(2, dtype=torch.int64)),
                lambda: ops.qk_norm_rope(q.double(), q.double(), g, g, rotary), lambda: ops.qk_norm_rope(q[0], q[0], g, g, rotary)):
        with pytest.raises(RuntimeError):
            bad()


# ---------------------------------------------------------------------------------------------------------------
# relative_attention
# ---------------------------------------------------------------------------------------------------------------


def attention_reference(q, k, v, table, plan, lengths, scale, dout=None):
    """The definition in 64 bits, with what the bounds need: out, P|v| and, with dout, gradients and error terms."""
    b, t, h, d = q.shape
    share = h // k.shape[2]
    q, k, v = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(share, 1), v.double().transpose(1, 2).repeat_interleave(share, 1)
    off = torch.arange(t, device="cuda")[None] - torch.arange(t, device="cuda")[:, None]
    index = plan.map.long().to("cuda")[off.clamp(-plan.max_distance, plan.max_distance) + plan.max_distance]
    live = torch.ones(b, t, dtype=torch.bool, device="cuda") if lengths is None else torch.arange(t, device="cuda") < lengths[:, None]
    q, k, v = (torch.where(live[:, None, :, None], x, 0.0) for x in (q, k, v))
    seen = live[:, None, :, None] & live[:, None, None, :]
    if plan.causal:
        seen = seen & (off <= 0)
    s = (q @ k.transpose(-1, -2) * scale + table.double()[index].permute(2, 0, 1)).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    r = {"out": back(p @ v), "out_abs": back(p @ v.abs())}
    if dout is not None:
        do = torch.where(live[:, None, :, None], dout.double().transpose(1, 2), 0.0)
        dp = do @ v.transpose(-1, -2)
        delta = (p * dp).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        fold = lambda x: back(x.unflatten(1, (h // share, share)).sum(2))  # noqa: E731
        r.update(dq=back(ds @ k) * scale, dk=fold(ds.transpose(-1, -2) @ q) * scale, dv=fold(p.transpose(-1, -2) @ do))
        pick = torch.nn.functional.one_hot(index.flatten(), plan.num_buckets).double()
        r["dtable"] = torch.einsum("hn,nb->bh", ds.sum(0).flatten(1), pick)
        # error terms: delta from a 16-bit output is off by at most |do| . (error of out)
        terms = do.abs() @ v.abs().transpose(-1, -2)
        r["e_delta"] = (do.abs() * (p @ v.abs())).sum(-1, keepdim=True)
        r["p"], r["ds"], r["terms"], r["q"], r["k"], r["do"], r["pick"], r["fold"], r["back"] = p, ds, terms, q, k, do, pick, fold, back
    return r


def attention_check(q, k, v, table, plan, lengths=None, scale=None, dout=None):
    """Forward and, with dout, backward of one call against the reference, within the derived bounds."""
    u = half_step(q.dtype)
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    ref = attention_reference(q, k, v, table, plan, lengths, sc, dout)
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 1e-30  # spacing of the type's smallest numbers
    if dout is None:
        out = ops.relative_attention(q, k, v, table, plan, lengths=lengths, scale=scale)
        within(out, ref["out"], (2 * u + SLACK) * ref["out_abs"] + tiny, "out")
        return
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, table)]
    out = ops.relative_attention(*leaves, plan, lengths=lengths, scale=scale)
    within(out, ref["out"], (2 * u + SLACK) * ref["out_abs"] + tiny, "out")
    got = torch.autograd.grad(out, leaves, dout)
    # dS = P (dP - delta): float32 terms, delta's error where it comes from the rounded output, one rounding
    ds_err = SLACK * ref["p"] * (ref["terms"] + ref["e_delta"]) + ref["p"] * ref["e_delta"] * (2 * u + SLACK)
    ds_round = ds_err + u * ref["ds"].abs() + (tiny if q.dtype == torch.float16 else 0.0) * (ref["p"] > 0)
    p_round = (u + SLACK) * ref["p"] + (tiny if q.dtype == torch.float16 else 0.0) * (ref["p"] > 0)
    fold, back = ref["fold"], ref["back"]
    within(got[0], ref["dq"], back(ds_round @ ref["k"].abs() + SLACK * (ref["ds"].abs() @ ref["k"].abs())) * sc + u * ref["dq"].abs() + tiny, "dq")
    within(got[1], ref["dk"], fold((ds_round + SLACK * ref["ds"].abs()).transpose(-1, -2) @ ref["q"].abs()) * sc + u * ref["dk"].abs() + tiny, "dk")
    within(got[2], ref["dv"], fold(p_round.transpose(-1, -2) @ ref["do"].abs()) + u * ref["dv"].abs() + tiny, "dv")
    spread = torch.einsum("hn,nb->bh", (ds_err + SLACK * ref["ds"].abs()).sum(0).flatten(1), ref["pick"])
    within(got[3], ref["dtable"], spread + u * ref["dtable"].abs() + tiny, "dtable")
    again = torch.autograd.grad(ops.relative_attention(*leaves, plan, lengths=lengths, scale=scale), leaves, dout)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


ATT_CASES = [
    # batch, tokens, heads, key heads, head_dim, type, causal, lengths, layout
    (1, 1, 1, 1, 32, "bf16", False, False, "packed"),
    (3, 2, 8, 8, 64, "f16", True, True, "packed"),
    (2, 15, 8, 8, 32, "bf16", False, False, "packed"),
    (5, 16, 3, 1, 32, "bf16", True, True, "packed"),
    (7, 17, 8, 8, 64, "bf16", False, True, "transposed"),
    (4, 31, 2, 2, 32, "f16", True, False, "packed"),
    (3, 32, 5, 5, 64, "f16", False, True, "shifted"),
    (4, 33, 8, 4, 32, "bf16", False, False, "packed"),
    (2, 48, 8, 8, 32, "bf16", True, True, "packed"),
    (1, 54, 8, 8, 32, "bf16", False, False, "packed"),
    (600, 54, 8, 8, 32, "bf16", False, False, "packed"),
    (300, 54, 2, 2, 64, "f16", False, True, "packed"),
    (9, 63, 4, 4, 64, "bf16", True, True, "packed"),
    (6, 64, 8, 8, 32, "bf16", False, False, "packed"),
    (6, 64, 8, 2, 64, "f16", True, True, "packed"),
    (3, 65, 8, 8, 32, "bf16", False, False, "packed"),
    (3, 65, 6, 2, 64, "f16", True, True, "transposed"),
    (2, 100, 2, 1, 32, "bf16", True, False, "shifted"),
    (5, 128, 4, 4, 64, "bf16", False, True, "packed"),
    (2, 129, 3, 3, 32, "f16", False, False, "packed"),
    (2, 321, 4, 2, 64, "bf16", True, True, "packed"),
    (1, 640, 2, 2, 32, "bf16", False, True, "packed"),
    (1, 1025, 2, 1, 64, "f16", False, False, "packed"),
    (1200, 70, 1, 1, 32, "bf16", False, True, "packed"),
    (0, 8, 2, 2, 32, "bf16", False, False, "packed"),
]


def attention_inputs(case, seed=0, buckets=32, reach=128):
    b, t, h, hk, d, dtype, causal, ragged, layout = case
    gen, dt = generator(seed), TYPES[dtype]
    if layout == "packed":
        x = normal(gen, b, t, h + 2 * hk, d, dtype=dt)
        q, k, v = x[:, :, :h], x[:, :, h:h + hk], x[:, :, h + hk:]
    elif layout == "transposed":
        q, k, v = (normal(gen, b, n, t, d, dtype=dt).transpose(1, 2) for n in (h, hk, hk))
    else:  # two bytes past a 16-byte boundary
        q, k, v = (normal(gen, b * t * n * d + 1, dtype=dt)[1:].view(b, t, n, d) for n in (h, hk, hk))
    plan = ops.RelativeBuckets(buckets, reach, causal=causal)
    table = normal(gen, buckets, h, dtype=dt)
    lengths = None
    if ragged:
        lengths = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        lengths[0] = t
        if b > 1:
            lengths[-1] = 0
        if b > 2:
            lengths[1] = 1
    return q, k, v, table, plan, lengths, normal(gen, b, t, h, d, dtype=dt)


@pytest.mark.parametrize("case", ATT_CASES, ids=str)
def test_relative_attention_forward(case):
    q, k, v, table, plan, lengths, _ = attention_inputs(case)
    attention_check(q, k, v, table, plan, lengths)


@pytest.mark.parametrize("case", ATT_CASES, ids=str)
def test_relative_attention_backward(case):
    q, k, v, table, plan, lengths, dout = attention_inputs(case, seed=1)
    attention_check(q, k, v, table, plan, lengths, dout=dout)


def test_relative_attention_no_tokens():
    q = torch.zeros(2, 0, 2, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    table = torch.ones(32, 2, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = ops.relative_attention(q, q, q, table, ops.RelativeBuckets())
    dq, dtable = torch.autograd.grad(out, (q, table), torch.zeros_like(out))
    assert out.shape == q.shape and dq.shape == q.shape and not dtable.any()


@pytest.mark.parametrize("tokens", [40, 200])
@pytest.mark.parametrize("buckets,reach", [(4, 2), (8, 5), (64, 200), (512, 1024)])
def test_relative_attention_other_buckets(tokens, buckets, reach):
    case = (3, tokens, 4, 4, 32, "bf16", buckets == 8, True, "packed")
    q, k, v, table, plan, lengths, dout = attention_inputs(case, seed=2, buckets=buckets, reach=reach)
    attention_check(q, k, v, table, plan, lengths, scale=0.5, dout=dout)


@pytest.mark.parametrize("tokens", [20, 150])
def test_relative_attention_never_reads_padding(tokens):
    case = (4, tokens, 2, 2, 32, "bf16", False, True, "packed")
    q, k, v, table, plan, lengths, dout = attention_inputs(case, seed=3)
    results = []
    for fill in (math.nan, math.inf, 0.0):
        xs = [x.clone() for x in (q, k, v, dout)]
        gone = torch.arange(tokens, device="cuda") >= lengths[:, None]
        for x in xs:
            x[gone] = fill
        leaves = [x.requires_grad_(True) for x in xs[:3]] + [table.clone().requires_grad_(True)]
        out = ops.relative_attention(*leaves, plan, lengths=lengths)
        results.append([out] + list(torch.autograd.grad(out, leaves, xs[3])))
    for other in results[:2]:
        assert all(torch.equal(x, y) for x, y in zip(results[2], other))
    assert all(torch.isfinite(x).all() for x in results[2])
    assert not results[2][0][gone].any() and not results[2][1][gone].any() and not results[2][3][gone].any()


@pytest.mark.parametrize("tokens", [30, 130])
def test_relative_attention_lowest_and_empty_biases(tokens):
    """A table at the type's lowest value leaves a plain softmax over equal scores' top; at -inf, no key: zeros."""
    case = (2, tokens, 2, 2, 32, "bf16", False, False, "packed")
    q, k, v, table, plan, _, dout = attention_inputs(case, seed=4)
    lowest = torch.finfo(torch.bfloat16).min
    table = table.clone()
    table[:, 0] = lowest  # all keys alike: the scores vanish beside the bias, P is uniform
    table[:, 1] = -math.inf
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, table)]
    out = ops.relative_attention(*leaves, plan)
    grads = torch.autograd.grad(out, leaves, dout)
    mean = v[:, :, 0].double().mean(1, keepdim=True).expand(-1, tokens, -1)
    spread = v[:, :, 0].double().abs().mean(1, keepdim=True).expand(-1, tokens, -1)
    within(out[:, :, 0], mean, (2 * half_step(torch.bfloat16) + SLACK) * spread, "uniform")
    assert not out[:, :, 1].any()
    assert all(torch.isfinite(g).all() for g in grads)
    assert not grads[0][:, :, 1].any() and not grads[1][:, :, 1].any() and not grads[2][:, :, 1].any() and not grads[3][:, 1].any()
    # some distances closed to a head, the others open
    table = attention_inputs(case, seed=4)[3].clone()
    table[3:9] = -math.inf
    table[20:24] = lowest
    attention_check(q, k, v, table, plan, dout=dout)


def test_relative_attention_many_sequences():
    """More sequences than a grid's second dimension would hold, in both forms."""
    for tokens in (3, 66):
        b = 70001 if tokens == 3 else 66001
        gen = generator(5)
        x = normal(gen, b, tokens, 3, 32, dtype=torch.bfloat16)
        plan = ops.RelativeBuckets()
        table = normal(gen, 32, 1, dtype=torch.bfloat16)
        out = ops.relative_attention(x[:, :, :1], x[:, :, 1:2], x[:, :, 2:], table, plan)
        for part in (slice(0, 50), slice(b - 50, b)):
            y = x[part]
            ref = attention_reference(y[:, :, :1], y[:, :, 1:2], y[:, :, 2:], table, plan, None, 32 ** -0.5)
            within(out[part], ref["out"], (2 * 2.0 ** -8 + SLACK) * ref["out_abs"], "out")


def test_relative_attention_gradient_against_differences():
    """Directional differences of the 64-bit definition against the kernels' gradients."""
    for tokens, hk in ((23, 2), (90, 1)):
        case = (2, tokens, 2, hk, 32, "f16", False, True, "packed")
        q, k, v, table, plan, lengths, dout = attention_inputs(case, seed=6)
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, table)]
        grads = torch.autograd.grad(ops.relative_attention(*leaves, plan, lengths=lengths), leaves, dout)
        gen = generator(7)

        def value(xs):
            return (attention_reference(*xs, plan, lengths, 32 ** -0.5)["out"] * dout.double()).sum()

        for n, g in enumerate(grads):
            v_ = normal(gen, *g.shape).double()
            plus, minus = [x.detach().double() for x in leaves], [x.detach().double() for x in leaves]
            plus[n], minus[n] = plus[n] + 1e-5 * v_, minus[n] - 1e-5 * v_
            want = (value(plus) - value(minus)) / 2e-5
            # every element of a gradient is off by a few roundings of sums of terms no larger than their absolute sum,
            # which for normal inputs is below 2^5 of the largest gradient
            bound = 2.0 ** -11 * 2.0 ** 5 * g.double().abs().max() * v_.norm()
            assert abs((g.double() * v_).sum() - want) <= bound, (tokens, n)


def test_relative_attention_refuses():
    plan = ops.RelativeBuckets()
    q, t = torch.zeros(1, 4, 2, 32, device="cuda", dtype=torch.bfloat16), torch.zeros(32, 2, device="cuda", dtype=torch.bfloat16)
    for bad in (lambda: ops.relative_attention(q.float(), q.float(), q.float(), t.float(), plan), lambda: ops.relative_attention(q, q, q, t.float(), plan),
                lambda: ops.relative_attention(q, q[:, :3], q[:, :3], t, plan), lambda: ops.relative_attention(q, q, q[..., :1, :], t, plan),
                lambda: ops.relative_attention(q[..., :16], q[..., :16], q[..., :16], t, plan), lambda: ops.relative_attention(q, q, q, t[:8], plan),
                lambda: ops.relative_attention(q, q, q, t, plan, scale=0.0), lambda: ops.relative_attention(q, q, q, t, plan, scale=math.nan),
                lambda: ops.relative_attention(q, q, q, t, plan, lengths=torch.ones(2, device="cuda", dtype=torch.int32)),
                lambda: ops.relative_attention(q, q, q, t, plan, lengths=torch.ones(1, device="cuda", dtype=torch.int64)),
                lambda: ops.relative_attention(q, q, q, t, plan, lengths=torch.ones(1, dtype=torch.int32)),
                lambda: ops.relative_attention(q[:, :, :1].expand(1, 4, 3, 32), q, q, t[:, :1].expand(32, 3), plan),
                lambda: ops.relative_attention(q[0], q[0], q[0], t, plan)):
        with pytest.raises(RuntimeError):
            bad()


# ---------------------------------------------------------------------------------------------------------------
# distill_top_logits
# ---------------------------------------------------------------------------------------------------------------


def distill_reference(logits, teacher, index, temperature, weight):
    """Loss and gradient in 64 bits, and the largest |argument| of a row's exponentials."""
    z = logits.double() / temperature
    rows, width = z.shape
    held = (index >= 0) & (index < width)
    t = (teacher.double() / temperature).masked_fill(~held, -math.inf)
    some = (t > -math.inf).any(1, keepdim=True)
    t = torch.where(some, t, 0.0) - torch.where(some, t, 0.0).amax(1, keepdim=True)
    log_p = t - t.exp().sum(1, keepdim=True).log()
    p = torch.where(held & some, log_p.exp(), 0.0)
    log_q = z.log_softmax(1)
    at = torch.where(held, index, 0)
    term = p * (log_p - log_q.gather(1, at.long()))
    loss = torch.where(p > 0, term, 0.0).sum(1)
    target = torch.zeros_like(z).scatter_add_(1, at.long(), p)
    grad = torch.where(some, log_q.exp() - target, 0.0) / temperature * weight[:, None].double()
    return loss, grad, log_q, target, some


def distill_check(logits, teacher, index, temperature, weight):
    loss_ref, grad_ref, log_q, target, some = distill_reference(logits, teacher, index, temperature, weight)
    loss, grad = ops.distill_top_logits_step(logits, teacher, index, temperature=temperature, row_weight=weight)
    assert loss.dtype == torch.float32 and grad.dtype == logits.dtype and grad.shape == logits.shape
    # arguments (z - max) / T carry 3 roundings of themselves; sums of a row's terms at most 2^8 dependent additions
    finite = torch.where(target > 0, -log_q, 0.0).amax(1)
    width_term = (log_q.exp() * -log_q.clamp_min(-1e30)).sum(1) if logits.numel() else loss_ref
    span = (teacher.double().abs().amax(1) / temperature * 2).clamp_max(1e4)
    within(loss, loss_ref, 2.0 ** -24 * (256 + 4 * (finite + width_term + span)) * some[:, 0] + 1e-30, "loss")
    u = half_step(logits.dtype)
    scale = weight[:, None].double() / temperature
    parts = (log_q.exp() * (1 + -log_q.clamp_min(-1e30) / 64) + target * (1 + span[:, None] / 64)) * scale * some
    tiny = 2.0 ** -25 if logits.dtype == torch.float16 else 1e-36
    within(grad, grad_ref, u * grad_ref.abs() + 2.0 ** -24 * 320 * parts + tiny, "grad")
    # the other entry points: the same loss, and the same gradient through autograd
    assert torch.equal(ops.distill_top_logits(logits, teacher, index, temperature=temperature), loss)
    leaf = logits.detach().requires_grad_(True)
    (ops.distill_top_logits(leaf, teacher, index, temperature=temperature) * weight).sum().backward()
    assert torch.equal(leaf.grad, grad)


DISTILL_CASES = [
    # rows, width, entries, type, index type
    (1, 1, 1, "f32", torch.int64),
    (5, 2, 2, "bf16", torch.int64),
    (300, 12, 4, "f32", torch.int64),
    (1000, 24, 24, "bf16", torch.int32),
    (77, 16, 3, "f16", torch.int64),
    (33, 17, 5, "f32", torch.int32),
    (9, 33, 7, "bf16", torch.int64),
    (50, 64, 1, "f16", torch.int64),
    (50, 65, 40, "f32", torch.int64),
    (31, 128, 8, "bf16", torch.int64),
    (31, 129, 8, "bf16", torch.int64),
    (17, 256, 300, "f16", torch.int64),
    (17, 257, 9, "f32", torch.int64),
    (6, 1000, 100, "bf16", torch.int64),
    (6, 1024, 1024, "f32", torch.int64),
    (6, 1025, 64, "bf16", torch.int64),
    (200, 4097, 8, "f32", torch.int32),
    (3, 8191, 64, "f16", torch.int64),
    (200, 20011, 50, "bf16", torch.int64),
    (180, 40001, 33, "bf16", torch.int64),
    (2, 50021, 1024, "f32", torch.int64),
    (1, 131072, 32, "f16", torch.int64),
    (160, 131072, 16, "f32", torch.int64),
    (2, 300007, 16, "f32", torch.int64),
    (0, 12, 4, "f32", torch.int64),
]


def distill_inputs(case, seed=0):
    rows, width, entries, dtype, itype = case
    gen = generator(seed)
    logits = normal(gen, rows, width, dtype=TYPES[dtype], scale=3.0)
    teacher = normal(gen, rows, entries, scale=2.0)
    index = torch.randint(0, width, (rows, entries), generator=gen, device="cuda").to(itype)  # doubles among them
    return logits, teacher, index, torch.rand((rows,), generator=gen, device="cuda") + 0.1


@pytest.mark.parametrize("case", DISTILL_CASES, ids=str)
def test_distill(case):
    distill_check(*distill_inputs(case)[:3], 1.5, distill_inputs(case)[3])


@pytest.mark.parametrize("width", [12, 700, 3001])
def test_distill_padding_and_empty_rows(width):
    logits, teacher, index, weight = distill_inputs((40, width, 6, "bf16", torch.int64), seed=1)
    index[:, 4:] = -1
    index[3] = -7
    index[4] = width
    index[5] = 1 << 40
    index[6] = 2  # one column six times
    teacher[7] = -math.inf
    teacher[8, :3] = -math.inf
    teacher[9] = torch.finfo(torch.float32).min
    distill_check(logits, teacher, index, 2.0, weight)
    loss, grad = ops.distill_top_logits_step(logits, teacher, index, temperature=2.0)
    for row in (3, 4, 5, 7):
        assert loss[row] == 0 and not grad[row].any()


@pytest.mark.parametrize("width", [12, 700, 3001])
@pytest.mark.parametrize("fill", [-math.inf, "lowest"])
def test_distill_closed_columns(width, fill):
    """Columns that the student may not choose, at -inf or at the type's lowest value, with and without the teacher's
    entries among them; and rows that are closed altogether."""
    logits, teacher, index, weight = distill_inputs((8, width, 3, "f32", torch.int64), seed=2)
    fill = torch.finfo(torch.float32).min if fill == "lowest" else fill
    index[:, :] = torch.tensor([1, 3, 5], device="cuda")
    logits[:, 6:] = fill
    logits[:, 0] = fill
    distill_check(logits, teacher, index, 1.0, weight)
    logits[1, 3] = -math.inf  # the teacher wants what the student cannot give
    loss, grad = ops.distill_top_logits_step(logits, teacher, index)
    assert loss[1] == math.inf and torch.isfinite(loss[[0, 2, 3, 4, 5, 6, 7]]).all() and torch.isfinite(grad).all()
    logits[2] = fill
    loss, grad = ops.distill_top_logits_step(logits, teacher, index)
    if fill == -math.inf:
        assert loss[2].isnan() and grad[2].isnan().all()
    else:  # equal logits: uniform
        want = (teacher[2].double().softmax(0) * teacher[2].double().log_softmax(0)).sum() + math.log(width)
        assert abs(loss[2].double() - want) < 1e-4
    logits[4, 2] = math.nan
    loss, grad = ops.distill_top_logits_step(logits, teacher, index)
    assert loss[4].isnan() and grad[4].isnan().all() and loss[3].isfinite()


def test_distill_strides_and_types():
    gen = generator(3)
    wide = normal(gen, 20, 5000, dtype=torch.bfloat16)
    for logits in (wide[:, 3:2503], wide[:, 1:1500], wide[::2, :2048], wide[:, 5:17], wide.t()[:20, :20]):
        rows, width = logits.shape
        teacher = normal(gen, rows, 12)[:, ::2]
        index = torch.randint(0, width, (rows, 12), generator=gen, device="cuda")[:, 1::2]
        distill_check(logits, teacher, index, 1.0, torch.ones(rows, device="cuda"))
    teacher, index = normal(gen, 20, 4, dtype=torch.bfloat16), torch.randint(0, 5000, (20, 4), generator=gen, device="cuda")
    assert torch.equal(ops.distill_top_logits(wide, teacher, index), ops.distill_top_logits(wide, teacher.float(), index))


def test_distill_gradient_against_differences():
    logits, teacher, index, weight = distill_inputs((6, 40, 5, "f32", torch.int64), seed=4)
    _, grad = ops.distill_top_logits_step(logits, teacher, index, temperature=1.5, row_weight=weight)
    v = normal(generator(5), 6, 40).double()
    value = lambda z: (distill_reference(z, teacher, index, 1.5, weight)[0] * weight.double()).sum()  # noqa: E731
    want = (value(logits.double() + 1e-5 * v) - value(logits.double() - 1e-5 * v)) / 2e-5
    assert abs((grad.double() * v).sum() - want) <= 2.0 ** -16 * (grad.double() * v).abs().sum() + 1e-8


def test_distill_refuses():
    z, t, i = torch.zeros(3, 5, device="cuda"), torch.zeros(3, 2, device="cuda"), torch.zeros(3, 2, device="cuda", dtype=torch.int64)
    for bad in (lambda: ops.distill_top_logits(z.double(), t, i), lambda: ops.distill_top_logits(z[0], t, i), lambda: ops.distill_top_logits(z, t[:2], i[:2]),
                lambda: ops.distill_top_logits(z, t, i[:, :1]), lambda: ops.distill_top_logits(z, t, i.float()), lambda: ops.distill_top_logits(z, t, i.cpu()),
                lambda: ops.distill_top_logits(z, t, i, temperature=0.0), lambda: ops.distill_top_logits(z, t[:, :0], i[:, :0]),
                lambda: ops.distill_top_logits(z, torch.zeros(3, 1025, device="cuda"), torch.zeros(3, 1025, device="cuda", dtype=torch.int64)),
                lambda: ops.distill_top_logits_step(z, t, i, row_weight=torch.ones(2, device="cuda")),
                lambda: ops.distill_top_logits_step(z, t, i, row_weight=torch.ones(3, device="cuda", dtype=torch.float64))):
        with pytest.raises(RuntimeError):
            bad()


# ---------------------------------------------------------------------------------------------------------------
# Streams, graphs, several calls
# ---------------------------------------------------------------------------------------------------------------


def everything(seed, tokens=54):
    """Forward and backward of all three as one layer would run them; results as a list."""
    gen = generator(seed)
    x = normal(gen, 4, tokens, 24, 32, dtype=torch.bfloat16)
    q, k, v = (x[:, :, 8 * n:8 * n + 8].detach().requires_grad_(True) for n in range(3))
    gain = torch.ones(32, device="cuda", requires_grad=True)
    table = normal(gen, 32, 8, dtype=torch.bfloat16).requires_grad_(True)
    dout = normal(gen, 4, tokens, 8, 32, dtype=torch.bfloat16)
    teacher, index = normal(gen, 4, 3), torch.randint(0, 256 * tokens, (4, 3), generator=gen, device="cuda")
    return (q, k, v, gain, table), dout, teacher, index


def run_everything(leaves, dout, teacher, index, rotary, plan):
    q, k, v, gain, table = leaves
    q2, k2 = ops.qk_norm_rope(q, k, gain, gain, rotary)
    out = ops.relative_attention(q2, k2, v, table, plan)
    loss = ops.distill_top_logits(out.flatten(1), teacher, index)
    grads = torch.autograd.grad([out, loss], leaves, [dout, torch.ones_like(loss)])
    return [out, loss, *grads]


@pytest.mark.parametrize("tokens", [54, 100])
def test_side_stream_and_interleaved_calls(tokens):
    rotary, plan = ops.RotaryFrequencies(32), ops.RelativeBuckets()
    sets = [everything(s, tokens) for s in range(4)]
    want = [[t.clone() for t in run_everything(*s, rotary, plan)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None] * len(sets)
    for _ in range(5):
        for n, st in enumerate(streams):  # in flight together, each with its own workspaces
            with torch.cuda.stream(st):
                got[n] = run_everything(*sets[n], rotary, plan)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("tokens", [54, 100])
def test_captured_and_replayed(tokens):
    """Two graphs of forward and backward, replayed in turn on new inputs, against eager calls."""
    rotary, plan = ops.RotaryFrequencies(32), ops.RelativeBuckets()
    sets = [everything(s, tokens) for s in (10, 11)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            run_everything(*s, rotary, plan)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run_everything(*s, rotary, plan))
        graphs.append(g)
    for trial in range(3):
        fresh = [everything(20 + 2 * trial + n, tokens) for n in range(2)]
        with torch.no_grad():
            for held, new in zip(sets, fresh):
                for x, y in zip((*held[0], *held[1:]), (*new[0], *new[1:])):
                    x.copy_(y)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for new, out in zip(fresh, outs):
            want = run_everything(*new, rotary, plan)
            assert all(torch.equal(x, y) for x, y in zip(want, out))


# ---------------------------------------------------------------------------------------------------------------
# Long sequences: layouts, shared heads, references that have to follow, padding
# ---------------------------------------------------------------------------------------------------------------

LONG_CASES = [
    (2, 66, 3, 3, 64, "bf16", False, True, "packed"),
    (3, 127, 6, 2, 64, "f16", True, False, "shifted"),
    (2, 130, 6, 1, 64, "bf16", False, True, "transposed"),
    (1, 200, 12, 1, 64, "f16", True, True, "transposed"),
    (1, 150, 7, 1, 32, "bf16", True, False, "packed"),
    (1, 150, 11, 1, 32, "bf16", False, True, "packed"),
    (1, 150, 16, 1, 32, "f16", True, False, "packed"),
    (70, 130, 2, 2, 64, "bf16", True, True, "packed"),
    (2, 330, 9, 3, 32, "bf16", True, True, "transposed"),
    (3, 385, 2, 2, 32, "f16", False, True, "shifted"),
    (2, 449, 2, 2, 32, "bf16", False, False, "packed"),
]


@pytest.mark.parametrize("case", LONG_CASES, ids=str)
def test_long_attention(case):
    q, k, v, table, plan, lengths, dout = attention_inputs(case, seed=30)
    attention_check(q, k, v, table, plan, lengths, dout=dout)
    assert plan.error_code() == 0


@pytest.mark.parametrize("tokens,d", [(20, 32), (150, 64), (330, 32)])
def test_relative_attention_broadcast_inputs(tokens, d):
    """Sequences, tokens and heads that share memory: strides of 0, and each reader's own gradient."""
    gen, plan = generator(31), ops.RelativeBuckets()
    table, dout = normal(gen, 32, 4, dtype=torch.bfloat16), normal(gen, 3, tokens, 4, d, dtype=torch.bfloat16)
    q = normal(gen, 1, tokens, 4, d, dtype=torch.bfloat16).expand(3, -1, -1, -1)
    k = normal(gen, 3, tokens, 1, d, dtype=torch.bfloat16).expand(-1, -1, 4, -1)
    v = normal(gen, 3, 1, 4, d, dtype=torch.bfloat16).expand(-1, tokens, -1, -1)
    attention_check(q, k, v, table, plan, dout=dout)
    whole = [x[:1].clone() for x in (q, k, v)]
    base = [x.requires_grad_(True) for x in whole]
    out = ops.relative_attention(*(x.expand(3, -1, -1, -1) for x in base), table, plan)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
    grads = torch.autograd.grad(out, base, dout[:1].expand(3, -1, -1, -1))
    # the same call with a gradient per reader: strides decide between two forms, whose float32 sums differ
    each = [x.detach().expand(3, -1, -1, -1).requires_grad_(True) for x in base]
    per = torch.autograd.grad(ops.relative_attention(*each, table, plan), each, dout[:1].expand(3, -1, -1, -1))
    for three, one in zip(grads, per):  # three equal 16-bit gradients: two roundings of their sum
        one = one[:1].double()
        within(three, 3 * one, 2 * half_step(torch.bfloat16) * 3 * one.abs(), "sum over the readers")


@pytest.mark.parametrize("tokens,d", [(300, 64), (700, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("way", ["rising", "falling", "leap"])
def test_long_attention_scores_that_grow(tokens, d, dtype, way):
    """Rows whose largest score comes late, early, or in one leap far beyond all before."""
    q, k, v, table, plan, _, dout = attention_inputs((2, tokens, 2, 2, d, dtype, False, False, "packed"), seed=32)
    grow = torch.linspace(0.05, 6.0, tokens, device="cuda")
    if way == "leap":
        grow = torch.where(torch.arange(tokens, device="cuda") == tokens - 9, 10.0, 0.2)
    k = (k.float() * (grow.flip(0) if way == "falling" else grow)[:, None, None]).to(k.dtype)
    ref = attention_reference(q, k, v, table, plan, None, d ** -0.5)
    out = ops.relative_attention(q, k, v, table, plan)
    u = half_step(k.dtype)
    # P is relative to a reference that some key reaches, so the sum is at least 1, and P below the type's smallest
    # normal number is off by half its spacing at most
    small = 2.0 ** -25 * v.double().abs().sum(1, keepdim=True) if dtype == "f16" else 0.0
    within(out, ref["out"], (2 * u + SLACK) * ref["out_abs"] + small + 2.0 ** -24, "out")
    if dtype == "bf16":
        attention_check(q, k, v, table, plan, dout=dout)


@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("at", [400, 401, 403, 405, 406, 407, 408, 414, 415])
def test_long_attention_one_key_beyond_all_range(d, at):
    """One key whose scores leave float32's exponents against the rows' references, and one that is NaN, at the places of
    a tile that take different ways to their exponential."""
    q, k, v, table, _, _, _ = attention_inputs((1, 700, 2, 2, d, "bf16", False, False, "packed"), seed=60)
    plan = ops.RelativeBuckets(32, 20)  # most tiles lie beyond the reach
    k, q = k.clone(), q.clone()
    q[:, torch.arange(700, device="cuda") % 32 != 5] = 0  # one row in 32, so that no neighbour notices for it
    keep = k[:, at].clone()
    k[:, at] *= 100
    ref = attention_reference(q, k, v, table, plan, None, d ** -0.5)
    # arguments of 2^9: twice the slack
    within(ops.relative_attention(q, k, v, table, plan), ref["out"], (2 * half_step(k.dtype) + 2 * SLACK) * ref["out_abs"] + 1e-30, "out")
    k[:, at] = keep
    k[:, at, :, 3] = math.nan
    assert ops.relative_attention(q, k, v, table, plan).isnan().all()


@pytest.mark.parametrize("tokens,d", [(321, 64), (700, 32), (130, 32)])
@pytest.mark.parametrize("open_", ["near", "far before", "far after", "tall"])
def test_long_attention_closed_distances(tokens, d, open_):
    """Tiles in which every bias is -inf, rows that see their first key late or none, a bias far above the scores."""
    q, k, v, table, plan, lengths, dout = attention_inputs((3, tokens, 2, 2, d, "bf16", False, True, "packed"), seed=33)
    table = table.clone()
    before, after = int(plan.map[0]), int(plan.map[-1])
    if open_ == "near":
        table[before] = table[after] = -math.inf
    elif open_ == "tall":
        table[after] = 80.0
    else:
        keep = before if open_ == "far before" else after
        table[torch.arange(32, device="cuda") != keep] = -math.inf
    attention_check(q, k, v, table, plan, lengths, dout=dout)


@pytest.mark.parametrize("tokens,d,shared", [(150, 64, 1), (150, 64, 3), (400, 32, 1)])
def test_long_attention_never_reads_padding(tokens, d, shared):
    q, k, v, table, plan, lengths, dout = attention_inputs((4, tokens, 3, 3 // shared, d, "bf16", False, True, "packed"), seed=34)
    gone = torch.arange(tokens, device="cuda") >= lengths[:, None]
    results = []
    for fill in (math.nan, math.inf, 0.0):
        xs = [x.clone() for x in (q, k, v, dout)]
        for x in xs:
            x[gone] = fill
        leaves = [x.requires_grad_(True) for x in xs[:3]] + [table.clone().requires_grad_(True)]
        out = ops.relative_attention(*leaves, plan, lengths=lengths)
        results.append([out] + list(torch.autograd.grad(out, leaves, xs[3])))
    for other in results[:2]:
        assert all(torch.equal(x, y) for x, y in zip(results[2], other))
    assert all(torch.isfinite(x).all() for x in results[2])
    assert not any(x[gone].any() for x in results[2][:4])


@pytest.mark.parametrize("tokens,d", [(20, 32), (100, 32), (100, 64)])
def test_relative_attention_length_out_of_range(tokens, d):
    """Lengths below 0 count as 0 and lengths above the tokens as all of them."""
    q, k, v, table, plan, _, _ = attention_inputs((3, tokens, 2, 2, d, "bf16", True, False, "packed"), seed=35)
    lengths = torch.tensor([-5, tokens + 7, 9], device="cuda", dtype=torch.int32)
    held = torch.tensor([0, tokens, 9], device="cuda", dtype=torch.int32)
    assert torch.equal(ops.relative_attention(q, k, v, table, plan, lengths=lengths), ops.relative_attention(q, k, v, table, plan, lengths=held))


@pytest.mark.parametrize("tokens,d", [(20, 32), (100, 64), (100, 32)])
def test_relative_attention_offsets_past_32_bits(tokens, d):
    """Sequences that lie 2^31 elements apart."""
    gen, apart = generator(36), (1 << 31) + 64
    room = torch.empty(apart + tokens * 6 * d, dtype=torch.bfloat16, device="cuda")
    x = room.as_strided((2, tokens, 6, d), (apart, 6 * d, d, 1))
    x.copy_(normal(gen, 2, tokens, 6, d, dtype=torch.bfloat16))
    table, plan = normal(gen, 32, 2, dtype=torch.bfloat16), ops.RelativeBuckets()
    near, leaves = x.clone(), []
    for y in (x, near):
        leaves.append([y[:, :, 2 * n:2 * n + 2].detach().requires_grad_(True) for n in range(3)])
    dout = normal(gen, 2, tokens, 2, d, dtype=torch.bfloat16)
    outs = [ops.relative_attention(*y, table, plan) for y in leaves]
    assert torch.equal(outs[0], outs[1])
    far_dout = torch.empty(apart + tokens * 2 * d, dtype=torch.bfloat16, device="cuda").as_strided((2, tokens, 2, d), (apart, 2 * d, d, 1))
    far_dout.copy_(dout)
    for a, b in zip(torch.autograd.grad(outs[0], leaves[0], far_dout), torch.autograd.grad(outs[1], leaves[1], dout)):
        assert torch.equal(a, b)


def test_qk_norm_rope_offsets_past_32_bits():
    gen, apart = generator(37), (1 << 31) + 64
    x = torch.empty(apart + 30 * 64, dtype=torch.bfloat16, device="cuda").as_strided((2, 10, 3, 64), (apart, 192, 64, 1))
    x.copy_(normal(gen, 2, 10, 3, 64, dtype=torch.bfloat16))
    gain, rotary = torch.rand(64, generator=gen, device="cuda"), ops.RotaryFrequencies(64)
    far, near = (ops.qk_norm_rope(y[:, :, :2], y[:, :, 2:], gain, gain, rotary) for y in (x, x.clone()))
    assert torch.equal(far[0], near[0]) and torch.equal(far[1], near[1])


def test_distill_offsets_past_32_bits():
    """More logits than 32 bits count, in rows that a few blocks hold and in rows that a few lanes hold."""
    gen = generator(38)
    for rows, width in ((17000, 131072), (9000000, 240)):
        logits = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
        part = [slice(0, 20), slice(rows - 20, rows)]
        logits.zero_()
        for p in part:
            logits[p] = normal(gen, 20, width, dtype=torch.bfloat16)
        teacher, index = normal(gen, rows, 2), torch.randint(0, width, (rows, 2), generator=gen, device="cuda")
        loss, grad = ops.distill_top_logits_step(logits, teacher, index)
        for p in part:
            one, some = ops.distill_top_logits_step(logits[p].clone(), teacher[p], index[p])
            assert torch.equal(loss[p], one) and torch.equal(grad[p], some)
        del logits, loss, grad


def test_second_derivatives_are_refused():
    """With a graph of the gradient the first derivative is the same and the second raises."""
    gen = generator(39)
    x = [normal(gen, 2, 10, 2, 32, dtype=torch.bfloat16).requires_grad_(True) for _ in range(3)]
    table, gain = normal(gen, 32, 2, dtype=torch.bfloat16).requires_grad_(True), torch.ones(32, device="cuda", requires_grad=True)
    z, index = normal(gen, 5, 20).requires_grad_(True), torch.zeros(5, 2, device="cuda", dtype=torch.int64)
    plan, rotary = ops.RelativeBuckets(), ops.RotaryFrequencies(32)
    for value, leaf in ((lambda: ops.relative_attention(*x, table, plan).float().square().sum(), x[0]),
                        (lambda: ops.qk_norm_rope(x[0], x[1], gain, gain, rotary)[0].float().square().sum(), x[0]),
                        (lambda: ops.distill_top_logits(z, torch.ones(5, 2, device="cuda"), index).sum(), z)):
        plain, = torch.autograd.grad(value(), leaf)
        grad, = torch.autograd.grad(value(), leaf, create_graph=True)
        assert torch.equal(plain, grad)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grad.float().sum(), leaf)


def long_step(seed):
    gen = generator(seed)
    x = normal(gen, 2, 200, 8, 64, dtype=torch.bfloat16)
    leaves = [y.detach().requires_grad_(True) for y in (x[:, :, :6], x[:, :, 6:7], x[:, :, 7:])] + [normal(gen, 32, 6, dtype=torch.bfloat16).requires_grad_(True)]
    return leaves, normal(gen, 2, 200, 6, 64, dtype=torch.bfloat16), torch.tensor([200, 133], device="cuda", dtype=torch.int32)


def run_long_step(leaves, dout, lengths, plan):
    out = ops.relative_attention(*leaves, plan, lengths=lengths)
    return [out, *torch.autograd.grad(out, leaves, dout)]


def test_long_attention_on_streams_and_replayed():
    plan = ops.RelativeBuckets(causal=True)
    sets = [long_step(s) for s in range(40, 44)]
    want = [[t.detach().clone() for t in run_long_step(*s, plan)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None] * len(sets)
    for _ in range(5):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[n] = run_long_step(*sets[n], plan)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    del got, b  # a backward pass is captured only while no eager graph of its leaves lives
    graphs, outs = [], []
    for s in sets[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run_long_step(*s, plan))
        graphs.append(g)
    with torch.no_grad():
        for held, new in zip(sets[:2], sets[2:]):
            for x, y in zip((*held[0], *held[1:]), (*new[0], *new[1:])):
                x.copy_(y)
    for st, g in zip(streams, graphs):  # both in flight
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want[2:], outs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_long_attention_first_in_a_process():
    """Forward and backward as a process's first calls, the backward on autograd's thread, for which torch's allocator has
    memory at hand, so that this is its first call of the runtime; then on threads of its own."""
    code = """
import threading, torch
from multigpubeamsearch_b200 import operators as ops
leaves = [torch.randn(*s, device="cuda", dtype=torch.bfloat16).requires_grad_(True) for s in [(2, 200, 1, 64)] * 3 + [(32, 1)]]
plan, ones = ops.RelativeBuckets(device="cuda"), torch.ones(2, 200, 1, 64, device="cuda", dtype=torch.bfloat16)
room = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (1 << 26, 1 << 20, 1 << 20, 1 << 19, 1 << 19)]
del room
step = lambda: torch.autograd.grad(ops.relative_attention(*leaves, plan), leaves, ones)[0]
first, later = step(), []
threads = [threading.Thread(target=lambda: later.append(step())) for _ in range(3)]
[n.start() for n in threads]; [n.join() for n in threads]
torch.cuda.synchronize()
assert len(later) == 3 and first.isfinite().all() and all(torch.equal(first, y) for y in later)
"""
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=240)
    assert done.returncode == 0, done.stderr[-2000:]


def test_distill_wide_on_streams_and_replayed():
    sets = [distill_inputs((40, 50021, 33, "bf16", torch.int64), seed=s) for s in range(50, 54)]
    run = lambda s: ops.distill_top_logits_step(*s[:3], temperature=1.5, row_weight=s[3])  # noqa: E731
    want = [[t.clone() for t in run(s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None] * len(sets)
    for _ in range(5):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[n] = run(sets[n])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(sets[0])
    for x, y in zip(sets[0], sets[1]):
        x.copy_(y)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[1][0]) and torch.equal(out[1], want[1][1])


@pytest.mark.parametrize("width", [50021, 131072, 300007])
@pytest.mark.parametrize("fill", [-math.inf, "lowest", 1e4])
def test_distill_wide_closed_columns(width, fill):
    """Rows that several blocks hold: closed columns, one entry far above the rest, rows closed altogether."""
    logits, teacher, index, weight = distill_inputs((4, width, 5, "f32", torch.int64), seed=55)
    index[:] = torch.tensor([0, 7, width // 2, width - 2, width - 1], device="cuda")
    if fill == 1e4:
        logits[:, width // 3] = fill
        distill_check(logits[:, :], teacher, index, 1.0, weight)
        return
    fill = torch.finfo(torch.float32).min if fill == "lowest" else fill
    hide = torch.ones(width, dtype=torch.bool, device="cuda")
    hide[index[0]] = False
    hide[100:200] = False
    logits[:, hide] = fill
    distill_check(logits, teacher, index, 1.0, weight)
    logits[2] = fill
    loss, grad = ops.distill_top_logits_step(logits, teacher, index)
    assert loss[[0, 1, 3]].isfinite().all() and grad[[0, 1, 3]].isfinite().all()
    if fill == -math.inf:
        assert loss[2].isnan() and grad[2].isnan().all()
    else:
        want = (teacher[2].double().softmax(0) * teacher[2].double().log_softmax(0)).sum() + math.log(width)
        assert abs(loss[2].double() - want) < 1e-4
