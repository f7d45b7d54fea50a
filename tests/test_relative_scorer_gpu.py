"""GPU tests of the operators where the framework calls them: the transformer scorer with relative positions, its
trainable form, and the distillation of an action scorer."""

import numpy as np
import pytest
import torch

from oracle import beam_oracle as bo
from multigpubeamsearch_b200 import operators as ops
from multigpubeamsearch_b200 import puzzles, scorers

pytestmark = pytest.mark.gpu


def states(count, seed):
    pz = puzzles.puzzle54()
    rng = np.random.default_rng(seed)
    g = pz.generators.astype(np.int64)
    rows = np.tile(pz.solved, (count, 1))
    for _ in range(30):
        rows = np.take_along_axis(rows, g[rng.integers(0, pz.fanout, size=count)], axis=1)
    out = np.zeros((count, 64), np.uint8)
    out[:, :54] = rows
    return out


def weights(norm, bias, base=10000.0, model=0):
    rng = np.random.default_rng(31 + model)
    w = puzzles.transformer_weights(54, 6, layers=2, model_idx=model)
    w["b_head"] = np.float32(0.05)
    w["rotary_base"] = base
    for L in w["layers"]:
        if norm:
            L["q_gain"], L["k_gain"] = ((1 + 0.2 * rng.standard_normal(32)).astype(np.float32) for _ in range(2))
        if bias:  # on the bfloat16 grid, as the scorer holds it
            L["rel_table"] = torch.from_numpy(rng.standard_normal((32, 8)).astype(np.float32)).bfloat16().float().numpy()
    return w


@pytest.mark.parametrize("norm,bias,base,dtype", [(True, True, 10000.0, "bf16"), (True, False, 100.0, "bf16"), (False, True, None, "bf16"),
                                                  (True, True, None, "bf16"), (True, False, 10000.0, "fp8")])
@pytest.mark.parametrize("count,micro", [(300, 32768), (257, 64)])
def test_scorer_with_relative_positions(norm, bias, base, dtype, count, micro):
    ws = [weights(norm, bias, base, model=i) for i in range(2)]
    sc = scorers.TransformerValueScorer(ws, 54, 64, 6, max_rows=count, micro_batch=micro, dtype=dtype)
    rows = states(count, seed=count)
    sc.score(torch.from_numpy(rows).cuda())
    torch.cuda.synchronize()
    assert sc.error_code() == 0
    q = (sc.last_q(count).cpu().numpy() + 0.1) / 2
    # the scorer's stated bounds: bf16 1e-2, e4m3 operands 2e-2 on this initialisation
    err = np.abs(q - bo.transformer_forward(rows[:, :54], ws)).max()
    assert err <= (2e-2 if dtype == "fp8" else 1e-2), err
    # and they do something: without them the values are others
    plain = [dict(w, layers=[{k: v for k, v in L.items() if k not in ("q_gain", "k_gain", "rel_table")} for L in w["layers"]]) for w in ws]
    assert np.abs(bo.transformer_forward(rows[:, :54], plain) - bo.transformer_forward(rows[:, :54], ws)).max() > 1.5e-2


def test_scorer_leaves_rows_behind_the_count_alone():
    """Fewer states than the micro-batch: activation rows behind the last state keep what they held."""
    sc = scorers.TransformerValueScorer(weights(True, True), 54, 64, 6, max_rows=128, micro_batch=128)
    sc.att.fill_(7.0)
    sc.score(torch.from_numpy(states(33, 1)).cuda())
    torch.cuda.synchronize()
    assert (sc.att[33 * 54: 34 * 54 - 1] == 7.0).all() and not (sc.att[:33 * 54] == 7.0).all(1).any()


def test_scorer_refuses():
    w = weights(True, True)
    with pytest.raises(RuntimeError, match="fp8"):
        scorers.TransformerValueScorer(w, 54, 64, 6, max_rows=8, dtype="fp8")
    for change in (lambda L: L.pop("q_gain"), lambda L: L.update(k_gain=np.ones(16, np.float32)), lambda L: L.update(rel_table=np.zeros((16, 8), np.float32))):
        w = weights(True, True)
        change(w["layers"][1])
        with pytest.raises(RuntimeError):
            scorers.TransformerValueScorer(w, 54, 64, 6, max_rows=8)
    with pytest.raises(RuntimeError, match="share"):
        scorers.TransformerValueScorer([weights(True, True), dict(weights(True, True), qk_eps=1e-3)], 54, 64, 6, max_rows=8)


def plain_net(net, rows):
    """TransformerValueNet in float32 torch operations on the same parameters."""
    F = torch.nn.functional
    s = rows[:, :54].long()
    x = net.tok_emb[s] + net.pos_emb
    b, t, d = x.shape
    freq = net.rotary_base ** (-torch.arange(16, device=x.device) / 16.0)
    ang = torch.arange(t, device=x.device)[:, None] * freq
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    index = torch.tensor([[ops.relative_bucket(j - i, *net.rel_buckets, False) for j in range(t)] for i in range(t)], device=x.device)

    def turn(y, gain):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + net.EPS) * gain
        p, q = y[..., :16], y[..., 16:]
        return torch.cat([p * cos - q * sin, q * cos + p * sin], -1)

    for L in net.layers:
        qkv = F.linear(F.layer_norm(x, (d,), L.ln1_g, L.ln1_b), L.wqkv, L.bqkv).view(b, t, 3, 8, 32)
        q, k, v = turn(qkv[:, :, 0], L.q_gain), turn(qkv[:, :, 1], L.k_gain), qkv[:, :, 2]
        p = (torch.einsum("bihd,bjhd->bhij", q, k) / 32 ** 0.5 + L.rel_table[index].permute(2, 0, 1)).softmax(-1)
        x = x + F.linear(torch.einsum("bhij,bjhd->bihd", p, v).reshape(b, t, d), L.wo, L.bo)
        x = x + F.linear(F.gelu(F.linear(F.layer_norm(x, (d,), L.ln2_g, L.ln2_b), L.w1, L.b1)), L.w2, L.b2)
    return F.layer_norm(x, (d,), net.lnf_g, net.lnf_b).mean(1) @ net.w_head + net.b_head


def test_trainable_net_gradients_and_export():
    """Values and every parameter's gradient against float32 torch, and the exported weights in the scorer."""
    torch.manual_seed(3)
    net = scorers.TransformerValueNet(54, 6, layers=2, ffn=512).cuda()
    with torch.no_grad():
        for L in net.layers:
            L.rel_table.normal_(0, 1)
            L.rel_table.copy_(L.rel_table.bfloat16().float())
            L.q_gain.normal_(1, 0.2)
            L.k_gain.normal_(1, 0.2)
            for n in ("wqkv", "wo", "w1", "w2"):
                getattr(L, n).mul_(3.0)
    rows = torch.from_numpy(states(64, 5)).cuda()
    want_dir = torch.randn(64, device="cuda")
    y = net(rows)
    grads = torch.autograd.grad(y @ want_dir, list(net.parameters()))
    y_ref = plain_net(net, rows)
    refs = torch.autograd.grad(y_ref @ want_dir, list(net.parameters()))
    # relative, 2-norm: each layer rounds some ten times to bfloat16 (2^-8 at most each) on the way there and back
    bound = 2 * 2 * 10 * 2.0 ** -8
    assert (y - y_ref).norm() <= bound * y_ref.norm()
    for (name, _), g, r in zip(net.named_parameters(), grads, refs):
        assert (g - r).norm() <= bound * r.norm() + 1e-6, (name, float((g - r).norm()), float(r.norm()))
    sc = scorers.TransformerValueScorer(net.encoder_weights(), 54, 64, 6, max_rows=64)
    sc.score(rows)
    torch.cuda.synchronize()
    q = sc.last_q(64) + net.b_head.detach()
    assert (q - y_ref.detach()).abs().max() <= 1e-2 + bound * y_ref.detach().abs().max()


def test_trainable_net_step_runs():
    net = scorers.TransformerValueNet(54, 6, layers=1, ffn=256, rotary_base=None).cuda()
    opt = torch.optim.SGD(net.parameters(), lr=1e-2)
    rows = torch.from_numpy(states(16, 6)).cuda()
    before = [p.detach().clone() for p in net.parameters()]
    (net(rows) - 1.0).square().mean().backward()
    opt.step()
    assert all(torch.isfinite(p).all() for p in net.parameters())
    assert sum(not torch.equal(a, b) for a, b in zip(before, net.parameters())) >= len(before) - 2


def test_net_refuses():
    for bad in (dict(state_len=65), dict(layers=9), dict(ffn=100), dict(state_len=0)):
        with pytest.raises(RuntimeError):
            scorers.TransformerValueNet(**{**dict(state_len=54, num_values=6), **bad})


def test_action_scorer_learns_from_an_ensemble():
    """A wide ensemble's best moves as teacher: the loss and its gradients in a student's parameters."""
    pz = puzzles.puzzle54()
    ws = [puzzles.q_mlp_weights(54 * 6, pz.fanout, model_idx=i) for i in range(3)]
    teacher = scorers.MLPActionValueScorer(ws, 54, 64, 6, pz.fanout, max_parents=200)
    rows = torch.from_numpy(states(200, 8)).cuda()
    teacher.score(rows)
    values, moves = (-teacher.last_q(200) / 3 * 50).topk(4, dim=1)
    student = scorers.MLPActionScorer(54, (128, 64), pz.fanout, value_scale=5.0).cuda()
    loss = student.distillation_loss(rows[:, :54], values, moves, temperature=2.0)
    grads = torch.autograd.grad(loss, list(student.parameters()))
    z = student(rows[:, :54]).double() / 2.0
    p = (values.double() / 2.0).softmax(1)
    want = (p * (p.log() - z.log_softmax(1).gather(1, moves))).sum(1).mean()
    refs = torch.autograd.grad(want, list(student.parameters()))
    assert abs(loss.double() - want) <= 2.0 ** -16 * (1 + want.abs())
    for g, r in zip(grads, refs):
        # float32 against float32 backward passes through the same layers
        assert (g - r).norm() <= 2.0 ** -14 * r.norm() + 1e-9
