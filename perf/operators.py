"""Measured cases of the operators that train and serve the attention scorers and distil action scorers.

Three operators, each in its plain form (elementary torch operations in 32 bits, rounded once at the end) and through
the package's own entry points:

* ``qk_norm_rope``: RMS norm of every query and key head with a learned gain, and the rotation by position, in one pass;
* ``relative_attention``: softmax(q k^T scale + table[bucket(j - i)]) v with a learned bias per head and distance bucket;
* ``distill_top_logits``: cross-entropy excess of a student's logits over a teacher's top entries, with its gradient.

``own`` selects which of the two ``run`` computes.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # one state of 54 stickers at the start of a search: only latency counts
        dict(name="qknorm_one_state", op="qknorm", train=False, b=1, t=54, h=8, hkv=8, d=32, dtype="bf16", far=False, pairs="half"),
        # one micro-batch of the transformer scorer (32 768 states of 54 tokens, 8 heads of 32)
        dict(name="qknorm_microbatch", op="qknorm", train=False, b=32768, t=54, h=8, hkv=8, d=32, dtype="bf16", far=False, pairs="half"),
        # training on long ragged sequences with shared key heads, wide heads, positions far into a stream
        dict(name="qknorm_train_shared_keys", op="qknorm", train=True, b=3, t=4097, h=16, hkv=4, d=128, dtype="bf16", far=True, pairs="half"),
        # training in 32 bits on a batch of states, neighbouring elements rotated together
        dict(name="qknorm_train_f32", op="qknorm", train=True, b=2048, t=54, h=8, hkv=8, d=32, dtype="f32", far=False, pairs="neighbours"),
        # attention of one state: only latency counts
        dict(name="attention_one_state", op="attention", train=False, b=1, t=54, h=8, hkv=8, d=32, dtype="bf16", causal=False, ragged=False),
        # attention of one micro-batch of the transformer scorer
        dict(name="attention_microbatch", op="attention", train=False, b=32768, t=54, h=8, hkv=8, d=32, dtype="bf16", causal=False, ragged=False),
        # a training step's attention over a batch of states, forward and backward
        dict(name="attention_train_states", op="attention", train=True, b=8192, t=54, h=8, hkv=8, d=32, dtype="bf16", causal=False, ragged=False),
        # long sequences, forward
        dict(name="attention_long", op="attention", train=False, b=2, t=4096, h=8, hkv=8, d=64, dtype="bf16", causal=False, ragged=False),
        # a padded batch of long odd-length sequences with shared key heads and a causal mask, forward and backward
        dict(name="attention_train_padded", op="attention", train=True, b=6, t=1501, h=8, hkv=2, d=64, dtype="f16", causal=True, ragged=True),
        # an action scorer's twelve moves over the benchmark's beam, loss and gradient
        dict(name="distill_moves", op="distill", grad=True, rows=65536, v=12, k=4, dtype="f32", padded=True, temperature=2.0),
        # a training batch over a wide odd vocabulary, loss and gradient
        dict(name="distill_wide", op="distill", grad=True, rows=4096, v=50021, k=64, dtype="bf16", padded=False, temperature=1.5),
        # a few rows of a very wide vocabulary, loss only
        dict(name="distill_few_rows", op="distill", grad=False, rows=8, v=131072, k=32, dtype="f16", padded=False, temperature=1.0),
    ]


def log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qknorm", "attention", "distill"])
    if op == "qknorm":
        h = rng.choice([1, 2, 4, 6, 8, 12, 16])
        hkv = rng.choice([n for n in (1, 2, 3, 4, 6, 8, 12, 16) if h % n == 0])
        d = rng.choice([32, 64, 80, 128])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        t = log_uniform(rng, 1, 4500)
        top = 4e8 / ((h + hkv) * d * SIZE[dtype] * t)
        return dict(op=op, train=rng.random() < 0.5, b=log_uniform(rng, 1, max(1.5, min(16384, top))), t=t, h=h, hkv=hkv, d=d, dtype=dtype,
                    far=rng.random() < 0.3, pairs=rng.choice(["half", "neighbours"]))
    if op == "attention":
        h = rng.choice([1, 2, 4, 8, 12])
        hkv = rng.choice([n for n in (1, 2, 4, 8, 12) if h % n == 0] + [h])
        d = rng.choice([32, 64])
        train = rng.random() < 0.5
        pairs = min(4e8, 9e10 / (d * (14 if train else 4)))
        t = rng.choice([log_uniform(rng, 1, 64), log_uniform(rng, 1, min(3500, math.sqrt(pairs / h)))])
        top = min(6e7 / (h * d * t), pairs / (h * t * t))
        return dict(op=op, train=train, b=log_uniform(rng, 1, max(1.5, min(16384, top))), t=t, h=h, hkv=hkv, d=d,
                    dtype=rng.choice(["bf16", "bf16", "f16"]), causal=rng.random() < 0.4, ragged=rng.random() < 0.4)
    v = log_uniform(rng, 12, 150000)
    return dict(op=op, grad=rng.random() < 0.7, rows=log_uniform(rng, 1, min(65536, 1.5e8 / v)), v=v, k=min(v, log_uniform(rng, 1, 100)),
                dtype=rng.choice(["bf16", "f16", "f32"]), padded=rng.random() < 0.4, temperature=rng.choice([1.0, 1.5, 2.0, 4.0]))


NUM_BUCKETS, MAX_DISTANCE = 32, 128


def bucket_map(causal):
    """Bucket of key minus query for offsets -MAX_DISTANCE .. MAX_DISTANCE (further ones share the ends' buckets), in whole numbers: half of
    each side's buckets hold one distance each, the others grow by equal factors up to MAX_DISTANCE."""
    side = NUM_BUCKETS if causal else NUM_BUCKETS // 2
    exact_ = side // 2
    got = []
    for off in range(-MAX_DISTANCE, MAX_DISTANCE + 1):
        n = max(-off, 0) if causal else abs(off)
        steps = side - exact_
        if n >= exact_:
            grown = 0  # the largest s with n >= exact * (MAX / exact) ** (s / steps)
            while grown < steps - 1 and n ** steps * exact_ ** (grown + 1) >= MAX_DISTANCE ** (grown + 1) * exact_ ** steps:
                grown += 1
            n = exact_ + grown
        got.append(n + (side if not causal and off > 0 else 0))
    return got


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if to == torch.float32 else to) * scale).to(to)

    s = dict(case=case)
    if case["op"] == "distill":
        rows, v, k = case["rows"], case["v"], case["k"]
        s["logits"] = normal(rows, v, scale=2.0)
        t = torch.empty((rows, k), device="cuda")
        i = torch.empty((rows, k), device="cuda", dtype=torch.int64)
        step = max(1, int(5e7 // v))
        for r in range(0, rows, step):  # the teacher agrees with the student up to some noise
            z = s["logits"][r:r + step].float()
            t[r:r + step], i[r:r + step] = (z + torch.randn(z.shape, generator=g, device="cuda")).topk(k, dim=1)
        if case["padded"]:  # rows with fewer entries, some of them with none
            left = torch.randint(0, k + 1, (rows, 1), generator=g, device="cuda")
            i = torch.where(torch.arange(k, device="cuda") < left, i, -1)
        s.update(teacher=t, index=i, weight=torch.rand((rows,), generator=g, device="cuda") / rows)
        return s
    b, t, h, hkv, d = (case[n] for n in ("b", "t", "h", "hkv", "d"))
    # queries, keys and values lie beside one another, as one projection of the layer's input leaves them
    packed = normal(b, t, h + 2 * hkv, d)
    s["q"], s["k"], s["v"] = packed[:, :, :h], packed[:, :, h:h + hkv], packed[:, :, h + hkv:]
    train = case["train"]
    if case["op"] == "qknorm":
        s["q_gain"] = 1 + 0.1 * normal(d, to=torch.float32)
        s["k_gain"] = 1 + 0.1 * normal(d, to=torch.float32)
        s["base"] = 10000.0
        s["positions"] = torch.arange(t, device="cuda")
        if case["far"]:
            s["positions"] = s["positions"] + torch.randint(0, 1 << 20, (b, 1), generator=g, device="cuda")
        if train:
            s["dq"], s["dk"] = normal(b, t, h, d), normal(b, t, hkv, d)
            for n in ("q", "k", "q_gain", "k_gain"):
                s[n] = s[n].detach().requires_grad_(True)
    else:
        s["table"] = normal(NUM_BUCKETS, h, scale=0.5)
        s["map"] = torch.tensor(bucket_map(case["causal"]), device="cuda")
        s["lengths"] = torch.randint(t // 2, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        if train:
            s["dout"] = normal(b, t, h, d)
            for n in ("q", "k", "v", "table"):
                s[n] = s[n].detach().requires_grad_(True)
    return s


PLANS = {}


def plan(make, *args, **more):
    """The package's handle for these frequencies or buckets: a program builds one for its model and keeps it."""
    key = (make.__name__, args, tuple(sorted(more.items())))
    if key not in PLANS:
        PLANS[key] = make(*args, device="cuda", **more)
    return PLANS[key]


def run(s):
    if own:
        return run_own(s)
    with torch.no_grad():
        return {"qknorm": plain_qknorm, "attention": plain_attention, "distill": plain_distill}[s["case"]["op"]](s)


def run_own(s):
    from multigpubeamsearch_b200 import operators as ops

    c = s["case"]
    if c["op"] == "qknorm":
        rotary = plan(ops.RotaryFrequencies, c["d"], base=s["base"])
        q, k = ops.qk_norm_rope(s["q"], s["k"], s["q_gain"], s["k_gain"], rotary, positions=s["positions"], eps=EPS, interleaved=c["pairs"] == "neighbours")
        if not c["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"], s["q_gain"], s["k_gain"]), (s["dq"], s["dk"]))]
    if c["op"] == "attention":
        buckets = plan(ops.RelativeBuckets, NUM_BUCKETS, MAX_DISTANCE, causal=c["causal"])
        out = ops.relative_attention(s["q"], s["k"], s["v"], s["table"], buckets, lengths=s["lengths"])
        if not c["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["table"]), s["dout"])]
    if not c["grad"]:
        return [ops.distill_top_logits(s["logits"], s["teacher"], s["index"], temperature=c["temperature"])]
    return list(ops.distill_top_logits_step(s["logits"], s["teacher"], s["index"], temperature=c["temperature"], row_weight=s["weight"]))


def halves(x, pairs):
    """The two members of every rotated pair."""
    if pairs == "half":
        return x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return x[..., 0::2], x[..., 1::2]


def joined(a, b, pairs):
    return torch.cat([a, b], dim=-1) if pairs == "half" else torch.stack([a, b], dim=-1).flatten(-2)


def plain_qknorm(s):
    c = s["case"]
    d, pairs, dtype = c["d"], c["pairs"], DTYPES[c["dtype"]]
    # far positions lose their angle in 32 bits
    freq = s["base"] ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = s["positions"].double()[..., None] * freq
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]

    def forward(x, gain):
        x = x.float()
        a, b = halves(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain, pairs)
        return joined(a * cos - b * sin, b * cos + a * sin, pairs).to(dtype)

    def backward(x, gain, dy):
        x = x.float()
        a, b = halves(dy.float(), pairs)
        u = joined(a * cos + b * sin, b * cos - a * sin, pairs)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n, w = x * r, u * gain
        return (r * (w - n * (w * n).mean(-1, keepdim=True))).to(dtype), (u * n).sum((0, 1, 2))

    out = [forward(s["q"], s["q_gain"]), forward(s["k"], s["k_gain"])]
    if c["train"]:
        (dq, dgq), (dk, dgk) = backward(s["q"], s["q_gain"], s["dq"]), backward(s["k"], s["k_gain"], s["dk"])
        out += [dq, dk, dgq, dgk]
    return out


def plain_attention(s):
    c = s["case"]
    b, t, h, hkv, d, dtype = c["b"], c["t"], c["h"], c["hkv"], c["d"], DTYPES[c["dtype"]]
    scale = 1 / math.sqrt(d)
    q = s["q"].float().transpose(1, 2)
    k, v = (s[n].float().transpose(1, 2).repeat_interleave(h // hkv, dim=1) for n in ("k", "v"))
    at = torch.arange(t, device="cuda")
    off = at[None, :] - at[:, None]
    index = s["map"][off.clamp(-MAX_DISTANCE, MAX_DISTANCE) + MAX_DISTANCE]
    p = q @ k.transpose(-1, -2) * scale
    p += s["table"].float()[index].permute(2, 0, 1)
    seen = torch.ones((1, 1, t, t), dtype=torch.bool, device="cuda")
    if c["causal"]:
        seen = seen & (off <= 0)
    if s["lengths"] is not None:
        valid = at < s["lengths"][:, None]
        seen = seen & valid[:, None, :, None] & valid[:, None, None, :]
    p.masked_fill_(~seen, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp_min(-1e30))
    p /= p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = p @ v
    out = [o.transpose(1, 2).to(dtype)]
    if c["train"]:
        do = s["dout"].float().transpose(1, 2)
        ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
        dv, dk = p.transpose(-1, -2) @ do, ds.transpose(-1, -2) @ q * scale
        dq = ds @ k * scale
        dtable = torch.zeros((NUM_BUCKETS, h), device="cuda").index_add_(0, index.flatten(), ds.sum(0).flatten(1).t())
        dk, dv = (x.unflatten(1, (hkv, h // hkv)).sum(2) for x in (dk, dv))
        out += [x.transpose(1, 2).to(dtype) for x in (dq, dk, dv)] + [dtable.to(dtype)]
    return out


def plain_distill(s):
    c = s["case"]
    z = s["logits"].float() / c["temperature"]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    log_q = z.gather(1, s["index"].clamp_min(0)) - m - torch.log(total)
    held = s["index"] >= 0
    t = (s["teacher"] / c["temperature"]).masked_fill(~held, -math.inf)
    t = t - t.amax(1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(t)
    sums = p.sum(1, keepdim=True)
    p = p / sums.clamp_min(1e-30)
    loss = torch.where(p > 0, p * (t - torch.log(sums) - log_q), 0.0).sum(1)
    if not c["grad"]:
        return [loss]
    some = held.any(1, keepdim=True)
    w = s["weight"][:, None] / c["temperature"]
    grad = e / total * (w * some)
    grad.scatter_add_(1, s["index"].clamp_min(0), -p * w)
    return [loss, grad.to(s["logits"].dtype)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"qknorm": exact_qknorm, "attention": exact_attention, "distill": exact_distill}[case["op"]](s, case)


def slices(total, size):
    size = max(1, size)
    return [slice(a, min(total, a + size)) for a in range(0, total, size)]


def exact_qknorm(s, case):
    """Pairs as complex numbers in 64 bits, gradients by differentiation."""
    b, t, d = case["b"], case["t"], case["d"]
    angle = s["positions"].double()[..., None] * torch.exp(-math.log(s["base"]) * torch.arange(d // 2, device="cuda", dtype=torch.float64) / (d / 2))
    turn = torch.polar(torch.ones_like(angle), angle)[..., None, :]
    done = {"q": [], "k": [], "dq": [], "dk": []}
    gains = {n: s[n + "_gain"].detach().double() for n in "qk"}
    dgain = {n: torch.zeros(d, device="cuda", dtype=torch.float64) for n in "qk"}
    for at in slices(b, int(3e7 // (t * d * case["h"]))):
        for n in "qk":
            x = s[n].detach()[at].double().requires_grad_(case["train"])
            gain = gains[n].clone().requires_grad_(case["train"])
            y = gain * x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
            z = torch.complex(y[..., :d // 2], y[..., d // 2:]) if case["pairs"] == "half" else torch.view_as_complex(y.reshape(*y.shape[:-1], d // 2, 2))
            z = z * (turn[at] if case["far"] else turn)
            y = torch.cat([z.real, z.imag], -1) if case["pairs"] == "half" else torch.view_as_real(z).flatten(-2)
            done[n].append(y.detach())
            if case["train"]:
                dx, dg = torch.autograd.grad(y, (x, gain), s["d" + n][at].double())
                done["d" + n].append(dx)
                dgain[n] += dg
    out = [torch.cat(done["q"]), torch.cat(done["k"])]
    return out + [torch.cat(done["dq"]), torch.cat(done["dk"]), dgain["q"], dgain["k"]] if case["train"] else out


def exact_attention(s, case):
    """One softmax per sequence in 64 bits, gradients by differentiation; buckets by counting the borders below a distance."""
    b, t, h, hkv, d, causal, train = (case[n] for n in ("b", "t", "h", "hkv", "d", "causal", "train"))
    if b * h * t * t > 4e9:
        return None
    side = NUM_BUCKETS if causal else NUM_BUCKETS // 2
    low = side // 2
    at = torch.arange(t, device="cuda")
    off = at - at[:, None]
    far = (-off).clamp_min(0) if causal else off.abs()
    index = far.clamp_max(low)
    for n in range(1, side - low):  # the first distance that lies at or over low * (MAX / low) ** (n / (side - low))
        first = next(x for x in range(low, MAX_DISTANCE + 1) if x ** (side - low) * low ** n >= MAX_DISTANCE ** n * low ** (side - low))
        index = index + (far >= first)
    if not causal:
        index = index + side * (off > 0)
    table = s["table"].detach().double().requires_grad_(train)
    outs, grads = [], [[], [], [], torch.zeros_like(table, requires_grad=False)]
    for part in slices(b, int(1e8 // (h * t * t))):
        q, k, v = (s[n].detach()[part].double().requires_grad_(train) for n in "qkv")
        w = torch.einsum("bighd,bjgd->bghij", q.unflatten(2, (hkv, h // hkv)), k) / d ** 0.5
        w = w + table.t()[:, index].unflatten(0, (hkv, h // hkv))
        dead = torch.zeros((1, t, t), dtype=torch.bool, device="cuda")
        if causal:
            dead = dead | (off > 0)
        if s["lengths"] is not None:
            gone = at >= s["lengths"][part][:, None]
            dead = dead | gone[:, :, None] | gone[:, None, :]
        dead = dead[:, None, None]
        # a row without keys gives zeros
        w = w.masked_fill(dead, -1e300).softmax(-1).masked_fill(dead, 0.0)
        o = torch.einsum("bghij,bjgd->bighd", w, v).flatten(2, 3)
        outs.append(o.detach())
        if train:
            got = torch.autograd.grad(o, (q, k, v, table), s["dout"][part].double())
            for n in range(3):
                grads[n].append(got[n])
            grads[3] = grads[3] + got[3]
    return [torch.cat(outs)] + ([torch.cat(grads[0]), torch.cat(grads[1]), torch.cat(grads[2]), grads[3]] if train else [])


def exact_distill(s, case):
    """Kullback-Leibler divergence in 64 bits from dense target rows, gradient by differentiation."""
    losses, grads = [], []
    for at in slices(case["rows"], int(5e7 // case["v"])):
        z = s["logits"][at].double().requires_grad_(case["grad"])
        held = s["index"][at] >= 0
        weight = (s["teacher"][at].double() / case["temperature"]).masked_fill(~held, -math.inf)
        log_p = (weight - weight.logsumexp(1, keepdim=True)).masked_fill(~held, 0.0)
        p = torch.where(held, log_p.exp(), 0.0)
        log_q = (z / case["temperature"]).log_softmax(1)
        target = torch.zeros_like(z, requires_grad=False).scatter_add(1, s["index"][at].clamp_min(0), p)
        loss = (p * log_p).sum(1) - (target * log_q).sum(1)
        losses.append(loss.detach())
        if case["grad"]:
            grads.append(torch.autograd.grad(loss, z, s["weight"][at].double())[0])
    return [torch.cat(losses)] + ([torch.cat(grads)] if case["grad"] else [])


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "distill":
        dense, top = case["rows"] * case["v"], case["rows"] * case["k"]
        return {"bytes": dense * e * (2 if case["grad"] else 1) + top * 12 + case["rows"] * (8 if case["grad"] else 4), "flops": dense * (6 if case["grad"] else 4)}
    b, t, h, hkv, d, train = (case[n] for n in ("b", "t", "h", "hkv", "d", "train"))
    if case["op"] == "qknorm":
        n = b * t * (h + hkv) * d
        return {"bytes": n * e * (4 if train else 2) + t * (b if case["far"] else 1) * 8, "flops": n * (20 if train else 7)}
    # padded sequences hold three quarters of the tokens and seven twelfths of the pairs on average
    rows = b * t * (0.75 if case["ragged"] else 1.0)
    pairs = b * h * t * t * (7 / 12 if case["ragged"] else 1.0) * (0.5 if case["causal"] else 1.0)
    read = rows * (h + 2 * hkv) * d + (rows * h * d if train else 0)
    written = b * t * h * d + (b * t * (h + 2 * hkv) * d if train else 0)
    return {"bytes": (read + written) * e, "flops": pairs * d * (14 if train else 4)}
