"""Cases of the operators around quantised, speculative serving and the training of its draft model.

Four operators, each in its plain form (elementary torch operations) and, with ``own`` set, as the
call that a user makes:

* ``norm``: ``ops.add_rms_norm_fp8``, the residual's addition, the root-mean-square norm and its e4m3
  output with one scale a row or a scale per 128 values;
* ``int4``: ``quantization.int4_linear``, a few tokens times a weight of 4 bits with group scales;
* ``distill``: ``ops.topk_distillation``, the loss against a teacher's stored top logits, with its gradient;
* ``verify``: ``ops.verify_draft``, which drafted tokens the target's probabilities accept, and the next token.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one new token of a 4096-wide model: the launch is what counts
        {"name": "norm 1x4096 row", "op": "norm", "rows": 1, "dim": 4096, "dtype": "bf16", "scaling": "rowwise"},
        # two sequences of 4096 tokens before the fp8 projections
        {"name": "norm 8192x4096 row", "op": "norm", "rows": 8192, "dim": 4096, "dtype": "bf16", "scaling": "rowwise"},
        # a ragged batch of an 8192-wide model, half precision, a scale per 128 values
        {"name": "norm 1023x8192 block", "op": "norm", "rows": 1023, "dim": 8192, "dtype": "f16", "scaling": "block"},
        # one token through an attention output projection
        {"name": "int4 1x4096x4096", "op": "int4", "tokens": 1, "out": 4096, "in": 4096, "group": 128, "zeros": False, "dtype": "bf16"},
        # four sequences through the gate or up projection of an 8192-wide model, with zero points
        {"name": "int4 4x28672x8192", "op": "int4", "tokens": 4, "out": 28672, "in": 8192, "group": 128, "zeros": True, "dtype": "bf16"},
        # a drafted block of seven tokens through a vocabulary projection, small groups, half precision
        {"name": "int4 7x128256x4096", "op": "int4", "tokens": 7, "out": 128256, "in": 4096, "group": 64, "zeros": False, "dtype": "f16"},
        # the loss alone on an evaluation batch, float logits, an odd vocabulary
        {"name": "distill loss 257x50257", "op": "distill", "rows": 257, "vocab": 50257, "top": 20, "temp": 2.0, "mode": "loss", "dtype": "f32"},
        # a training step through autograd
        {"name": "distill train 2048x128256", "op": "distill", "rows": 2048, "vocab": 128256, "top": 64, "temp": 1.0, "mode": "train", "dtype": "bf16"},
        # loss and gradient asked for together, as a training loop with its own backward pass does
        {"name": "distill grad 4096x128256", "op": "distill", "rows": 4096, "vocab": 128256, "top": 100, "temp": 1.5, "mode": "grad", "dtype": "bf16"},
        # one user, four drafted tokens
        {"name": "verify 1x4x32000", "op": "verify", "batch": 1, "drafted": 4, "vocab": 32000, "draft_probs": True, "dtype": "f32"},
        # a small batch, ragged drafts
        {"name": "verify 32x5x128256", "op": "verify", "batch": 32, "drafted": 5, "vocab": 128256, "draft_probs": True, "dtype": "f32"},
        # a full server
        {"name": "verify 256x7x128256", "op": "verify", "batch": 256, "drafted": 7, "vocab": 128256, "draft_probs": True, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "int4", "distill", "verify"])
    if op == "norm":
        scaling = rng.choice(["rowwise", "rowwise", "block"])
        dim = 128 * _log_int(rng, 1, 64) if scaling == "block" else _log_int(rng, 64, 8192)
        if scaling == "rowwise" and rng.random() < 0.7:
            dim = max(16, dim // 16 * 16)
        return {"op": op, "rows": _log_int(rng, 1, 8192), "dim": dim, "dtype": rng.choice(["bf16", "bf16", "f16"]), "scaling": scaling}
    if op == "int4":
        k = 32 * _log_int(rng, 8, 896)
        n = _log_int(rng, 64, min(128256, 250_000_000 // k))
        return {"op": op, "tokens": _log_int(rng, 1, 32), "out": n, "in": k, "group": rng.choice([32, 64, 128, 128]),
                "zeros": rng.random() < 0.5, "dtype": rng.choice(["bf16", "f16"])}
    if op == "distill":
        v = _log_int(rng, 1000, 128256)
        return {"op": op, "rows": _log_int(rng, 1, 3000), "vocab": v, "top": _log_int(rng, 1, 128), "temp": rng.choice([1.0, 1.5, 2.0, 4.0]),
                "mode": rng.choice(["loss", "train", "grad"]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    return {"op": op, "batch": _log_int(rng, 1, 200), "drafted": rng.randint(1, 7), "vocab": _log_int(rng, 1000, 128256),
            "draft_probs": rng.random() < 0.7, "dtype": rng.choice(["f32", "f32", "bf16"])}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"norm": _norm_in, "int4": _int4_in, "distill": _distill_in, "verify": _verify_in}[case["op"]](case, g)


def _norm_in(c, g):
    dt, m, d = _TYPES[c["dtype"]], c["rows"], c["dim"]
    x = torch.randn(m, d, device="cuda", generator=g).to(dt)
    # the residual stream: row sizes of several orders, a few channels far above the others
    r = torch.randn(m, d, device="cuda", generator=g) * torch.exp(torch.randn(m, 1, device="cuda", generator=g))
    r[:, :: max(1, d // 5)] *= 20.0
    w = (1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dt)
    return {"case": c, "x": x, "r": r.to(dt), "w": w, "eps": 1e-5}


def _int4_in(c, g):
    dt, m, n, k, group = _TYPES[c["dtype"]], c["tokens"], c["out"], c["in"], c["group"]
    groups = -(-k // group)
    x = torch.randn(m, k, device="cuda", generator=g).to(dt)
    packed = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = (torch.rand(n, groups, device="cuda", generator=g) * 0.01 + 0.005).to(dt)
    zeros = torch.randint(5, 11, (n, groups), device="cuda", generator=g, dtype=torch.uint8) if c["zeros"] else None
    return {"case": c, "x": x, "packed": packed, "scales": scales, "zeros": zeros, "group": group}


def _distill_in(c, g):
    dt, m, v, k = _TYPES[c["dtype"]], c["rows"], c["vocab"], min(c["top"], c["vocab"])
    logits = torch.randn(m, v, device="cuda", generator=g).mul_(2.0)
    # the teacher's k largest logits, sorted, at distinct ids; some rows keep fewer, and padded tokens none
    first = torch.randint(0, v, (m, 1), device="cuda", generator=g)
    step = torch.randint(1, max(2, v // k + 1), (m, 1), device="cuda", generator=g)
    ids = (first + step * torch.arange(k, device="cuda")) % v
    top = 12.0 + 2.0 * torch.randn(m, 1, device="cuda", generator=g) - torch.rand(m, k, device="cuda", generator=g).mul_(0.6).cumsum(1)
    logits.scatter_(1, ids, top + torch.randn(m, k, device="cuda", generator=g))
    kept = torch.where(torch.rand(m, 1, device="cuda", generator=g) < 0.2, torch.randint(0, k + 1, (m, 1), device="cuda", generator=g), k)
    if m == 1:
        kept.fill_(k)
    ids = torch.where(torch.arange(k, device="cuda") < kept, ids, -1)
    logits = logits.to(dt).requires_grad_(c["mode"] == "train")
    return {"case": c, "logits": logits, "values": top.float(), "ids": ids, "temp": c["temp"]}


def _verify_in(c, g):
    dt, b, k, v = _TYPES[c["dtype"]], c["batch"], c["drafted"], c["vocab"]
    target = torch.randn(b, k + 1, v, device="cuda", generator=g).mul_(3.0)
    draft = target[:, :k] + torch.randn(b, k, v, device="cuda", generator=g)
    draft = torch.softmax(draft, -1)
    # drafted tokens: drawn from the draft's probabilities by an exponential race
    race = torch.empty_like(draft).exponential_(generator=g)
    tokens = (draft / race).argmax(-1)
    del race
    target = torch.softmax(target, -1).to(dt)
    lens = torch.randint(max(0, k - 2), k + 1, (b,), device="cuda", generator=g, dtype=torch.int32) if b > 1 else None
    u = torch.rand(b, k + 1, device="cuda", generator=g)
    return {"case": c, "target": target, "draft": draft.to(dt) if c["draft_probs"] else None, "tokens": tokens, "lens": lens, "u": u}


# ------------------------------------------------------------------ one pass
def run(state):
    return {"norm": _norm, "int4": _int4, "distill": _distill, "verify": _verify}[state["case"]["op"]](state)


def _norm(st):
    x, r, w, eps, scaling = st["x"], st["r"], st["w"], st["eps"], st["case"]["scaling"]
    if own:
        from brain_b200 import ops

        return ops.add_rms_norm_fp8(x, r, w, eps, scaling)
    s = (x.float() + r.float()).to(x.dtype)
    f = s.float()
    y = f * (f.pow(2).mean(-1, keepdim=True) + eps).pow(-0.5) * w.float()
    if scaling == "block":
        y = y.view(y.shape[0], -1, 128)
    amax = y.abs().amax(-1)
    scale = torch.where(amax > 0, (amax / 448.0).clamp_min(2.0 ** -126), 1.0)
    q = (y / scale[..., None]).to(torch.float8_e4m3fn).view(x.shape)
    return q, scale, s


def _nibbles(packed):
    return torch.stack([packed & 15, packed >> 4], -1).view(packed.shape[0], -1)


def _int4(st):
    x, packed, scales, zeros, group = st["x"], st["packed"], st["scales"], st["zeros"], st["group"]
    if own:
        from brain_b200 import quantization

        return quantization.int4_linear(x, packed, scales, zeros, group_size=group)
    q = _nibbles(packed)
    k = q.shape[1]
    # values without zero points are two's complement
    q = q.float() - zeros.float().repeat_interleave(group, 1)[:, :k] if zeros is not None else (q ^ 8).float() - 8.0
    w = q * scales.float().repeat_interleave(group, 1)[:, :k]
    return (x.float() @ w.t()).to(x.dtype)


def _distill(st):
    z, t, ids, temp, mode = st["logits"], st["values"], st["ids"], st["temp"], st["case"]["mode"]
    if own:
        from brain_b200 import ops

        if mode == "grad":
            return ops.topk_distillation_grad(z, t, ids, temp)
        loss = ops.topk_distillation(z, t, ids, temp)
        return (loss, *torch.autograd.grad(loss, z)) if mode == "train" else loss
    with torch.no_grad():
        f = z.float() / temp
        top = f.amax(-1, keepdim=True)
        e = torch.exp(f - top)
        total = e.sum(-1, keepdim=True)
        lse = top + torch.log(total)
        on = ids >= 0
        t = torch.where(on, t.float() / temp, -math.inf)
        tmax = t.amax(-1, keepdim=True)
        some = tmax > -math.inf
        t = torch.where(some, t - tmax, -math.inf)
        te = torch.exp(t)
        tsum = te.sum(-1, keepdim=True).clamp_min(1.0)
        p = te / tsum
        at = ids.clamp_min(0)
        rows = torch.where(p > 0, p * (t - torch.log(tsum) - (f.gather(1, at) - lse)), 0.0).sum(-1) * temp ** 2
        n = some.sum().clamp_min(1)
        loss = rows.sum() / n
        if mode == "loss":
            return loss
        grad = e.div_(total).scatter_add_(1, at, -p)
        return loss, (grad * (some * (temp / n))).to(z.dtype)


def _verify(st):
    target, draft, tokens, lens, u = st["target"], st["draft"], st["tokens"], st["lens"], st["u"]
    if own:
        from brain_b200 import ops

        return ops.verify_draft(target, tokens, u, draft, lens)
    b, k = tokens.shape
    v = target.shape[-1]
    p = target[:, :k].gather(2, tokens[..., None])[..., 0].double()
    q = draft.gather(2, tokens[..., None])[..., 0].double() if draft is not None else torch.ones_like(p)
    yes = u[:, :k].double() * q < p
    if lens is not None:
        yes &= torch.arange(k, device=u.device) < lens[:, None]
    n = yes.long().cumprod(1).sum(1)
    row = torch.arange(b, device=u.device)
    rest = target[row, n].double()
    refused = n < (lens if lens is not None else k)
    at = n.clamp_max(k - 1)
    if draft is not None:
        left = (rest - draft[row, at].double()).clamp_min(0)
    else:
        left = rest.scatter(1, tokens[row, at][:, None], 0.0)
    left = torch.where((left > 0).any(1, keepdim=True), left, rest)
    rest = torch.where(refused[:, None], left, rest)
    run_ = rest.cumsum(1)
    goal = u[:, k].double()[:, None] * run_[:, -1:]
    nxt = (run_ > goal).long().argmax(1)
    out = torch.cat([tokens, torch.full_like(tokens[:, :1], -1)], 1)
    out = torch.where(torch.arange(k + 1, device=u.device) < n[:, None], out, -1)
    return out.scatter(1, n[:, None], nxt[:, None]), n


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "norm":
        n, size = c["rows"] * c["dim"], _BYTES[c["dtype"]]
        scales = c["rows"] * (c["dim"] // 128 if c["scaling"] == "block" else 1)
        return {"bytes": n * (3 * size + 1) + c["dim"] * size + 4 * scales, "flops": 8 * n}
    if c["op"] == "int4":
        m, n, k = c["tokens"], c["out"], c["in"]
        return {"bytes": n * k // 2 + n * -(-k // c["group"]) * (3 if c["zeros"] else 2) + 2 * m * (n + k), "flops": 2 * m * n * k}
    if c["op"] == "distill":
        n, size = c["rows"] * c["vocab"], _BYTES[c["dtype"]]
        grad = c["mode"] != "loss"
        return {"bytes": n * size * (2 if grad else 1) + c["rows"] * min(c["top"], c["vocab"]) * 12 + 4, "flops": n * (8 if grad else 4)}
    # one row of the target a sequence, and of the draft where a token is refused (most sequences here)
    rows = c["batch"] * (2 if c["draft_probs"] else 1)
    return {"bytes": rows * c["vocab"] * _BYTES[c["dtype"]] + c["batch"] * (c["drafted"] + 1) * 28, "flops": 3 * rows * c["vocab"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _norm64, "int4": _int464, "distill": _distill64, "verify": _verify64}[case["op"]](st)


def _norm64(st):
    total = st["x"].double() + st["r"].double()
    s = total.to(st["x"].dtype).double()
    size = s.square().sum(1) / s.shape[1] + st["eps"]
    y = s / size.sqrt()[:, None] * st["w"].double()
    width = 128 if st["case"]["scaling"] == "block" else s.shape[1]
    cut = y.reshape(-1, width)
    scale = cut.abs().max(1).values / 448.0
    scale[scale == 0] = 1.0
    q = (cut / scale[:, None]).reshape(y.shape)
    return q, scale.view(y.shape[0], -1) if width == 128 and st["case"]["scaling"] == "block" else scale, total


def _int464(st):
    x, packed, scales, zeros, group = st["x"].double(), st["packed"], st["scales"].double(), st["zeros"], st["group"]
    k = x.shape[1]
    y = torch.zeros(x.shape[0], packed.shape[0], dtype=torch.float64, device=x.device)
    for j, at in enumerate(range(0, k, group)):
        end = min(k, at + group)
        byte = packed[:, at // 2:end // 2].int()
        lo, hi = byte % 16, byte // 16
        if zeros is None:
            lo, hi = lo - 16 * (lo > 7), hi - 16 * (hi > 7)
        else:
            lo, hi = lo - zeros[:, j, None].int(), hi - zeros[:, j, None].int()
        y += (x[:, at:end:2] @ lo.double().t() + x[:, at + 1:end:2] @ hi.double().t()) * scales[:, j]
    return y


def _distill64(st):
    z, temp, mode = st["logits"].detach().double() / st["temp"], st["temp"], st["case"]["mode"]
    t = (st["values"].double() / temp).masked_fill(st["ids"] < 0, -math.inf)
    some = (st["ids"] >= 0).any(1)
    n = max(1, int(some.sum()))
    logp = torch.where(some[:, None], t, 0.0).log_softmax(1)
    p = logp.exp() * some[:, None]
    lse = torch.logsumexp(z, 1)
    logq = torch.take_along_dim(z, st["ids"].clamp(min=0), 1) - lse[:, None]
    loss = (p * torch.where(p > 0, logp - logq, 0.0)).sum() * temp * temp / n
    if mode == "loss":
        return loss
    z.sub_(lse[:, None]).exp_()
    z.mul_(some[:, None])
    z.scatter_add_(1, st["ids"].clamp(min=0), -p)
    return loss, z.mul_(temp / n)


def _verify64(st):
    target, u, tokens = st["target"], st["u"].double().cpu(), st["tokens"].cpu()
    b, k = tokens.shape
    out, count = torch.full((b, k + 1), -1, dtype=torch.int64), torch.zeros(b, dtype=torch.int64)
    for i in range(b):
        n, drafted = 0, k if st["lens"] is None else int(st["lens"][i])
        while n < drafted:
            x = int(tokens[i, n])
            share = float(target[i, n, x])
            if st["draft"] is not None:
                share /= float(st["draft"][i, n, x])
            if float(u[i, n]) >= share:
                break
            out[i, n] = x
            n += 1
        left = target[i, n].double().cpu()
        if n < drafted:
            other = left.clone()
            if st["draft"] is not None:
                other -= st["draft"][i, n].double().cpu()
            else:
                other[tokens[i, n]] = 0.0
            other[other < 0] = 0.0
            left = other if other.sum() > 0 else left
        sums = torch.cumsum(left, 0)
        out[i, n] = int(torch.searchsorted(sums, u[i, k] * sums[-1], right=True))
        count[i] = n
    return out.to(target.device), count.to(target.device)
