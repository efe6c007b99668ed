"""What is measured of the operators at the end of a training step: the block-level norms with their backward passes and the
head's losses, which take the normalised rows through the vocabulary projection to a loss and its gradients.

`run` computes a case either with elementary torch operations (`own` false) or through the package's entry points (`own`
true); `exact` restates each operator in 64 bits from its definition.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
EPS = 1.0e-5


def listed():
    return [
        # one row between two blocks, the shortest call: bound by launches
        {"name": "norm_one_row", "op": "norm", "rows": 1, "channels": 2048},
        # the norm of a block, 8 sequences of 1024 tokens
        {"name": "norm_block", "op": "norm", "rows": 8192, "channels": 2048},
        # a packed batch whose length and width fit no tile
        {"name": "norm_odd", "op": "norm", "rows": 1237, "channels": 1000},
        # a short batch of a small model, residual stream added in the same pass
        {"name": "add_norm_short", "op": "add_norm", "rows": 64, "channels": 768},
        # the norms between the blocks of a larger model, 2 sequences of 4096 tokens
        {"name": "add_norm_block", "op": "add_norm", "rows": 8192, "channels": 4096},
        # a handful of tokens against the whole vocabulary (tuning a state on one short sample): bound by the weight's bytes
        {"name": "ce_few_tokens", "op": "ce", "rows": 16, "channels": 1024, "vocab": 65536, "ignored": 0.0, "train": True},
        # the loss of a pretraining step, 8 sequences of 1024 tokens
        {"name": "ce_pretrain", "op": "ce", "rows": 8192, "channels": 2048, "vocab": 65536, "ignored": 0.0, "train": True},
        # the losses of a held-out set, token by token, without gradients
        {"name": "ce_eval", "op": "ce", "rows": 4096, "channels": 1024, "vocab": 65536, "ignored": 0.0, "train": False},
        # a padded fine-tuning batch: odd length, odd vocabulary, a third of the tokens without a label
        {"name": "ce_padded_odd", "op": "ce", "rows": 777, "channels": 1544, "vocab": 50277, "ignored": 0.3, "train": True},
        # a step of distillation from a cache of a teacher's 64 highest logits per token
        {"name": "distill_step", "op": "distill", "rows": 2048, "channels": 2048, "vocab": 65536, "top": 64,
         "temperature": 2.0, "missing": 0.0},
        # a small student with a ragged cache: some entries and some rows without any teacher
        {"name": "distill_ragged", "op": "distill", "rows": 33, "channels": 512, "vocab": 8191, "top": 8,
         "temperature": 1.0, "missing": 0.25},
    ]


def _spread(rng, low, high, step=1):
    """A whole number of low..high, even in its logarithm, a multiple of step."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(value) // step * step))


def draw(rng):
    kind = rng.choice(["norm", "add_norm", "ce", "ce", "ce_eval", "distill", "distill"])
    if kind in ("norm", "add_norm"):
        channels = _spread(rng, 64, 8192, 8)
        return {"op": kind, "rows": _spread(rng, 1, min(32768, 8192 * 4096 // channels)), "channels": channels}
    most = 8192 * 2048 * 65536
    channels = _spread(rng, 64, 4096, 8)
    vocab = _spread(rng, 500, 65536)
    if kind == "distill":
        case = {"op": "distill", "rows": _spread(rng, 1, min(4096, most // 4 // (channels * vocab) + 1)), "channels": channels,
                "vocab": vocab, "top": _spread(rng, 1, 128), "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]),
                "missing": rng.choice([0.0, 0.1, 0.5])}
        return case
    return {"op": "ce", "rows": _spread(rng, 1, min(8192, most // (channels * vocab))), "channels": channels, "vocab": vocab,
            "ignored": rng.choice([0.0, 0.0, 0.1, 0.6]), "train": kind == "ce"}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * scale

    rows, channels = case["rows"], case["channels"]
    state = {"case": case}
    if case["op"] in ("norm", "add_norm"):
        # the residual stream has a mean, and its channels differ in size
        spread = torch.exp(normal(channels, scale=0.5))
        x = normal(1, rows, channels) * spread + 0.3 * normal(channels)
        state["x"] = x.to(BF16)
        if case["op"] == "add_norm":
            state["residual"] = normal(1, rows, channels, scale=2.0).to(BF16)
            state["grad_sum"] = normal(1, rows, channels, scale=0.01).to(BF16)
        state["weight"] = (1.0 + normal(channels, scale=0.2)).to(BF16)
        state["bias"] = normal(channels, scale=0.1).to(BF16)
        state["grad"] = normal(1, rows, channels, scale=0.01).to(BF16)
        leaves = ("x", "residual", "weight", "bias")
    else:
        vocab = case["vocab"]
        # logits of a deviation of about two, and tokens that range from unlikely to nearly certain
        weight = normal(vocab, channels, scale=2.0 / math.sqrt(channels))
        target = torch.randint(vocab, (rows,), generator=gen, device="cuda")
        sure = 3.0 * torch.rand(rows, 1, generator=gen, device="cuda")
        x = normal(rows, channels) + 2.0 * sure * weight[target]
        state["x"], state["weight"] = x.to(BF16), weight.to(BF16)
        if case["op"] == "ce":
            drop = torch.rand(rows, generator=gen, device="cuda") < case["ignored"]
            state["targets"] = torch.where(drop, torch.full_like(target, -100), target)
        else:
            top = min(case["top"], vocab)
            # distinct tokens with falling logits, the likely token first
            step = vocab // top
            order = torch.rand(rows, top, generator=gen, device="cuda").argsort(dim=1)
            order = torch.where(order == 0, order[:, :1], order)
            order[:, 0] = 0
            state["indices"] = ((target[:, None] + order * step) % vocab).to(torch.int32)
            gaps = torch.rand(rows, top, generator=gen, device="cuda") * (8.0 / top)
            logits = 10.0 + normal(rows, 1) - torch.cumsum(gaps, dim=1)
            if case["missing"] > 0:
                kept = torch.randint(0, top + 1, (rows, 1), generator=gen, device="cuda")
                whole = torch.rand(rows, 1, generator=gen, device="cuda") >= case["missing"]
                absent = (torch.arange(top, device="cuda")[None, :] >= kept) & ~whole
                logits = logits.masked_fill(absent, float("-inf"))
            state["teacher"] = logits
        leaves = ("x", "weight")
    if own:
        import flashrwkv_b200

        state["package"] = flashrwkv_b200
        for name in leaves:
            if name in state:
                state[name].requires_grad_(case.get("train", True))
    return state


# ---- the package's entry points -------------------------------------------------------------------------------------
def _run_own(state):
    case, F = state["case"], state["package"]
    if case["op"] == "norm":
        leaves = (state["x"], state["weight"], state["bias"])
        out = F.pretrain_tmix_layer_norm_bf16(*leaves, eps=EPS)
        return (out.detach(), *torch.autograd.grad(out, leaves, state["grad"]))
    if case["op"] == "add_norm":
        leaves = (state["x"], state["residual"], state["weight"], state["bias"])
        total, out = F.pretrain_tmix_add_layer_norm_bf16(*leaves, eps=EPS)
        grads = torch.autograd.grad((total, out), leaves, (state["grad_sum"], state["grad"]))
        return (total.detach(), out.detach(), *grads)
    leaves = (state["x"], state["weight"])
    if case["op"] == "ce":
        if not case["train"]:
            with torch.no_grad():
                return F.pretrain_head_cross_entropy_bf16(*leaves, state["targets"], reduction="none")
        loss = F.pretrain_head_cross_entropy_bf16(*leaves, state["targets"])
    else:
        loss = F.pretrain_head_distill_bf16(*leaves, state["teacher"], state["indices"], temperature=case["temperature"])
    return (loss.detach(), *torch.autograd.grad(loss, leaves))


# ---- the plain form -------------------------------------------------------------------------------------------------
def _norm_plain(total, weight, bias, grad):
    """The normalised rows, the gradient of the rows, and those of weight and bias; all in 32 bits."""
    mean = total.mean(dim=-1, keepdim=True)
    centred = total - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=-1, keepdim=True) + EPS)
    unit = centred * rstd
    out = unit * weight + bias
    gw = grad * weight
    dx = rstd * (gw - gw.mean(dim=-1, keepdim=True) - unit * (gw * unit).mean(dim=-1, keepdim=True))
    return out, dx, (grad * unit).sum(dim=(0, 1)), grad.sum(dim=(0, 1))


def _run_plain(state):
    case = state["case"]
    if case["op"] == "norm":
        parts = _norm_plain(*(state[n].float() for n in ("x", "weight", "bias", "grad")))
        return tuple(p.to(BF16) for p in parts)
    if case["op"] == "add_norm":
        total = (state["x"].float() + state["residual"].float()).to(BF16)  # the sum is an output, rounded like one
        out, dx, dw, db = _norm_plain(total.float(), *(state[n].float() for n in ("weight", "bias", "grad")))
        dx = (dx + state["grad_sum"].float()).to(BF16)
        return total, out.to(BF16), dx, dx, dw.to(BF16), db.to(BF16)
    x, weight = state["x"].float(), state["weight"].float()
    logits = x @ weight.t()
    if case["op"] == "ce":
        targets = state["targets"]
        valid = targets != -100
        at = torch.where(valid, targets, torch.zeros_like(targets))[:, None]
        top = logits.max(dim=1, keepdim=True).values
        lse = top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True))
        losses = torch.where(valid[:, None], lse - logits.gather(1, at), torch.zeros_like(lse))[:, 0]
        if not case["train"]:
            return losses
        count = valid.sum().clamp_min(1).float()
        delta = torch.exp(logits - lse)
        del logits
        delta.scatter_add_(1, at, torch.full_like(lse, -1.0))
        delta *= valid[:, None].float() / count
        loss = losses.sum() / count
    else:
        temperature, teacher, at = case["temperature"], state["teacher"], state["indices"].long()
        logits /= temperature
        there = teacher > float("-inf")
        valid = there.any(dim=1, keepdim=True)
        count = valid.sum().clamp_min(1).float()
        soft = teacher.float() / temperature
        high = torch.where(valid, soft.max(dim=1, keepdim=True).values, torch.zeros_like(soft[:, :1]))
        power = torch.where(there, torch.exp(soft - high), torch.zeros_like(soft))
        total = torch.where(valid, power.sum(dim=1, keepdim=True), torch.ones_like(high))
        p = power / total
        log_p = torch.where(there, soft - high - torch.log(total), torch.zeros_like(soft))
        top = logits.max(dim=1, keepdim=True).values
        lse = top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True))
        safe = torch.where(there, at, torch.zeros_like(at))
        log_q = logits.gather(1, safe) - lse
        loss = temperature * temperature * (p * (log_p - log_q)).sum() / count
        delta = torch.exp(logits - lse)
        del logits
        delta.scatter_add_(1, safe, -p)
        delta *= valid.float() * (temperature / count)
    return loss, (delta @ weight).to(BF16), (delta.t() @ x).to(BF16)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    rows, channels = case["rows"], case["channels"]
    if case["op"] == "norm":  # x, its gradient's source, the output and dx, all in 16 bits; weight, bias and their gradients
        return {"bytes": 4 * rows * channels * 2 + 4 * channels * 2, "flops": 20 * rows * channels}
    if case["op"] == "add_norm":  # x, residual, two upstream gradients in; sum, output and one gradient for both addends out
        return {"bytes": 7 * rows * channels * 2 + 4 * channels * 2, "flops": 22 * rows * channels}
    vocab = case["vocab"]
    operands = (rows * channels + vocab * channels) * 2
    if case["op"] == "ce" and not case["train"]:
        return {"bytes": operands + rows * 12, "flops": 2 * rows * vocab * channels}
    labels = rows * 8 if case["op"] == "ce" else rows * min(case["top"], vocab) * 8
    labelled = rows * (1.0 - case.get("ignored", 0.0))  # a row without a label needs no product
    return {"bytes": 2 * operands + labels + 4, "flops": int(6 * labelled * vocab * channels)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_norm(rows, weight, bias, grad):
    rows = rows.double().flatten(0, 1)
    weight, bias, grad = weight.double(), bias.double(), grad.double().flatten(0, 1)
    n = rows.shape[1]
    deviation = rows - rows.sum(1, keepdim=True) / n
    scale = ((deviation ** 2).sum(1, keepdim=True) / n + EPS) ** -0.5
    hat = deviation * scale
    inner = grad * weight
    along = (inner * hat).sum(1, keepdim=True) / n
    d_rows = (inner - inner.sum(1, keepdim=True) / n - hat * along) * scale
    return (hat * weight + bias)[None], d_rows[None], (grad * hat).sum(0), grad.sum(0)


def exact(case, seed):
    state = prepare(case, seed)
    state = {k: (v.detach() if isinstance(v, torch.Tensor) else v) for k, v in state.items()}
    if case["op"] == "norm":
        return _exact_norm(state["x"], state["weight"], state["bias"], state["grad"])
    if case["op"] == "add_norm":
        whole = state["x"].double() + state["residual"].double()
        # the rows that are normalised are the sum as the caller gets it
        out, dx, dw, db = _exact_norm(whole.to(BF16), state["weight"], state["bias"], state["grad"])
        dx = dx + state["grad_sum"].double()
        return whole, out, dx, dx, dw, db
    x, weight = state["x"].double(), state["weight"].double()
    rows, vocab = x.shape[0], weight.shape[0]
    train = case.get("train", True)
    if case["op"] == "ce":
        heat = 1.0
        labels = state["targets"][:, None]
        share = (labels >= 0).double()
        entropy = torch.zeros(rows, dtype=torch.float64, device="cuda")
    else:
        heat = case["temperature"]
        labels = state["indices"].long()
        soft = state["teacher"].double() / heat
        some = torch.isfinite(soft).any(1)
        soft[~some] = 0.0
        share = torch.softmax(soft, dim=1)
        share[~some] = 0.0
        entropy = torch.special.entr(share).sum(1)
    used = share.sum(1) > 0
    count = max(1, int(used.sum()))
    labels = labels.clamp_min(0)
    losses = torch.zeros(rows, dtype=torch.float64, device="cuda")
    dx = torch.zeros_like(x) if train else None
    dw = torch.zeros_like(weight) if train else None
    for lo in range(0, rows, 512):
        piece = slice(lo, min(rows, lo + 512))
        log_q = torch.log_softmax(x[piece] @ weight.T / heat, dim=1)
        cross = -(share[piece] * log_q.gather(1, labels[piece])).sum(1)
        losses[piece] = heat * heat * (cross - entropy[piece])
        if train:
            slope = log_q.exp_()
            slope.scatter_add_(1, labels[piece], -share[piece])
            slope *= (heat / count) * used[piece, None]
            dx[piece] = slope @ weight
            dw += slope.T @ x[piece]
    if not train:
        return losses
    return losses.sum() / count, dx, dw
