"""Measured cases of the vocabulary operators: the teacher's top logits, the distillation from them and the linear cross
entropy, each in a plain form of elementary torch operations (``own`` false) and through the framework (``own`` true).

Two regimes stand beside each other, as the framework's users have them: token rows over a large vocabulary, and dense
depth classification, where every pixel is a row and the depth bins are the classes (640 x 192 images, batch 12, and
their quarter resolution).
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100


def listed():
    return [
        # --- linear cross entropy: hidden [rows, dim] x weight [vocab, dim] -> loss (and gradients)
        # a handful of tokens through a small float32 head: pure latency
        _ce("ce_tokens5_v1003_f32", 5, 1003, 192, "f32", train=False),
        # scoring one short prompt: every weight is read for sixteen rows
        _ce("ce_tokens16_v65536_bf16", 16, 65536, 2048, "bf16", train=False),
        # a training step's whole batch of tokens over a large vocabulary
        _ce("ce_train8192_v131072_bf16", 8192, 131072, 4096, "bf16"),
        # odd sizes everywhere, half precision, a seventh of the targets padded
        _ce("ce_train2011_v32003_f16", 2011, 32003, 1000, "f16"),
        # float32 training, as the framework's losses run by default
        _ce("ce_train1536_v10007_f32", 1536, 10007, 512, "f32"),
        # depth bins at quarter resolution of a batch of 12: few classes, very many rows, a bias, pixels without ground truth
        _ce("ce_bins_b12_quarter_bf16", 12 * 48 * 160, 128, 256, "bf16", bias=True),
        # --- distillation from a teacher's top logits
        # validation of a few tokens, row by row
        _kd("kd_tokens7_v32000_f32", 7, 32000, 16, "f32", tail=False, temperature=1.0, train=False),
        # a training step's whole batch of tokens, the teacher's remaining mass as one class
        _kd("kd_train4096_v131072_bf16", 4096, 131072, 64, "bf16", tail=True, temperature=1.0),
        # every pixel of a batch of 12 at full resolution, teacher and student share 128 depth bins
        _kd("kd_bins_b12_full_bf16", 12 * 192 * 640, 128, 8, "bf16", tail=True, temperature=2.0),
        # --- the teacher's top logits themselves
        # one token being answered
        _top("top_token1_v50021_bf16", 1, 50021, 32, "bf16"),
        # the teacher's pass over the same training batch
        _top("top_train4096_v131072_bf16", 4096, 131072, 64, "bf16"),
        # the teacher's depth bins at half resolution
        _top("top_bins_b12_half_f16", 12 * 96 * 320, 96, 8, "f16"),
    ]


def _ce(name, rows, vocab, dim, dtype, train=True, bias=False):
    case = {"op": "ce", "rows": rows, "vocab": vocab, "dim": dim, "dtype": dtype, "train": train, "bias": bias}
    return dict(case, name=name) if name else case


def _kd(name, rows, vocab, k, dtype, tail, temperature, train=True, padded=0):
    case = {"op": "kd", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype, "tail": tail, "temperature": temperature,
            "train": train, "padded": padded}
    return dict(case, name=name) if name else case


def _top(name, rows, vocab, k, dtype):
    case = {"op": "top", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype}
    return dict(case, name=name) if name else case


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm; odd about as often as even."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["ce", "kd", "top"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "ce":
        train = rng.random() < 0.75
        limit = 2.0 ** 36 if dtype == "f32" else 2.0 ** 39
        while True:
            rows, vocab, dim = _spread(rng, 1, 65536), _spread(rng, 64, 131072), _spread(rng, 32, 4096)
            if rng.random() < 0.5:                      # most models' widths are multiples of 64
                dim = max(64, dim // 64 * 64)
            if float(rows) * vocab * dim <= limit and rows * vocab <= 2 ** 30:
                return _ce(None, rows, vocab, dim, dtype, train=train, bias=rng.random() < 0.4)
    while True:
        rows, vocab = _spread(rng, 1, 12 * 192 * 640), _spread(rng, 64, 131072)
        if rows * vocab * SIZE[dtype] <= 2 ** 29:
            break
    k = min(vocab, _spread(rng, 1, 128))
    if op == "top":
        return _top(None, rows, vocab, k, dtype)
    padded = rng.choice([0, 0, rng.randint(1, 40)])     # classes behind the last one, at minus infinity
    return _kd(None, rows, vocab, min(k, vocab - padded), dtype, tail=rng.random() < 0.5,
               temperature=rng.choice([1.0, 1.0, 2.0, 3.5]), train=rng.random() < 0.75, padded=padded)


# ---------------------------------------------------------------------- inputs
def _classes(rows, vocab, gen):
    """Logits as networks produce them: noise over a large vocabulary, a noisy peak over ordered depth bins."""
    if vocab > 1024:
        return torch.randn(rows, vocab, generator=gen, device=DEVICE).mul_(2.5)
    centre = torch.rand(rows, 1, generator=gen, device=DEVICE) * vocab
    width = 2.0 + 0.06 * vocab
    bins = torch.arange(vocab, device=DEVICE, dtype=torch.float32)
    x = (bins - centre).div_(width).square_().mul_(-0.5).clamp_(min=-9.0)
    return x.add_(torch.randn(rows, vocab, generator=gen, device=DEVICE).mul_(0.4))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    rows, vocab = case["rows"], case["vocab"]
    state = dict(case)
    if case["op"] == "ce":
        dim = case["dim"]
        weight = torch.randn(vocab, dim, generator=gen, device=DEVICE).mul_(2.5 / math.sqrt(dim))
        target = torch.randint(vocab, (rows,), generator=gen, device=DEVICE)
        hidden = torch.randn(rows, dim, generator=gen, device=DEVICE)
        for i in range(0, rows, 1 << 16):               # the network already leans towards the right class
            hidden[i:i + (1 << 16)].add_(weight[target[i:i + (1 << 16)]], alpha=1.0)
        if rows > 8:
            target[torch.rand(rows, generator=gen, device=DEVICE) < 1 / 7] = IGNORE
        bias = torch.randn(vocab, generator=gen, device=DEVICE).mul_(0.5).to(dtype) if case["bias"] else None
        state.update(hidden=hidden.to(dtype), weight=weight.to(dtype), target=target, bias=bias)
        if case["train"]:
            state["upstream"] = torch.ones((), device=DEVICE)
            for name in ("hidden", "weight", "bias"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    x = _classes(rows, vocab, gen)
    if case["op"] == "kd":
        k, padded, t = case["k"], case["padded"], case["temperature"]
        live = vocab - padded
        step = live // k                                # distinct classes: one of every step, in a shuffled order
        first = torch.randint(step, (rows, 1), generator=gen, device=DEVICE)
        order = torch.randperm(k, generator=gen, device=DEVICE)
        index = (first + order * step).to(torch.int32)
        value = torch.randn(rows, k, generator=gen, device=DEVICE).mul_(1.5).add_(6.0).sort(dim=1, descending=True).values.to(dtype)
        x.scatter_add_(1, index.long(), value.float().mul(0.5))     # the student follows the teacher halfway
        if padded:
            x[:, live:] = -math.inf
        seen = torch.logsumexp(value.double() / t, dim=1)
        share = torch.rand(rows, generator=gen, device=DEVICE, dtype=torch.float64).mul_(0.3).add_(0.02)
        lse = (seen - torch.log1p(-share)).float()      # the teacher's whole log sum: 2..32 % of the mass is elsewhere
        weights = (torch.rand(rows, generator=gen, device=DEVICE) > 0.1).float()
        state.update(logits=x.to(dtype), values=value, indices=index, lse=lse if case["tail"] and live > k else None,
                     weights=weights if rows > 8 else None)
        if case["train"]:
            state["upstream"] = torch.ones((), device=DEVICE)
            state["logits"].requires_grad_(True)
        return state
    state["logits"] = x.to(dtype)
    return state


# ---------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"ce": _plain_ce, "kd": _plain_kd, "top": _plain_top}[state["op"]](state)


def _run_own(s):
    from mde_amd.vocab_losses import linear_cross_entropy, top_logits, topk_distillation_loss
    if s["op"] == "top":
        top = top_logits(s["logits"], s["k"])
        return top.values, top.indices, top.lse
    if s["op"] == "ce":
        reduction = "mean" if s["train"] else "none"
        loss = linear_cross_entropy(s["hidden"], s["weight"], s["target"], s["bias"], ignore_index=IGNORE, reduction=reduction)
        leaves = [s["hidden"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else [])
    else:
        reduction = "mean" if s["train"] else "none"
        loss = topk_distillation_loss(s["logits"], s["values"], s["indices"], s["lse"], temperature=s["temperature"],
                                      weights=s["weights"], reduction=reduction)
        leaves = [s["logits"]]
    if not s["train"]:
        return loss
    return (loss.detach(),) + torch.autograd.grad(loss, leaves, s["upstream"])


def _log_sum(z):
    top = z.max(dim=1, keepdim=True).values
    return (top + (z - top).exp_().sum(dim=1, keepdim=True).log_())


def _plain_ce(s):
    hidden, weight, target = s["hidden"].float(), s["weight"].float(), s["target"]
    z = hidden @ weight.t()
    if s["bias"] is not None:
        z += s["bias"].float()
    kept = target != IGNORE
    at = target.clamp(min=0).unsqueeze(1)
    lse = _log_sum(z)
    row = ((lse - z.gather(1, at)).squeeze(1) * kept)
    if not s["train"]:
        return row
    count = kept.sum().clamp(min=1)
    g = z.sub_(lse).exp_()
    g.scatter_add_(1, at, torch.full_like(lse, -1.0))
    g.mul_((kept.float() / count * s["upstream"]).unsqueeze(1))
    out = [row.sum() / count, (g @ weight).to(s["hidden"].dtype), (g.t() @ hidden).to(s["weight"].dtype)]
    if s["bias"] is not None:
        out.append(g.sum(dim=0).to(s["bias"].dtype))
    return tuple(out)


def _plain_kd(s):
    t = s["temperature"]
    z = s["logits"].float() / t
    at = s["indices"].long()
    v = s["values"].double() / t
    rest = s["lse"] is not None
    if rest:
        q = (v - s["lse"].double().unsqueeze(1)).exp()
        tail = (1.0 - q.sum(dim=1, keepdim=True)).clamp(min=0)
    else:
        q = (v - v.max(dim=1, keepdim=True).values).exp()
        q = q / q.sum(dim=1, keepdim=True)
    q32 = q.float()
    lse = _log_sum(z)
    row = (q * q.log()).sum(dim=1, keepdim=True).float() - (q32 * (z.gather(1, at) - lse)).sum(dim=1, keepdim=True)
    if rest:
        elsewhere = _log_sum(z.scatter(1, at, -math.inf))
        row += (tail * tail.log()).float() - tail.float() * (elsewhere - lse)
    row = row.squeeze(1) * (t * t)
    weights = s["weights"] if s["weights"] is not None else torch.ones_like(row)
    row = row * weights
    if not s["train"]:
        return row
    total = weights.sum()
    scale = (weights * (t / total) * s["upstream"]).unsqueeze(1)
    p = z.sub_(lse).exp_()
    if rest:
        g = p * (1.0 - tail.float() * (lse - elsewhere).exp())
        g.scatter_(1, at, p.gather(1, at) * (q.sum(dim=1, keepdim=True) + tail).float() - q32)
    else:
        g = p.scatter_add_(1, at, -q32)
    return row.sum() / total, g.mul_(scale).to(s["logits"].dtype)


def _plain_top(s):
    logits, k = s["logits"], s["k"]
    values, indices, lse = [], [], []
    piece = max(1, (1 << 27) // s["vocab"])
    for i in range(0, s["rows"], piece):
        z = logits[i:i + piece].float()
        order = z.sort(dim=1, descending=True, stable=True)
        values.append(order.values[:, :k].to(logits.dtype))
        indices.append(order.indices[:, :k].to(torch.int32))
        lse.append(_log_sum(z).squeeze(1))
    return torch.cat(values), torch.cat(indices), torch.cat(lse)


# ---------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    if case["op"] == "ce" and float(case["rows"]) * case["vocab"] * case["dim"] > 6e12:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return {"ce": _exact_ce, "kd": _exact_kd, "top": _exact_top}[case["op"]](s)


def _pieces(s, elements=1 << 27):
    step = max(1, elements // s["vocab"])
    return [slice(i, min(i + step, s["rows"])) for i in range(0, s["rows"], step)]


def _exact_ce(s):
    weight = s["weight"].double()
    bias = s["bias"].double() if s["bias"] is not None else torch.zeros((), dtype=torch.float64, device=DEVICE)
    losses, grad_hidden = [], []
    grad_weight, grad_bias = torch.zeros_like(weight), torch.zeros(s["vocab"], dtype=torch.float64, device=DEVICE)
    count = max(int((s["target"] != IGNORE).sum()), 1)
    for part in _pieces(s):
        hidden, target = s["hidden"][part].double(), s["target"][part]
        logp = torch.log_softmax(torch.mm(hidden, weight.T) + bias, dim=1)
        live = torch.nonzero(target != IGNORE).squeeze(1)
        loss = torch.zeros(len(target), dtype=torch.float64, device=DEVICE)
        loss[live] = -logp[live, target[live]]
        losses.append(loss)
        if s["train"]:
            delta = torch.zeros_like(logp)
            delta[live] = logp[live].exp()
            delta[live, target[live]] -= 1.0
            delta /= count
            grad_hidden.append(torch.mm(delta, weight))
            grad_weight += torch.mm(delta.T.contiguous(), hidden)
            grad_bias += delta.sum(dim=0)
    losses = torch.cat(losses)
    if not s["train"]:
        return losses
    out = (losses.sum() / count, torch.cat(grad_hidden), grad_weight)
    return out + (grad_bias,) if s["bias"] is not None else out


def _exact_kd(s):
    t = s["temperature"]
    weights = s["weights"].double() if s["weights"] is not None else torch.ones(s["rows"], dtype=torch.float64, device=DEVICE)
    losses, grads = [], []
    for part in _pieces(s):
        z, at, w = s["logits"][part].double() / t, s["indices"][part].long(), weights[part]
        teacher = s["values"][part].double() / t
        logp = torch.log_softmax(z, dim=1)
        if s["lse"] is None:
            logq = torch.log_softmax(teacher, dim=1)
        else:
            logq = teacher - s["lse"][part].double().unsqueeze(1)
        kl = (logq.exp() * (logq - torch.gather(logp, 1, at))).sum(dim=1)
        grad = torch.exp(logp)
        if s["lse"] is not None:
            member = torch.zeros_like(logp, dtype=torch.bool).scatter_(1, at, True)
            logr = torch.logsumexp(logp.masked_fill(member, -math.inf), dim=1)
            mass = logq.exp().sum(dim=1)
            tail = torch.clamp(1.0 - mass, min=0.0)
            kl += torch.special.xlogy(tail, tail) - tail * logr
            own_share = grad * (mass + tail).unsqueeze(1)
            grad = torch.where(member, own_share, own_share - tail.unsqueeze(1) * torch.exp(logp - logr.unsqueeze(1)))
        grad.scatter_add_(1, at, -logq.exp())
        losses.append(kl * t * t * w)
        grads.append(grad * (t * w / weights.sum()).unsqueeze(1) if s["train"] else None)
    losses = torch.cat(losses)
    return (losses.sum() / weights.sum(), torch.cat(grads)) if s["train"] else losses


def _exact_top(s):
    values, indices, lse = [], [], []
    behind = torch.arange(s["vocab"] - 1, -1, -1, device=DEVICE)
    for part in _pieces(s, 1 << 26):
        logits = s["logits"][part]
        bits = logits.float().add(0.0).view(torch.int32).long()
        rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)      # orders as the values do
        best = torch.topk(rank * (1 << 20) + behind, s["k"], dim=1).values
        at = s["vocab"] - 1 - (best & ((1 << 20) - 1))
        values.append(torch.gather(logits, 1, at).double())
        indices.append(at.to(torch.int32))
        lse.append(torch.logsumexp(logits.double(), dim=1))
    return torch.cat(values), torch.cat(indices), torch.cat(lse)


# ---------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size, rows, vocab = SIZE[case["dtype"]], case["rows"], case["vocab"]
    if case["op"] == "ce":
        operands = (rows + vocab) * case["dim"] * size + (vocab * size if case["bias"] else 0)
        product = 2.0 * rows * vocab * case["dim"]
        if case["train"]:                               # logits and the two gradients; operands in, their gradients out
            return {"bytes": 2 * operands + 8 * rows + 4, "flops": 3 * product}
        return {"bytes": operands + 8 * rows + 4 * rows, "flops": product}
    table = rows * vocab * size
    if case["op"] == "kd":
        teacher = rows * (case["k"] * (size + 4) + 8)
        if case["train"]:
            return {"bytes": 2 * table + teacher + 4, "flops": 8.0 * rows * vocab}
        return {"bytes": table + teacher + 4 * rows, "flops": 4.0 * rows * vocab}
    return {"bytes": table + rows * (case["k"] * (size + 4) + 4), "flops": 4.0 * rows * vocab}
