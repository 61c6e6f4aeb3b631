"""Plain float64 CPU implementations of the losses over a set of classes (mde_amd.vocab_losses) for the tests, with the
error bounds that float32 arithmetic allows.  u = 2^-24 is float32's half step."""
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # smallest subnormal


def sum_error(vocab):
    """Relative error of a sum of `vocab` exponentials: at least 16 lanes add a share each one after the other, then a
    tree; the exponential itself (2 u) and its rescaling by a later maximum (3 u a tile) come on top."""
    return (vocab / 16 + 64) * U if vocab <= 2048 else (vocab / 256 * 2 + 128) * U


def finite_max(x):
    x = x[torch.isfinite(x)].abs()
    return float(x.max()) if x.numel() else 0.0


def exponent_error(x, temperature):
    """Absolute error of x / T as the kernels hold it: scaled by a rounded log2(e) / T, one rounding of the product and
    one of the difference to the maximum, which is at most twice as large; back to base e: 8 u of the largest."""
    return 8 * U * (finite_max(x) / temperature + 1)


def top_logits(x, k, temperature=1.0):
    x = x.double().cpu()
    order = torch.where(torch.isnan(x), torch.full_like(x, float("inf")), x)
    rank = torch.isnan(x)                                   # NaN above +inf: sort by (isnan, value), stable
    idx = torch.sort(order, dim=1, descending=True, stable=True).indices
    idx = torch.gather(idx, 1, torch.sort(torch.gather(rank.int(), 1, idx), dim=1, descending=True, stable=True).indices)
    idx = idx[:, :k]
    return torch.gather(x, 1, idx), idx, torch.logsumexp(x / temperature, dim=1)


def distill(x, values, indices, lse=None, temperature=1.0, weights=None):
    """(row losses, gradient of their plain sum, sizes of the gradient's terms), by the definition, row by row."""
    x, values = x.double().cpu(), values.double().cpu()
    indices = indices.cpu().long()
    rows, vocab = x.shape
    t = temperature
    loss = torch.zeros(rows, dtype=torch.float64)
    grad, size = torch.zeros_like(x), torch.zeros_like(x)
    for r in range(rows):
        w = 1.0 if weights is None else float(weights[r])
        if w == 0.0:
            continue
        z, v = x[r] / t, values[r] / t
        if bool(((indices[r] < 0) | (indices[r] >= vocab)).any()):
            loss[r], grad[r] = float("nan"), float("nan")
            continue
        norm = torch.logsumexp(v, 0) if lse is None else lse[r].double().cpu()
        if bool(norm == -float("inf")) or bool(torch.logsumexp(z, 0) == -float("inf")):
            continue
        logp, logq = torch.log_softmax(z, 0), v - norm
        q = logq.exp()
        on = q != 0
        loss[r] = (q[on] * (logq[on] - logp[indices[r]][on])).sum()
        share = torch.zeros(vocab, dtype=torch.float64).index_add_(0, indices[r], q)
        member = torch.zeros(vocab, dtype=torch.bool)
        member[indices[r]] = True
        rest, qt = ~member, torch.zeros((), dtype=torch.float64)
        other = torch.logsumexp(logp[rest], 0) if bool(rest.any()) else torch.tensor(-float("inf"))
        mass = q.sum()
        tail = torch.zeros(vocab, dtype=torch.float64)
        if lse is not None and bool(other != -float("inf")):
            qt = torch.clamp(1 - mass, min=0)
            if bool(qt > 0):
                loss[r] += qt * (qt.log() - other)
                tail[rest] = qt * (logp[rest] - other).exp()
        p = logp.exp()
        grad[r] = w * t * ((mass + qt) * p - share - tail)
        size[r] = abs(w) * t * ((mass + qt) * p + share + tail + (1 if lse is not None else 0) * (logp - other).exp() * rest
                                if bool(other != -float("inf")) else (mass + qt) * p + share)
        loss[r] *= w * t * t
    return loss, grad, size


def linear_ce(hidden, weight, target, bias=None, ignore_index=-100, z_loss=0.0, device="cpu"):
    """(row losses, lse, logits, dS = derivative of every row's loss), NaN rows for targets outside the vocabulary."""
    h, w = hidden.double().to(device), weight.double().to(device)
    target = target.to(device).long()
    z = h @ w.T
    if bias is not None:
        b = bias.double().to(device)
        z = torch.where(b == -float("inf"), b, z + b)
    lse = torch.logsumexp(z, 1)
    live = target != ignore_index
    bad = live & ((target < 0) | (target >= w.shape[0]))
    at = target.clamp(0, w.shape[0] - 1)
    empty = lse == -float("inf")
    loss = lse - torch.gather(z, 1, at[:, None])[:, 0] + z_loss * lse * lse
    loss = torch.where(live & ~empty, loss, torch.zeros_like(loss))
    loss = torch.where(bad, torch.full_like(loss, float("nan")), loss)
    ds = (z - lse[:, None]).exp() * (1 + 2 * z_loss * lse[:, None])
    ds[torch.arange(len(target), device=device), at] -= 1
    ds = torch.where((live & ~empty)[:, None], ds, torch.zeros_like(ds))
    ds = torch.where(bad[:, None], torch.full_like(ds, float("nan")), ds)
    return loss, lse, z, ds
