"""Float64 definitions of the losses over a set of classes, row by row, each with a bound on what float32 arithmetic may add.

The bounds know no size of a logit, only its distance d = (max - x) / T to its row's maximum: a softmax does not change when
all logits of a row move together, and neither may its error.  u = 2^-24 is float32's half step.

An exponential of a kernel is off by (relative, first order)
    5 u d       the scale log2(e) / T, the product and the difference are each rounded once, where the running maximum
                moved and where parts are joined a second time (the distances of one class's moves sum to at most d)
    R u         the product is formed before the difference: its rounding, at most R = min(64, u |max| log2(e) / T) in the
                exponent, is taken out again; R is what the exponent's own rounding sees of it.  Above |max| log2(e) / T =
                2^31 the kernels scale by a power of two and R is 0
    (5 + 3 J) u the exponential itself (one step of the last place), its correction, and J changes of the maximum
and a sum of them by A u for A additions one after the other.
"""
import math

import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # smallest subnormal
INF = float("inf")


def stream_sum(vocab):
    """J and A of the logits' programs: groups of at least 2048 classes per block, at most 10 additions a thread each, then
    lanes, waves and segments; a short row is one group."""
    groups = -(-vocab // 2048)
    return (13 * groups + 48) * U


def tile_sum(vocab):
    """J and A of the linear cross entropy: at most 64 additions a lane, then halves, waves, and tiles of at least 128 classes
    one after the other."""
    return (5 * -(-vocab // 128) + 128) * U


def log_sum_error(z, sum_error, shift=None):
    """Bound on the error of log sum exp z over the last dimension, z = logits / T in float64, -infinity masked.  shift: the
    largest |max| of the row in the kernel's scale, for R."""
    top = z.max(-1, keepdim=True).values
    d = torch.where(z == -INF, torch.zeros_like(z), top - z)
    p = torch.where(z == -INF, torch.zeros_like(z), (-d).exp())
    p = p / p.sum(-1, keepdim=True)
    y = (top[..., 0].abs() if shift is None else shift) * 1.4427
    r = torch.where(y < 2.0 ** 31, (y * U).clamp(max=64.0), torch.zeros_like(y))
    return 5 * U * (p * d).sum(-1) + (r + 8 + 4 * math.log(z.shape[-1] + 1)) * U + sum_error   # the logarithm, and sums with it


def log_sum(z):
    return torch.logsumexp(z.double(), -1)


def close(got, want, tol, what):
    want = want.double().cpu()
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what + ": infinities"
    on = torch.isfinite(want)
    tol = (torch.zeros_like(want) + tol)[on]
    off = (got[on] - want[on]).abs()
    assert bool((off <= tol).all()), "%s: off by %.3g, allowed %.3g" % (
        what, off[(off - tol).argmax()], tol[(off - tol).argmax()])


def distill(x, values, indices, lse=None, temperature=1.0):
    """Row losses and the gradient of their sum, with the bounds of both; every row finite, indices of a row distinct."""
    t = temperature
    z, v, at = x.double() / t, values.double() / t, indices.long()
    vocab = z.shape[1]
    top = z.max(1, keepdim=True).values
    dist = torch.where(z == -INF, torch.zeros_like(z), top - z)
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    e_all = log_sum_error(z, stream_sum(vocab))[:, None]
    # (float64 has no room for the logarithm of k beside a value of 1e30)
    logq = torch.log_softmax(v - v.max(1, keepdim=True).values, 1) if lse is None else v - lse.double()[:, None]
    q = logq.exp()
    mass = q.sum(1, keepdim=True)
    k = values.shape[1]
    e_q = (16 + k / 8) * U                                # a q, and a lane's sum of them
    step = logp.gather(1, at)
    loss = (q * (logq - step)).sum(1)
    bound = (q * ((logq.abs() + step.abs()) * 8 * U + 3 * U * dist.gather(1, at) + e_all + e_q * ((logq - step).abs() + 1))).sum(1)
    grad = p * mass
    size = grad * (5 * U * dist + e_all + e_q + 8 * U)
    if lse is not None:
        member = torch.zeros_like(z, dtype=torch.bool).scatter_(1, at, True)
        zr = z.masked_fill(member, -INF)
        e_rest = log_sum_error(zr, stream_sum(vocab))[:, None]
        logr = torch.logsumexp(logp.masked_fill(member, -INF), 1, keepdim=True)
        qt = (1 - mass).clamp(min=0)
        e_t = e_q * mass + U                              # absolute, of 1 - sum q
        loss = loss + (qt * (qt.log() - logr))[:, 0]
        bound = bound + (e_t * ((qt.log() - logr).abs() + 1) + qt * (e_all + e_rest + 8 * U * (qt.log().abs() + logr.abs())))[:, 0]
        share = torch.where(member, torch.zeros_like(p), (logp - logr).exp())
        grad = p * (mass + qt) - qt * share
        size = torch.where(member, p * (mass + qt) * (5 * U * dist + e_all + e_q + e_t + 8 * U),
                           share * (logr.exp() * (mass + qt) * (e_all + e_rest + e_q + e_t + 16 * U) + e_t + qt * 8 * U)
                           + grad.abs() * (5 * U * dist + e_rest + 8 * U))
    grad = grad.scatter_add(1, at, -q)
    size = size.scatter_add(1, at, q * e_q) + 8 * U * grad.abs()
    return loss * t * t, 2 * bound * t * t, grad * t, 2 * size * t


def linear_ce(z, target, z_loss=0.0):
    """Row losses, derivatives of their sum by the logits, and the bounds of both, for logits that float32 holds exactly."""
    z = z.double()
    rows = torch.arange(z.shape[0])
    top = z.max(1, keepdim=True).values
    dist = torch.where(z == -INF, torch.zeros_like(z), top - z)
    lse = torch.logsumexp(z, 1)
    e = log_sum_error(z, tile_sum(z.shape[1]))
    # lse - z_target without the cancellation of their size
    above = torch.logsumexp(z - top, 1)
    gap = (top[:, 0] - z[rows, target])
    loss = above + gap + z_loss * lse * lse
    bound = e + 2 * U * gap.abs() + 4 * U * above.abs() + 4 * U * loss.abs() + z_loss * 2 * (lse.abs() + 1) * (e + 4 * U * lse.abs())
    slope = (1 + 2 * z_loss * lse)[:, None]
    p = (z - top - above[:, None]).exp()
    ds = p * slope
    err = ds.abs() * (5 * U * dist + e[:, None] + 16 * U)
    ds[rows, target] -= 1
    err[rows, target] += 4 * U
    return loss, 2 * bound, ds, 2 * err
