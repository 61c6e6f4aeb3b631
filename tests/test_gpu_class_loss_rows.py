"""The losses over a set of classes, row by row: bounds that know the distances within a row and not its size
(tests/class_loss_bounds.py), rows that do not feel their neighbours, and calls that are refused."""
import math

import pytest
import torch

import class_loss_bounds as B

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def spacing(offset, dtype):
    """Distance of the type's values on either side of `offset`, the wider one."""
    return 2.0 ** math.floor(math.log2(abs(offset) * (1 - 1e-9))) * torch.finfo(dtype).eps * 2 if offset else 0.0


def shifted(rows, vocab, offset, dtype, seed):
    """Logits around `offset` that the type holds exactly."""
    step = max(2.0 ** -6, spacing(offset, dtype))
    x = torch.round(torch.randn(rows, vocab, generator=gen(seed), dtype=torch.float64) * 2.5 / step).clamp(-50, 50) * step
    got = (x + offset).to(dtype)
    assert torch.equal(got.double(), x + offset) or dtype != torch.float32 or step > 64
    return got


def teacher(rows, vocab, k, seed, dtype, offset=0.0):
    g = gen(seed)
    at = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    step = max(2.0 ** -6, spacing(offset, dtype))
    v = torch.round(torch.randn(rows, k, generator=g, dtype=torch.float64) * 1.5 / step) * step + offset
    return v.to(dtype), at


def check_distill(x, val, idx, lse, t):
    import mde_amd.vocab_losses as L
    loss, ltol, grad, gtol = B.distill(x, val, idx, lse, t)
    a = x.to(DEV).requires_grad_(True)
    out = L.topk_distillation_loss(a, val.to(DEV), idx.to(DEV), None if lse is None else lse.to(DEV), temperature=t, reduction="none")
    B.close(out, loss, ltol, "row losses")
    up = torch.randn(x.shape[0], generator=gen(7))
    (got,) = torch.autograd.grad(out, a, up.to(DEV))
    want = grad * up.double()[:, None]
    flushed = 2.0 ** -125 * t * up.double().abs()[:, None]     # exponentials below 2^-126 come out as 0
    B.close(got, want, gtol * up.double().abs()[:, None] + (B.HALF_STEP[x.dtype] + 4 * B.U) * want.abs() + B.TINY[x.dtype] + flushed,
            "gradient")


# ------------------------------------------------------------------ a softmax does not feel its row's offset
SMALL = torch.tensor(0.01).item()                           # a temperature is a float32 in the library
SHIFTS = [(0.0, 1.0), (1000.0, 1.0), (-10000.0, 1.0), (0.0, SMALL), (-1.0e9, 1.0), (-1.0e9, 40.0), (-1e30, 1.0)]
SHAPES = [(5, 9, 4), (7, 128, 8), (6, 200, 20), (5, 300, 12), (4, 900, 33), (3, 2048, 9), (3, 5000, 16), (2, 70001, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,t", SHIFTS)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_does_not_feel_an_offset_of_the_students_logits(offset, t, tail, dtype):
    if dtype == torch.float16 and abs(offset) > 6e4:
        offset = math.copysign(6e4, offset)
    for rows, vocab, k in SHAPES:
        x = shifted(rows, vocab, offset, dtype, vocab)
        val, idx = teacher(rows, vocab, k, vocab + k, torch.float32)
        val = val * min(t, 1.0)
        lse = (torch.logsumexp(val.double() / t, 1) + 0.1).float() if tail else None
        check_distill(x, val, idx, lse, t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,t", SHIFTS)
def test_distillation_does_not_feel_an_offset_of_the_teachers_values(offset, t, dtype):
    if dtype == torch.float16 and abs(offset) > 6e4:
        offset = math.copysign(6e4, offset)
    for rows, vocab, k in SHAPES:
        x = shifted(rows, vocab, 0.0, torch.float32, vocab) * min(t, 1.0)
        val, idx = teacher(rows, vocab, k, vocab + k, dtype, offset)
        check_distill(x, val, idx, None, t)
        if abs(offset) <= 1e4:                              # above, a float32 log sum holds no digit of the teacher's rest
            check_distill(x, val, idx, (torch.logsumexp(val.double() / t, 1) + 0.1).float(), t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [torch.tensor(1e-4).item(), 1e4])
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_at_the_extreme_temperatures(t, tail, dtype):
    for rows, vocab, k in SHAPES:
        x = shifted(rows, vocab, 0.0, dtype, vocab + 5)
        val, idx = teacher(rows, vocab, k, vocab + 6, torch.float32)
        lse = None
        if tail:                                            # the whole sum over some more classes like the k, as float32 holds it
            z = val.double() / t
            lse = (z.max(1).values + torch.logsumexp(z - z.max(1, keepdim=True).values, 1) + 0.1).float()
            if float(lse.abs().max()) > 3e3:                # no digit left for what the k leave over: only rows that are whole
                continue
        check_distill(x, val, idx, lse, t)


def exact_operands(rows, vocab, dim, offset, dtype, seed):
    """hidden, weight, bias whose logits float32 holds exactly whatever the order of the sums: small whole numbers times a power
    of two, few of a row's features not zero."""
    g = gen(seed)
    step = max(0.25, spacing(offset, torch.float32))
    live = torch.rand(dim, generator=g) < 40.0 / dim
    h = torch.randint(-1, 2, (rows, dim), generator=g).double() * live
    w = torch.randint(-3, 4, (vocab, dim), generator=g).double() * step
    b = torch.full((vocab,), offset, dtype=torch.float64)
    bias = b.to(dtype)
    z = h @ w.T + bias.double()
    assert torch.equal(z.float().double(), z)
    return h.to(dtype), w.to(dtype), bias, z, torch.randint(vocab, (rows,), generator=g)


def check_linear_ce(h, w, b, t, z, z_loss=0.0):
    import mde_amd.vocab_losses as L
    dtype, rows, vocab = h.dtype, h.shape[0], w.shape[0]
    loss, ltol, ds, dtol = B.linear_ce(z, t, z_loss)
    leaves = [x.to(DEV).requires_grad_(True) for x in (h, w, b)]
    out = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2], z_loss=z_loss, reduction="none")
    B.close(out, loss, ltol, "row losses")
    up = torch.randn(rows, generator=gen(8)).double()
    got = torch.autograd.grad(out, leaves, up.float().to(DEV), retain_graph=True)
    mean = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2], z_loss=z_loss)
    total = float(loss.sum())
    assert abs(float(mean.detach()) - total / rows) <= float(ltol.sum()) / rows + 4 * B.U * abs(total) / rows
    got_mean = torch.autograd.grad(mean, leaves, torch.tensor(3.0, device=DEV))
    for grads, u in ((got, up.float().double()), (got_mean, torch.full((rows,), 3.0 / rows, dtype=torch.float64))):
        u = u[:, None]
        d, half = ds * u, B.HALF_STEP[dtype]
        largest = float(u.abs().max()) * (1 + 2 * z_loss * float(B.log_sum(z).abs().max()))
        floor = largest * 2.0 ** -36 if dtype == torch.float16 else 0.0     # its smallest step under a scale of 2^11 at least
        err = dtol * u.abs() + d.abs() * half * 1.01 + floor
        n = max(rows, vocab) + 4
        h6, w6 = h.double(), w.double()
        for name, g, want, tol in (
                ("grad hidden", grads[0], d @ w6, err @ w6.abs() + n * B.U * (d.abs() @ w6.abs())),
                ("grad weight", grads[1], d.T @ h6, err.T @ h6.abs() + n * B.U * (d.abs().T @ h6.abs())),
                ("grad bias", grads[2], d.sum(0), err.sum(0) + n * B.U * d.abs().sum(0))):
            B.close(g, want, tol + (half + 8 * B.U) * want.abs() + B.TINY[dtype], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0.0, 1024.0, -8192.0, -2.0 ** 30, -2.0 ** 100])
@pytest.mark.parametrize("rows,vocab,dim", [
    (5, 40, 24), (12, 500, 3000), (40, 3000, 64), (64, 700, 200), (200, 300, 96), (130, 1000, 40), (1030, 4000, 330),
    (70, 9001, 1003), (2100, 8200, 128)])
def test_linear_cross_entropy_does_not_feel_an_offset_of_the_logits(rows, vocab, dim, offset, dtype):
    """Latency sizes, logits in parts of the features, thin, narrow, small and large tiles, float32 directly and by planes."""
    if dtype == torch.float16 and abs(offset) > 6e4:
        offset = -2.0 ** 15
    h, w, b, z, t = exact_operands(rows, vocab, dim, offset, dtype, rows + vocab)
    check_linear_ce(h, w, b, t, z)


# ------------------------------------------------------------------ masks of the type's lowest value
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_of_lowest_values(tail, dtype):
    """Classes masked by the type's lowest value, and rows that hold nothing else: uniform ones."""
    low = torch.finfo(dtype).min
    for rows, vocab, k in SHAPES:
        x = shifted(rows, vocab, 0.0, dtype, vocab + 3)
        live = max(k, vocab // 2)
        x[:, live:] = low
        val, idx = teacher(rows, live, k, vocab + 4, torch.float32)
        lse = (torch.logsumexp(val.double(), 1) + 0.1).float() if tail and live > k else None
        check_distill(x, val, idx, lse, 1.0)
        x[:] = low
        lse = (torch.logsumexp(val.double(), 1) + 0.1).float() if tail and vocab > k else None
        check_distill(x, val, idx, lse, 1.0)
        if not tail:                                        # a teacher whose k are all masked alike
            check_distill(shifted(rows, vocab, 0.0, dtype, vocab), torch.full((rows, k), low, dtype=dtype), idx, None, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, SMALL, 40.0])
def test_top_logits_log_sums_row_by_row(temperature, dtype):
    import mde_amd.vocab_losses as L
    low = torch.finfo(dtype).min
    for vocab in (9, 60, 128, 300, 900, 2048, 5000, 70001):
        x = shifted(8, vocab, 0.0, dtype, vocab)
        x[1] = low
        x[2, vocab // 2:] = low
        x[3, 4:] = -INF
        x[4] += 500
        x[5] -= 2000
        z = x.double() / temperature
        want = torch.logsumexp(z - z.max(1, keepdim=True).values, 1) + z.max(1).values
        got = L.top_logits(x.to(DEV), 4, temperature).lse
        # the largest / T is rounded twice, its sum with the logarithm once; beyond float32 the sum is infinite
        beyond = want.abs() > torch.finfo(torch.float32).max
        assert torch.equal(got.cpu()[beyond], torch.full_like(got.cpu()[beyond], -INF))
        tol = B.log_sum_error(z, B.stream_sum(vocab)) + 4 * B.U * want.abs()
        B.close(got.cpu()[~beyond], want[~beyond], tol[~beyond], "log sum")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(5, 40, 24), (12, 500, 3000), (40, 3000, 64), (200, 300, 96), (70, 9001, 1003), (1500, 5000, 512)])
def test_linear_cross_entropy_of_lowest_biases(rows, vocab, dim, dtype):
    """Beside other classes such a bias masks as -infinity does, to the bit; a row of nothing else is uniform."""
    import mde_amd.vocab_losses as L
    low = torch.finfo(dtype).min
    h, w, b, _, t = exact_operands(rows, vocab, dim, 0.0, dtype, 11)
    masked = torch.arange(vocab) % 3 == 1
    t[masked[t]] -= 1
    outs = []
    for value in (low, -INF):
        b2 = torch.where(masked, torch.full_like(b, value), b)
        leaves = [x.to(DEV).requires_grad_(True) for x in (h, w, b2)]
        rows_out = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2], reduction="none")
        mean = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2])
        outs.append([rows_out.detach(), mean.detach()] + list(torch.autograd.grad(mean, leaves)))
    for a, c in zip(*outs):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, c)
    if dtype == torch.float16:
        return                                              # its lowest value is an ordinary logit
    b[:] = low
    z = b.double().expand(rows, vocab).clone()
    assert torch.equal((z + h.double() @ w.double().T).float().double(), z)
    check_linear_ce(h, w, b, t, z)


@pytest.mark.parametrize("weighted", [False, True])
def test_the_mean_is_the_sum_over_its_divisor(weighted):
    import mde_amd.vocab_losses as L
    for rows, vocab, k in ((7000, 60, 5), (300, 3000, 8)):
        x = shifted(rows, vocab, 0.0, torch.float32, rows).to(DEV)
        val, idx = (a.to(DEV) for a in teacher(rows, vocab, k, 5, torch.float32))
        weights = torch.rand(rows, generator=gen(6)).to(DEV) if weighted else None
        each, total, mean = (L.topk_distillation_loss(x, val, idx, weights=weights, reduction=r).double() for r in ("none", "sum", "mean"))
        count = weights.double().sum() if weighted else rows
        assert float((total - each.sum()).abs()) <= B.U * float(each.sum())
        assert float((mean - each.sum() / count).abs()) <= B.U * float(each.sum() / count)
        h, w, b, _, t = exact_operands(rows, vocab, 24, 0.0, torch.float32, 12)
        t[::5] = -100
        args = (h.to(DEV), w.to(DEV), t.to(DEV), b.to(DEV))
        each, total, mean = (L.linear_cross_entropy(*args, reduction=r).double() for r in ("none", "sum", "mean"))
        count = int((t != -100).sum())
        assert float((total - each.sum()).abs()) <= B.U * float(each.sum())
        assert float((mean - each.sum() / count).abs()) <= B.U * float(each.sum() / count)


# ------------------------------------------------------------------ rows beside other rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [12, 60, 128, 250, 500, 1000])
def test_a_row_has_the_same_bits_alone_and_beside_any_other(vocab, dtype):
    """Up to eight rows share a wave: ordinary ones beside rows whose rest class vanishes, is empty or masked, that are not
    looked at, repeat an index or hold a NaN."""
    import mde_amd.vocab_losses as L
    rows, k = 16, 5
    x = shifted(rows, vocab, 0.0, dtype, vocab + 1)
    val, idx = teacher(rows, vocab, k, vocab + 2, torch.float32)
    lse = (torch.logsumexp(val.double(), 1) + 0.1).float()
    weights = torch.ones(rows)
    at = torch.arange(rows)[:, None]
    x[at, idx[:, :1]] += 3                                  # the student follows: the largest logit is not the rest's
    x[at[1::8], idx[1::8]] += 60                            # the rest class vanishes
    keep = torch.zeros(rows, vocab, dtype=torch.bool).scatter_(1, idx, True)
    x[2::8] = torch.where(keep[2::8], x[2::8], torch.full_like(x[2::8], -INF))     # is empty
    weights[3::8] = 0.0
    x[4::8] = -INF
    idx[5::8, 1] = idx[5::8, 0]
    x[6::8, 0] = float("nan")

    def step(pick):
        for tail in (lse[pick].to(DEV), None):
            a = x[pick].to(DEV).requires_grad_(True)
            out = L.topk_distillation_loss(a, val[pick].to(DEV), idx[pick].to(DEV), tail, weights=weights[pick].to(DEV),
                                           reduction="none")
            (g,) = torch.autograd.grad(out, a, torch.ones(len(pick), device=DEV))
            yield out.detach().cpu(), g.cpu()
        top = L.top_logits(x[pick].to(DEV), k)
        yield top.lse.cpu(), top.values.cpu()

    together = list(step(list(range(rows))))
    for r in range(rows):
        for (loss, grad), (loss1, grad1) in zip(together, step([r])):
            for name, a, b in (("loss", loss[r], loss1[0]), ("gradient", grad[r], grad1[0])):
                assert torch.equal(torch.nan_to_num(a.float(), nan=7e4), torch.nan_to_num(b.float(), nan=7e4)), (name, r)


SIZES = [(5, 40, 24, False), (12, 500, 3000, True), (40, 3000, 64, True), (200, 300, 96, False), (1030, 4000, 330, True),
         (70, 9001, 1003, True), (2100, 8200, 128, False)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,dim,bias", SIZES)
@pytest.mark.parametrize("bad", [INF, -INF, float("nan")])
def test_a_gradient_that_is_not_finite_stays_in_its_row(rows, vocab, dim, bias, bad, dtype):
    import mde_amd.vocab_losses as L
    h, w, b, _, t = exact_operands(rows, vocab, dim, 0.0, dtype, 5)
    leaves = [x.to(DEV).requires_grad_(True) for x in ((h, w, b) if bias else (h, w))]
    for z_loss in (0.0, 1e-2):
        out = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2] if bias else None, z_loss=z_loss, reduction="none")
        up = torch.randn(rows, generator=gen(3)).to(DEV)
        want = torch.autograd.grad(out, leaves, up, retain_graph=True)
        worse = up.clone()
        worse[2] = bad
        got = torch.autograd.grad(out, leaves, worse)
        others = torch.arange(rows, device=DEV) != 2
        assert bool(torch.isfinite(want[0]).all()) and torch.equal(got[0][others], want[0][others])
        assert not torch.isfinite(got[0][2]).any()
        assert not any(torch.isfinite(g).any() for g in got[1:])      # sums over all rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,dim,bias", SIZES)
def test_rows_of_very_different_gradients_keep_their_digits(rows, vocab, dim, bias, dtype):
    """Powers of two between 2^-30 and 2^15 (float16: results down to its subnormal numbers), 2^-110 and 2^15: a row's
    grad_hidden is the one of a gradient of 1, times its own."""
    import mde_amd.vocab_losses as L
    h, w, b, _, t = exact_operands(rows, vocab, dim, 0.0, dtype, 6)
    leaves = [x.to(DEV).requires_grad_(True) for x in ((h, w, b) if bias else (h, w))]
    out = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2] if bias else None, reduction="none")
    (ones,) = torch.autograd.grad(out, leaves[:1], torch.ones(rows, device=DEV), retain_graph=True)
    low = -30 if dtype == torch.float16 else -110
    power = torch.randint(low, 16, (rows,), generator=gen(4))
    power[0], power[1] = 15, low
    up = torch.tensor([2.0 ** p for p in power.tolist()], device=DEV)      # exactly (torch.ldexp is off by a step there)
    got = torch.autograd.grad(out, leaves, up)
    want = ones.double() * up.double()[:, None]
    if dtype != torch.float16:
        # a power of two changes no digit of a normal number; below 2^-126 the type's step is fixed and a result is rounded to
        # it (float32: half a step; bfloat16: after float32's, half a step of its own and 2^-150), less than one step
        small = want.abs() < 2.0 ** -126
        assert torch.equal(got[0].double()[~small], want[~small])
        B.close(got[0].double()[small], want[small], B.TINY[dtype], "subnormal results")
        return
    # both are rounded to float16: by half a step of the value, below 2^-14 by half its fixed step of 2^-24, which the comparison
    # multiplies by the gradient where it is that of 1 which was rounded
    fixed = B.TINY[dtype] / 2 * (1 + up.double()[:, None].cpu())
    B.close(got[0], want, 2 * B.HALF_STEP[dtype] * want.abs().cpu() + fixed, "grad hidden")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(40, 300, 96), (12, 500, 3000), (1030, 4000, 330), (2100, 8200, 128), (1500, 5000, 512)])
@pytest.mark.parametrize("strided", [False, True])
def test_infinite_operands_mean_the_same_at_every_size(rows, vocab, dim, strided, dtype):
    """float32 directly, in parts and by planes: a class at -infinity by its weight is masked, a row that has only such
    classes adds nothing, and a row that meets +infinity is NaN; no other row is."""
    import mde_amd.vocab_losses as L
    h, w, b, z, t = exact_operands(rows, vocab, dim, 0.0, dtype, 9)
    h, w = h.double(), w.double()
    h[:, 5], w[:, 5] = 1.0, -1.0
    w[7, 5] = -INF                                          # masked: every row has a positive feature there
    h[3, 5] = INF                                           # nothing is left of this row
    h[rows - 2, 4], w[:, 4] = INF, 1.0                      # +infinity, and against class 7 infinity minus infinity
    t[t == 7] = 8
    h, w = h.to(dtype), w.to(dtype)
    z = h.double() @ w.double().T + b.double()
    fine = [r for r in range(rows) if r not in (3, rows - 2)]
    assert bool((z[3] == -INF).all()) and bool((z[fine, 7] == -INF).all()) and bool(torch.isnan(z[rows - 2, 7]))
    place = lambda x: torch.nn.functional.pad(x, (3, 2)).to(DEV)[:, 3:-2] if strided else x.to(DEV)
    leaves = [place(h).detach().requires_grad_(True), place(w).detach().requires_grad_(True), b.to(DEV).requires_grad_(True)]
    out = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2], reduction="none")
    loss, ltol, ds, dtol = B.linear_ce(z[fine], t[fine])
    B.close(out[fine], loss, ltol, "row losses")
    assert float(out[3].detach()) == 0.0 and bool(torch.isnan(out[rows - 2]))
    up = torch.ones(rows, device=DEV)
    up[rows - 2] = 0.0                                      # not asked for: the row's NaN stays out of the sums
    gh, gw, gb = (g.detach().cpu().double() for g in torch.autograd.grad(out, leaves, up))
    cols = [c for c in range(dim) if c != 5]
    # 0 times -infinity where the masked class meets grad_hidden's feature 5: as in any product with it
    assert bool(torch.isnan(gh[:, 5]).all()) and not gh[3, cols].any() and not gh[rows - 2, cols].any()
    half, n = B.HALF_STEP[dtype], max(rows, vocab) + 4
    floor = 2.0 ** -36 if dtype == torch.float16 else 0.0
    err = dtol + ds.abs() * half * 1.01 + floor
    h6, w6 = h.double()[fine], w.double()[:, cols]
    for name, got, want, tol in (
            ("grad hidden", gh[fine][:, cols], ds @ w6, err @ w6.abs() + n * B.U * (ds.abs() @ w6.abs())),
            ("grad weight", gw, ds.T @ h6, err.T @ h6.abs() + n * B.U * (ds.abs().T @ h6.abs())),
            ("grad bias", gb, ds.sum(0), err.sum(0) + n * B.U * ds.abs().sum(0))):
        B.close(got, want, tol + (half + 8 * B.U) * want.abs() + B.TINY[dtype], name)


@pytest.mark.parametrize("rows,vocab,dim", [(40, 300, 96), (1500, 5000, 512), (2100, 8200, 128)])
def test_a_row_that_is_not_finite_changes_no_bit_of_another(rows, vocab, dim):
    """Every third row of hidden infinite or NaN, and a class that is masked out with weights of NaN: the others as without."""
    import mde_amd.vocab_losses as L
    g = gen(13)
    h, w, b = torch.randn(rows, dim, generator=g), torch.randn(vocab, dim, generator=g) / math.sqrt(dim), torch.zeros(vocab)
    t = torch.randint(vocab - 4, (rows,), generator=g)
    b[vocab - 4:] = -INF
    fine = torch.arange(rows) % 3 != 1
    outs = []
    for spoiled in (False, True):
        h2, w2 = h.clone(), w.clone()
        if spoiled:
            h2[1::6, 7], h2[4::6, 9] = INF, float("nan")
            w2[vocab - 4:] = float("nan")
        leaves = [h2.to(DEV).requires_grad_(True), w2.to(DEV), b.to(DEV)]
        out = L.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2], reduction="none")
        (grad,) = torch.autograd.grad(out, leaves[:1], torch.ones(rows, device=DEV))
        outs.append((out.detach().cpu()[fine], grad.cpu()[fine]))
        assert bool(torch.isfinite(out[fine]).all()) and bool(torch.isnan(out[~fine]).all()) == spoiled
    assert all(torch.equal(x, y) for x, y in zip(*outs))


# ------------------------------------------------------------------ pieces of the vocabulary
@pytest.mark.parametrize("rows,vocab,dim,dtype,off", [
    (2048, 70001, 330, torch.float32, 0),                   # by planes, pieces of 2^27 derivatives
    (300, 70001, 4096, torch.float32, 0),                   # by planes, pieces of 2^30 bytes of weight, forward as well
    (1200, 140000, 4099, torch.bfloat16, 1),                 # rows that 16-byte loads cannot take, copied piece by piece
    (300, 140000, 4000, torch.float16, 0),                   # only the transposed weight goes in pieces
    (100, 40000, 4096, torch.float32, 1),                   # few rows: the weight as it lies
    (1030, 257, 64, torch.bfloat16, 0), (1030, 129, 96, torch.float32, 3), (9000, 100, 40, torch.float16, 0)])   # one, ragged
def test_linear_cross_entropy_lays_out_piece_by_piece(rows, vocab, dim, dtype, off):
    from test_gpu_vocab_losses import ce_inputs, check_ce
    h, w, b, t = ce_inputs(rows, vocab, dim, dtype, rows + dim, bias=True)
    t[torch.rand(rows, generator=gen(21)) < 0.2] = -100
    masked = torch.cat([torch.arange(vocab - 3, vocab), torch.arange(5, vocab, 301)])
    b[masked], w[masked] = -INF, float("nan")
    t = torch.where(torch.isin(t, masked), torch.ones_like(t), t)
    wide = torch.zeros(vocab, dim + 2 * off, dtype=dtype, device=DEV)
    wide[:, off:off + dim] = w.to(DEV)
    check_ce(h, w, b, t, on_device=(h.to(DEV), wide[:, off:off + dim]))


# ------------------------------------------------------------------ the trainer's surface
@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [True, False])
def test_depth_bins_under_autocast(low, bias):
    """A 16-bit decoder with float32 parameters: the head's cross entropy beside the convolution's own, gradients in float32."""
    import types
    from mde_amd.trainer_loss import ViewSynthesisLoss
    vs = ViewSynthesisLoss(types.SimpleNamespace(height=12, width=20))
    g = gen(31)
    image = torch.randn(2, 8, 12, 20, generator=g).to(DEV)
    body, head = torch.nn.Conv2d(8, 32, 1).to(DEV), torch.nn.Conv2d(32, 48, 1, bias=bias).to(DEV)
    with torch.no_grad():
        for p in list(body.parameters()) + list(head.parameters()):
            p.copy_(torch.randn(p.shape, generator=g).to(DEV) * 0.5)
    target = torch.randint(48, (2, 12, 20), generator=g)
    target[torch.rand(2, 12, 20, generator=g) < 0.3] = -100
    with torch.autocast("cuda", dtype=low):
        features = body(image)
        assert features.dtype == low
        features.retain_grad()
        loss = vs.compute_bin_cross_entropy(features, head.weight, target.to(DEV), head.bias)
    loss.backward()
    assert loss.dtype == torch.float32 and features.grad.dtype == low
    params = [head.weight] + ([head.bias] if bias else [])
    assert all(p.grad.dtype == torch.float32 and p.grad.shape == p.shape for p in params)
    # the definition on what the call rounds: features and parameters in 16 bits
    f6, w6 = (x.detach().cpu().double().requires_grad_(True) for x in (features, head.weight.to(low)))
    b6 = head.bias.detach().to(low).cpu().double().requires_grad_(True) if bias else None
    want = torch.nn.functional.cross_entropy(torch.nn.functional.conv2d(f6, w6, b6), target)
    want.backward()
    # 32 features of below 8 x 2.5: a logit's products and their sum are off by 34 u of their sizes' sum, below 200, and the
    # log sum's own error comes on top, twice for the difference
    assert abs(float(loss.detach()) - float(want.detach())) <= 2 * (34 * B.U * 200 + B.tile_sum(48) + 100 * B.U)
    # derivatives are rounded to 16 bits and so are the gradients' sums: two half steps of every term at most, and in float16
    # the fixed step of its subnormal numbers, under 2^12 of scale for the derivatives
    half = B.HALF_STEP[low]
    n = int((target >= 0).sum())
    z = torch.nn.functional.conv2d(f6, w6, b6).detach().movedim(1, -1).reshape(-1, 48)
    ds = torch.softmax(z, 1)
    live = target.reshape(-1) >= 0
    ds[live, target.reshape(-1)[live]] -= 1
    ds = (ds * live[:, None]).abs() / n
    err = ds * (half * 1.01) + 2e-5 / n + (2.0 ** -36 / n if low == torch.float16 else 0.0)
    rows = f6.detach().movedim(1, -1).reshape(-1, 32)
    pairs = [(features.grad, f6.grad, (err @ w6.detach().reshape(48, 32).abs()).reshape(2, 12, 20, 32).movedim(-1, 1)),
             (head.weight.grad, w6.grad, (err.T @ rows.abs()).reshape(48, 32, 1, 1))]
    if bias:
        pairs.append((head.bias.grad, b6.grad, err.sum(0)))
    for got, ref, tol in pairs:
        B.close(got, ref, tol + (half + 8 * B.U) * ref.abs() + B.TINY[low], "gradient")


# ------------------------------------------------------------------ calls that are refused
def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwad

    import mde_amd._abi as abi
    import mde_amd.vocab_losses as L
    x, w, b = (torch.randn(s, generator=gen(1)).to(DEV) for s in ((6, 20), (30, 20), (30,)))
    v, i = L.top_logits(x, 3)[:2]
    t = torch.arange(6, device=DEV)
    with fwad.dual_level():
        for needs in (False, True):
            dual = [fwad.make_dual(a.clone().requires_grad_(needs), torch.ones_like(a)) for a in (x, w, b)]
            calls = [lambda: L.topk_distillation_loss(dual[0], v, i), lambda: L.topk_distillation_loss(dual[0][:, ::2], v, i // 2),
                     lambda: L.linear_cross_entropy(dual[0], w, t, b), lambda: L.linear_cross_entropy(x, dual[1], t, b),
                     lambda: L.linear_cross_entropy(x, w, t, dual[2])]
            for call in calls:
                with pytest.raises(abi.VslError, match="forward-mode"):
                    call()
                with torch.no_grad(), pytest.raises(abi.VslError, match="forward-mode"):
                    call()
        # what carries no gradient backwards carries none forwards
        assert fwad.unpack_dual(L.top_logits(dual[0], 3).values).tangent is None
        loss = L.topk_distillation_loss(x, fwad.make_dual(v, torch.ones_like(v)), i)
        assert fwad.unpack_dual(loss).tangent is None
    assert bool(torch.isfinite(L.topk_distillation_loss(x, v, i)))
