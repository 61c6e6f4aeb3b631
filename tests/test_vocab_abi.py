"""CPU-side checks of the C boundary of the losses over a set of classes: the ctypes mirrors match the C structs, malformed
descriptors are refused before anything is launched, and workspaces are sized for them."""
import ctypes

import pytest
import torch

FAKE = 0x1000       # never dereferenced: validation fails first


def err(abi):
    return abi.lib.vsl_last_error_string()


def top(abi, **kw):
    return abi.TopDesc(**dict(dict(rows=8, vocab=5000, stride=5000, k=4, type=0, temperature=1.0, logits=FAKE), **kw))


def distill(abi, **kw):
    return abi.DistillDesc(**dict(dict(rows=8, vocab=5000, stride=5000, k=4, type=1, value_type=0, index_bytes=4, reduction=2,
                                       temperature=1.0, logits=FAKE, teacher_values=FAKE, teacher_indices=FAKE), **kw))


def linear(abi, **kw):
    return abi.LinearCeDesc(**dict(dict(rows=8, vocab=500, dim=64, hidden_stride=64, weight_stride=64, ignore_index=-100, type=1,
                                        reduction=2, z_loss=0.0, hidden=FAKE, weight=FAKE, target=FAKE), **kw))


def test_mirrors_and_version():
    import mde_amd._abi as abi
    assert ctypes.sizeof(abi.TopDesc) == 48 and ctypes.sizeof(abi.DistillDesc) == 88 and ctypes.sizeof(abi.LinearCeDesc) == 96
    assert abi.lib.vsl_version() >= 220


BAD_ROWS = [dict(rows=-1), dict(rows=1 << 31), dict(vocab=0, stride=9), dict(vocab=1 << 30, stride=1 << 30), dict(stride=4999),
            dict(type=3), dict(k=0), dict(k=257), dict(k=5, vocab=4), dict(temperature=0.0), dict(temperature=float("nan")),
            dict(temperature=float("inf")), dict(temperature=9e-5), dict(temperature=1.1e4), dict(logits=None), dict(logits=FAKE + 1)]


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_top_logits_refuses(bad):
    import mde_amd._abi as abi
    d = top(abi, **bad)
    assert abi.lib.vsl_top_logits(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE * 16, 1 << 40, None) == -1 and err(abi)


def test_top_logits_outputs_and_workspace():
    import mde_amd._abi as abi
    d = top(abi, vocab=50000, stride=50000)
    need = abi.lib.vsl_top_logits_workspace_bytes(ctypes.byref(d))
    assert need >= 8 * 2 * 4 * 8 and need % 256 == 0         # few long rows are split, by 16384 classes at least
    call = lambda v, i, ws, n: abi.lib.vsl_top_logits(ctypes.byref(d), v, i, None, ws, n, None)
    assert call(None, FAKE, FAKE * 16, need) == -1 and call(FAKE, None, FAKE * 16, need) == -1
    assert call(FAKE, FAKE, FAKE * 16, need - 1) == -2 and b"workspace" in err(abi)
    assert call(FAKE, FAKE, FAKE * 16 + 8, need) == -1 and b"aligned" in err(abi)
    assert call(FAKE, FAKE, None, need) == -1
    assert call(FAKE + 2, FAKE, FAKE * 16, need) == -1 and call(FAKE, FAKE + 2, FAKE * 16, need) == -1
    assert abi.lib.vsl_top_logits_workspace_bytes(ctypes.byref(top(abi, vocab=1000, stride=1000))) == 0   # short rows need none
    assert abi.lib.vsl_top_logits(None, FAKE, FAKE, None, None, 0, None) == -1
    assert abi.lib.vsl_top_logits(ctypes.byref(top(abi, rows=0, logits=None)), None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("bad", BAD_ROWS + [dict(value_type=7), dict(index_bytes=2), dict(reduction=3), dict(reduction=-1),
                                            dict(teacher_values=None), dict(teacher_indices=None)])
def test_distill_refuses(bad):
    import mde_amd._abi as abi
    d = distill(abi, **bad)
    assert abi.lib.vsl_distill_fwd(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE * 16, 1 << 40, None) == -1 and err(abi)
    assert abi.lib.vsl_distill_bwd(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, 1 << 31, None) == -1


def test_distill_outputs_and_workspace():
    import mde_amd._abi as abi
    d = distill(abi)
    need = abi.lib.vsl_distill_workspace_bytes(ctypes.byref(d))
    assert need > 0 and need % 256 == 0
    fwd = lambda r, l, v, s, ws, n: abi.lib.vsl_distill_fwd(ctypes.byref(d), r, l, v, s, ws, n, None)
    for missing in range(4):
        args = [FAKE] * 4
        args[missing] = None
        assert fwd(*args, FAKE * 16, need) == -1
    assert fwd(FAKE, FAKE, FAKE, FAKE, FAKE * 16, need - 1) == -2
    assert fwd(FAKE, FAKE, FAKE, FAKE, FAKE * 16 + 128, need) == -1
    bwd = lambda s, v, g, out, stride: abi.lib.vsl_distill_bwd(ctypes.byref(d), s, v, g, out, stride, None)
    assert bwd(None, FAKE, FAKE, FAKE, 5000) == -1 and bwd(FAKE, None, FAKE, FAKE, 5000) == -1
    assert bwd(FAKE, FAKE, None, FAKE, 5000) == -1 and bwd(FAKE, FAKE, FAKE, None, 5000) == -1
    assert bwd(FAKE, FAKE, FAKE, FAKE, 4999) == -1 and b"stride" in err(abi)
    assert bwd(FAKE + 4, FAKE, FAKE, FAKE, 5000) == -1 and bwd(FAKE, FAKE, FAKE, FAKE + 1, 5000) == -1 and b"misaligned" in err(abi)
    assert fwd(FAKE, FAKE, FAKE, FAKE + 4, FAKE * 16, need) == -1 and b"aligned" in err(abi)
    assert abi.lib.vsl_distill_fwd(None, FAKE, FAKE, FAKE, FAKE, FAKE, 1, None) == -1


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(rows=1 << 28), dict(vocab=0), dict(vocab=1 << 30), dict(dim=0), dict(dim=1 << 24, hidden_stride=1 << 25, weight_stride=1 << 25),
    dict(hidden_stride=63), dict(weight_stride=63), dict(type=-1), dict(reduction=5), dict(z_loss=-1.0), dict(z_loss=float("nan")),
    dict(z_loss=float("inf")), dict(hidden=None), dict(weight=None), dict(target=None), dict(hidden=FAKE + 1), dict(weight=FAKE + 1),
    dict(bias=FAKE + 1), dict(rows=1 << 20, vocab=1 << 18), dict(rows=1 << 27, dim=1024, hidden_stride=1024, weight_stride=1024),
    dict(vocab=1 << 27, dim=1024, hidden_stride=1024, weight_stride=1024)])
def test_linear_ce_refuses(bad):
    import mde_amd._abi as abi
    d = linear(abi, **bad)
    assert abi.lib.vsl_linear_ce_fwd_workspace_bytes(ctypes.byref(d)) == 0
    assert abi.lib.vsl_linear_ce_bwd_workspace_bytes(ctypes.byref(d), 7) == 0
    assert abi.lib.vsl_linear_ce_fwd(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE * 16, 1 << 40, None) == -1 and err(abi)
    assert abi.lib.vsl_linear_ce_bwd(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE * 16, 1 << 40, None) == -1


def test_linear_ce_outputs_and_workspace():
    import mde_amd._abi as abi
    d = linear(abi)
    need = abi.lib.vsl_linear_ce_fwd_workspace_bytes(ctypes.byref(d))
    fwd = lambda r, s, l, v, ws, n: abi.lib.vsl_linear_ce_fwd(ctypes.byref(d), r, s, l, v, ws, n, None)
    for missing in range(4):
        args = [FAKE] * 4
        args[missing] = None
        assert fwd(*args, FAKE * 16, need) == -1
    assert fwd(FAKE, FAKE, FAKE, FAKE, FAKE * 16, need - 1) == -2
    assert fwd(FAKE, FAKE, FAKE, FAKE, FAKE * 16 + 16, need) == -1
    sizes = [abi.lib.vsl_linear_ce_bwd_workspace_bytes(ctypes.byref(d), m) for m in (1, 2, 4, 7)]
    assert all(0 < s <= sizes[3] and s % 256 == 0 for s in sizes)
    bwd = lambda s, v, g, gh, ws, n: abi.lib.vsl_linear_ce_bwd(ctypes.byref(d), s, v, g, gh, None, None, ws, n, None)
    assert bwd(None, FAKE, FAKE, FAKE, FAKE * 16, sizes[0]) == -1 and bwd(FAKE, None, FAKE, FAKE, FAKE * 16, sizes[0]) == -1
    assert bwd(FAKE, FAKE, None, FAKE, FAKE * 16, sizes[0]) == -1
    assert bwd(FAKE, FAKE, FAKE, FAKE, FAKE * 16, sizes[0] - 1) == -2
    assert bwd(FAKE, FAKE, FAKE, FAKE + 1, FAKE * 16, sizes[0]) == -1 and b"misaligned" in err(abi)
    assert bwd(FAKE, FAKE, FAKE, None, None, 0) == 0                       # no gradient is wanted
    # odd widths and rows that 16-byte loads cannot take: through registers, or laid out anew, which takes more workspace
    for kw in (dict(dim=65, hidden_stride=65, weight_stride=65), dict(hidden=FAKE + 2), dict(hidden_stride=65)):
        assert abi.lib.vsl_linear_ce_fwd_workspace_bytes(ctypes.byref(linear(abi, **kw))) >= need
    # one size for every extent of the documented limits, without overflow
    for rows, vocab, dim in ((1, 1, 1), (1, (1 << 27) - 1, 1), ((1 << 27) - 1, 100, 8), (1 << 18, 1 << 18, 64), (3, 3, (1 << 24) - 1)):
        d = linear(abi, rows=rows, vocab=vocab, dim=dim, hidden_stride=dim, weight_stride=dim)
        for n in (abi.lib.vsl_linear_ce_fwd_workspace_bytes(ctypes.byref(d)), abi.lib.vsl_linear_ce_bwd_workspace_bytes(ctypes.byref(d), 7)):
            assert 0 < n < 1 << 46


def test_python_refuses_cpu_tensors():
    import mde_amd.vocab_losses as L
    x, i = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        L.top_logits(x, 2)
    with pytest.raises(ValueError, match="GPU"):
        L.topk_distillation_loss(x, x[:, :2], i)
    with pytest.raises(ValueError, match="GPU"):
        L.linear_cross_entropy(x, x, i[:, 0])
