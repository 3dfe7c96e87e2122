"""Host checks of the operators around the attention call: their refusals (before any launch; the
pointers given to the C entry points are never dereferenced), the overlap rule of outputs, and
the rotary tables."""

import math

import pytest
import torch

import recap_amd
from recap_amd import _lib
from recap_amd import kernels as K

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def test_rotary_axes_are_the_formula():
    grid, channels = (5, 3, 7), (44, 42, 42)
    where = [None, [0.5, 1.25, 300.0], None]
    tables = recap_amd.rotary_axes(grid, channels, theta=256.0, positions=where)
    for axis, table in enumerate(tables):
        assert table.dtype == F32 and table.shape == (grid[axis], channels[axis] // 2, 2)
        for p in range(grid[axis]):
            at = p if where[axis] is None else where[axis][p]
            for i in range(channels[axis] // 2):
                angle = at * 256.0 ** (-2 * i / channels[axis])
                for got, want in zip(table[p, i].tolist(), (math.cos(angle), math.sin(angle))):
                    # half a step of fp32, and the angle's own few 64-bit roundings
                    assert abs(got - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -50 * (1 + abs(angle))


def test_rotary_axes_far_position():
    """A position far out: the angle is taken in 64 bits (32 would be off by ~1e-1)."""
    table = recap_amd.rotary_axes((1, 1, 1), (0, 2, 2), positions=[None, [16777217.0], None])
    assert table[0].shape == (1, 0, 2)
    assert abs(table[1][0, 0, 0].item() - math.cos(16777217.0)) < 1e-7


@pytest.mark.parametrize("bad", [
    dict(grid=(2, 3), channels=(2, 2, 2)), dict(grid=(0, 3, 3), channels=(2, 2, 2)),
    dict(grid=(2, 3, 3), channels=(3, 2, 2)), dict(grid=(2, 3, 3), channels=(-2, 2, 2)),
    dict(grid=(2, 3, 3), channels=(2, 2, 2), theta=0.0),
    dict(grid=(2, 3, 3), channels=(2, 2, 2), positions=[None, [0.0], None]),
    dict(grid=(2, 3, 3), channels=(2, 2, 2), positions=[None, None])])
def test_rotary_axes_refusals(bad):
    with pytest.raises(ValueError):
        recap_amd.rotary_axes(**bad)


def axes64():
    return recap_amd.rotary_axes((2, 3, 4), (16, 24, 24))


@pytest.mark.parametrize("bad,match", [
    (dict(q=torch.zeros(2, 30, 64, dtype=BF)), "batch, heads, tokens, dim"),
    (dict(q=torch.zeros(1, 2, 30, 96, dtype=BF)), "head dim"),
    (dict(q=torch.zeros(1, 2, 30, 64)), "dtype"),
    (dict(k=torch.zeros(1, 2, 30, 64, dtype=FP)), "match"),
    (dict(k=torch.zeros(1, 2, 31, 64, dtype=BF)), "match"),
    (dict(k=torch.zeros(2, 2, 30, 64, dtype=BF)), "match"),
    (dict(k_weight=torch.zeros(64, dtype=BF), norm="rms"), "need a k"),
    (dict(norm="max"), "norm"), (dict(pairing="odd"), "pairing"),
    (dict(q_weight=torch.zeros(64, dtype=BF)), "needs a norm"),
    (dict(q_weight=torch.zeros(32, dtype=BF), norm="rms"), "expected"),
    (dict(q_weight=torch.zeros(64, dtype=BF), norm="rms_all"), "expected"),
    (dict(q_weight=torch.zeros(64, dtype=FP), norm="rms"), "weights"),
    (dict(q_weight=torch.zeros(64, dtype=BF), q_bias=torch.zeros(64), norm="rms"), "one type"),
    (dict(axes=axes64()[:2]), "three"), (dict(axes=[t.double() for t in axes64()]), "fp32"),
    (dict(axes=recap_amd.rotary_axes((2, 3, 4), (16, 24, 22))), "channels"),
    (dict(axes=axes64(), offset=7), "sequence"), (dict(axes=axes64(), offset=-1), "sequence"),
    (dict(), "GPU")])
def test_qk_rotary_refusals(bad, match):
    args = dict(q=torch.zeros(1, 2, 30, 64, dtype=BF), **{})
    args.update(bad)
    with pytest.raises(ValueError, match=match):
        K.qk_rotary(args.pop("q"), args.pop("k", None), args.pop("axes", None), **args)


X = torch.zeros(2, 5, 24, dtype=BF)
X32 = torch.zeros(2, 5, 24)


@pytest.mark.parametrize("call,match", [
    (lambda: K.norm_modulate(X[0]), "batch, tokens, width"),
    (lambda: K.norm_modulate(torch.zeros(2, 5, 0, dtype=BF)), "batch, tokens, width"),
    (lambda: K.norm_modulate(X, norm=None), "norm"),
    (lambda: K.norm_modulate(X, norm="batch"), "norm"),
    (lambda: K.norm_modulate(X.double()), "dtype"),
    (lambda: K.norm_modulate(X32, dtype=torch.float64), "dtype"),
    (lambda: K.norm_modulate(X, dtype=F32), "stream"),
    (lambda: K.norm_modulate(X, dtype=FP), "stream"),
    (lambda: K.norm_modulate(X, torch.zeros(23, dtype=BF)), "scale is"),
    (lambda: K.norm_modulate(X, torch.zeros(3, 24, dtype=BF)), "scale is"),
    (lambda: K.norm_modulate(X, None, torch.zeros(2, 4, 24, dtype=BF)), "shift is"),
    (lambda: K.norm_modulate(X, torch.zeros(1, 2, 5, 24, dtype=BF)), "scale is"),
    (lambda: K.norm_modulate(X, torch.zeros(24, dtype=FP)), "scale is"),
    (lambda: K.norm_modulate(X, torch.zeros(24), torch.zeros(24, dtype=BF)), "one type"),
    (lambda: K.norm_modulate(X, weight=torch.zeros(23, dtype=BF)), "expected"),
    (lambda: K.norm_modulate(X, weight=torch.zeros(24), bias=torch.zeros(24, dtype=BF)), "weights"),
    (lambda: K.gated_residual(X, X[:, :4]), "branch is"),
    (lambda: K.gated_residual(X, X32), "stream"),
    (lambda: K.gated_residual(X, X, branch_weight=torch.zeros(24, dtype=BF)), "needs a norm"),
    (lambda: K.gated_residual(X, X, branch_norm="all"), "branch_norm"),
    (lambda: K.gated_residual_norm(X, X, norm=None), "norm"),
    (lambda: K.gated_residual_norm(X, X, branch_norm="rms", branch_weight=torch.zeros(24),
                                   weight=torch.zeros(24, dtype=BF)), "weights"),
    (lambda: K.norm_modulate(X), "GPU"), (lambda: K.gated_residual(X, X), "GPU"),
    (lambda: K.gated_residual_norm(X, X), "GPU")])
def test_residual_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


@pytest.mark.parametrize("call", [
    lambda x, w: K.norm_modulate(x), lambda x, w: K.norm_modulate(x.detach(), weight=w),
    lambda x, w: K.gated_residual(x, x.detach()), lambda x, w: K.gated_residual_norm(X[:, :, :1].expand(2, 5, 64), x),
    lambda x, w: K.qk_rotary(x.view(1, 2, 5, 64)),
    lambda x, w: K.qk_rotary(x.detach().view(1, 2, 5, 64), norm="rms", q_weight=w)])
def test_derivatives_are_refused(call):
    """No call drops a derivative silently: neither a gradient it would have to record nor, also
    under no_grad, the tangent of forward mode."""
    from torch.autograd import forward_ad
    x, w = torch.randn(2, 5, 64).to(BF), torch.ones(64, dtype=BF)
    with pytest.raises(ValueError, match="gradient"):
        call(x.clone().requires_grad_(), w.clone().requires_grad_())
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(ValueError, match="tangent"):
            call(*(forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w)))
        with pytest.raises(ValueError, match="GPU"):
            call(x, w)


def test_output_overlap_rule():
    """An output may be the input it is named for, or take turns with inputs in rows of one
    pitch; anything else that shares memory is refused."""
    check = lambda out, same="x", **inputs: K._check_output(  # noqa: E731
        "out", out, out.shape, out.dtype, inputs, same)
    x = torch.zeros(2, 5, 24)
    check(x, x=x)
    check(x[:, :, :], x=x, other=torch.zeros(2, 5, 24))
    for bad in (dict(same="", x=x), dict(x=x.view(5, 2, 24)), dict(x=x, y=x)):
        with pytest.raises(ValueError, match="overlaps"):
            check(x, **bad)
    with pytest.raises(ValueError, match="overlaps"):
        check(x[:, 1:], x=x[:, :4])
    with pytest.raises(ValueError, match="share memory"):
        check(torch.zeros(1, 5, 24).expand(2, 5, 24), x=x)
    with pytest.raises(ValueError, match="share memory"):
        check(torch.as_strided(x, (2, 5, 24), (12, 24, 1)), x=torch.zeros(2, 5, 24))
    with pytest.raises(ValueError, match="unit stride"):
        check(torch.zeros(2, 5, 48)[:, :, ::2], x=x)
    qkv = torch.zeros(2, 7, 3, 4, 64)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    check(q, same="q", q=q, k=k, v=v)
    check(k, same="k", q=q, k=k, v=v)
    with pytest.raises(ValueError, match="overlaps"):
        check(q, same="q", q=q, k=qkv.flatten(2)[:, :, 100:356].unflatten(2, (4, 64)).transpose(1, 2))
    wide = torch.zeros(2, 5, 60)
    check(wide[:, :, :24], x=wide[:, :, 24:48])
    with pytest.raises(ValueError, match="overlaps"):
        check(wide[:, :, :24], x=wide[:, :, 20:44])
    with pytest.raises(ValueError, match="overlaps"):   # two elements of other types
        check(wide[:, :, :24], x=wide[:, :, 30:42].view(BF))


GOOD_QK = dict(q=16, k=16, dtype=_lib.RECAP_BF16, batch=1, tokens=30, dim=64, qh=2, kh=2, qb=0, qs=64,
               qn=128, kb=0, ks=64, kn=128, t0=16, t1=16, t2=16, lengths=(2, 3, 4), pairs=(8, 12, 12),
               offset=6, pairing=0, norm=1, qw=16, qbias=None, kw=16, kbias=None, wt=_lib.RECAP_BF16,
               eps=1e-6, qo=16, qob=0, qos=64, qon=128, ko=16, kob=0, kos=64, kon=128)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(q=8), dict(qo=None), dict(ko=None), dict(k=None), dict(dtype=_lib.RECAP_F32),
    dict(dim=96), dict(tokens=0), dict(batch=0), dict(qh=0), dict(qh=1 << 17), dict(kn=3), dict(kon=0),
    dict(batch=1 << 30), dict(pairing=2), dict(norm=4), dict(norm=-1), dict(norm=0), dict(eps=0.0),
    dict(eps=float("nan")), dict(wt=_lib.RECAP_F16), dict(qw=17), dict(t0=None),
    dict(t1=12), dict(lengths=None), dict(lengths=(2, 3, 0)), dict(lengths=(2, 3, 31)),
    dict(lengths=(3, 4, 4)), dict(pairs=(8, 12, 11)), dict(pairs=(-8, 28, 12)), dict(offset=7),
    dict(offset=-1)])
def test_qk_rotary_entry_refusals(bad):
    import ctypes
    a = {**GOOD_QK, **bad}
    for name in ("lengths", "pairs"):
        a[name] = a[name] and (ctypes.c_int64 * 3)(*a[name])
    with pytest.raises(ValueError):
        _lib.call("recap_qk_rotary", *a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(qos=0), dict(kos=0), dict(qos=32), dict(kon=64), dict(qon=64), dict(qos=64, qon=72),
    dict(batch=2, qob=0, kob=30 * 128), dict(batch=2, qob=30 * 128, kob=0),
    dict(batch=2, qob=29 * 128, kob=30 * 128), dict(batch=2, qob=64, kob=30 * 128),
    dict(batch=3, qob=1 << 62, kob=1 << 62, qos=1 << 62)])
def test_qk_rotary_entry_refuses_outputs_that_share_memory(bad):
    """Two (token, head) rows of an output at one address would be written by two waves."""
    import ctypes
    a = {**GOOD_QK, **bad}
    for name in ("lengths", "pairs"):
        a[name] = (ctypes.c_int64 * 3)(*a[name])
    with pytest.raises(ValueError, match="overlap"):
        _lib.call("recap_qk_rotary", *a.values(), None)


GOOD_ROWS = dict(x=16, xt=_lib.RECAP_F32, batch=2, tokens=5, width=24, xb=120, xn=24, branch=16,
                 t=_lib.RECAP_BF16, bb=120, bn=24, gate=16, gb=24, gn=0, scale=16, sb=24, sn=0,
                 shift=16, hb=24, hn=0, mt=_lib.RECAP_F32, bw=16, bbias=16, w=16, bias=16,
                 wt=_lib.RECAP_BF16, post=1, norm=2, eps=1e-6, r=16, rb=120, rn=24, out=16, ob=120,
                 on=24)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(branch=None), dict(r=None), dict(out=None), dict(xt=_lib.RECAP_F16), dict(t=7),
    dict(xt=0), dict(mt=_lib.RECAP_F16), dict(wt=_lib.RECAP_F16), dict(batch=0), dict(tokens=0),
    dict(width=0), dict(width=(1 << 24) + 1), dict(batch=1 << 31), dict(post=3), dict(post=0),
    dict(norm=0), dict(norm=3), dict(eps=0.0), dict(eps=float("inf")), dict(x=18), dict(branch=17),
    dict(gate=18), dict(scale=2), dict(w=3), dict(xn=-1), dict(gb=-1), dict(rn=23), dict(rb=24),
    dict(on=0), dict(ob=119)])
def test_gated_residual_norm_entry_refusals(bad):
    with pytest.raises(ValueError):
        _lib.call("recap_gated_residual_norm", *{**GOOD_ROWS, **bad}.values(), None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(out=None), dict(xt=_lib.RECAP_F16), dict(norm=0), dict(eps=-1.0), dict(out=17),
    dict(on=23), dict(sb=-1), dict(bias=17)])
def test_norm_modulate_entry_refusals(bad):
    names = ["x", "xt", "batch", "tokens", "width", "xb", "xn", "scale", "sb", "sn", "shift", "hb", "hn",
             "mt", "w", "bias", "wt", "norm", "eps", "out", "t", "ob", "on"]
    a = {**GOOD_ROWS, **bad}
    with pytest.raises(ValueError):
        _lib.call("recap_norm_modulate", *(a[n] for n in names), None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(branch=None), dict(r=None), dict(post=3), dict(post=0), dict(rb=119),
    dict(mt=_lib.RECAP_F16), dict(eps=0.0)])
def test_gated_residual_entry_refusals(bad):
    names = ["x", "xt", "batch", "tokens", "width", "xb", "xn", "branch", "t", "bb", "bn", "gate", "gb",
             "gn", "mt", "bw", "bbias", "wt", "post", "eps", "r", "rb", "rn"]
    a = {**GOOD_ROWS, **bad}
    with pytest.raises(ValueError):
        _lib.call("recap_gated_residual", *(a[n] for n in names), None)


def test_attention_block_checks_its_grid():
    """Axes of another grid than the layout's, and a stream of another length, are refused."""
    from recap_amd.layout import Layout, SparseGeometry, hilbert_permutation
    layout = Layout.from_permutation(hilbert_permutation((2, 3, 4)), text_tokens=6, text_first=False)
    op = recap_amd.Operator.build(recap_amd.OperatorConfig(), SparseGeometry.build(layout, 128),
                                  n_layers=1)
    same = lambda y: y  # noqa: E731
    block = recap_amd.AttentionBlock(op, 0, 1, same, same, same, same,
                                     axes=recap_amd.rotary_axes((2, 3, 3), (16, 24, 24)))
    with pytest.raises(ValueError, match="video tokens"):
        block(torch.zeros(1, 30, 64, dtype=BF))
    with pytest.raises(ValueError, match="sequence"):
        block(torch.zeros(1, 29, 64, dtype=BF))
