"""Row operators at their edges: gradients at an h that is stored in 16 bits, and calls whose answers once were wrong.  Definitions and
bounds are those of tests/test_row_ops.py."""
import os
import subprocess
import sys

import pytest
import torch

from fiery_amd import native, row_ops
from tests.test_row_ops import BF16, F16, F32, U, check_stored, depth, kept, make, norm64, on, philox, skip_long, xhat_error  # noqa: F401


# ---- gradients of the joined operator at the h before its rounding -----------------------------------------------------------
def grads_near(dy, h, off, weight, eps, dh):
    """64-bit gradients at h and the bounds of 32-bit ones whose h is up to `off` away, as test_row_ops.norm_grads.  What off adds, to
    first order: a row's rstd moves by rstd^2 mean(|xhat| (off + mean off)), which xhat and the gradient are multiples of."""
    mean, rstd, xhat = norm64(h, weight, None, eps)
    w = weight.double().cpu()
    moved = rstd * (xhat.abs() * (off + off.mean(-1, keepdim=True))).mean(-1, keepdim=True)
    d, ex = depth(h.shape[-1]), xhat_error(h, mean, rstd, xhat, off) + xhat.abs() * moved
    gg = dy * w
    m1, m2 = gg.mean(-1, keepdim=True), (gg * xhat).mean(-1, keepdim=True)
    e1 = (d + 2) * U * gg.abs().mean(-1, keepdim=True)
    e2 = (d + 3) * U * (gg * xhat).abs().mean(-1, keepdim=True) + (gg.abs() * ex).mean(-1, keepdim=True)
    norm = rstd * (gg - (m1 + xhat * m2))
    tol = rstd * (2 * U * gg.abs() + e1 + xhat.abs() * e2 + ex * m2.abs() + 4 * U * (m1.abs() + (xhat * m2).abs())) + ((d / 2 + 8) * U + moved) * norm.abs()
    if dh is not None:
        norm = norm + dh
        tol = tol + 2 * U * (norm.abs() + dh.abs())
    lead = tuple(range(h.dim() - 1))
    rows = h.numel() // h.shape[-1]
    dw, db = (dy * xhat).sum(lead), dy.sum(lead)
    return (norm, tol), (dw, (dy.abs() * ex).sum(lead) + (rows + 4) * U * (dy * xhat).abs().sum(lead)), (db, (rows + 4) * U * dy.abs().sum(lead))


def join_case(on, shape, dtype, params, seed=30, shift=0.5, pad=0):  # noqa: F811
    x, r = make(shape, dtype, on.device, seed, 1.5, pad=pad).requires_grad_(), make(shape, dtype, on.device, seed + 1, 1.0, shift, pad=pad).requires_grad_()
    w, b = make(shape[-1:], params, on.device, seed + 2, 0.3, 1.0).requires_grad_(), make(shape[-1:], params, on.device, seed + 3, 0.3).requires_grad_()
    return x, r, w, b, make(shape, dtype, on.device, seed + 4), make(shape, dtype, on.device, seed + 5)


@pytest.mark.parametrize('per,p', [('element', 0.3), ('channel', 0.3), ('sample', 0.3), ('element', 0.0)])
@pytest.mark.parametrize('shape,shift,pad', [((1, 1), 0.5, 0), ((3, 7), 0.5, 3), ((4, 5, 35), 0.5, 0), ((9, 64), 60.0, 8), ((2, 3, 200), 20.0, 1), ((40, 3, 24), 0.5, 0),
                                             ((2, 1000), 0.5, 5), ((3, 2049), 0.5, 0), ((1, 8201), 0.5, 0), ((2, 16400), 0.5, 0)], ids=str)
@pytest.mark.parametrize('dtype,params', [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)], ids=str)
def test_gradients_at_the_unrounded_sum(on, per, p, shape, shift, pad, dtype, params):  # noqa: F811
    """keep='inputs': dweight and the others are those of the h that y comes from, at 32-bit accuracy, however far the rows' mean is from
    zero; y and h are what they are with keep='h'."""
    skip_long(on, shape[-1] > 8201 or shape[-1] > 2000 and (per != 'element' or p == 0.0 or dtype is not BF16 or params is not F32))
    seed, eps = 1 << 50, 1e-3
    rng = row_ops.dropout_rng(seed, on.device)
    x, r, w, b, dy, dh = join_case(on, shape, dtype, params, shift=shift, pad=pad)
    call = lambda keep: row_ops.dropout_add_layer_norm(x, r, w, b, p, rng, call=3, per=per, eps=eps, keep=keep, lib=on.lib)
    y, h = call('inputs')
    other = call('h')
    assert torch.equal(y, other[0]) and torch.equal(h, other[1])
    m = kept(shape, p, seed, 3, per)
    dropped = x.detach().double().cpu() * m
    h64 = dropped + r.detach().double().cpu()
    off = 3 * U * (dropped.abs() + h64.abs())
    rng[1] += 17
    g64, dh64 = dy.double().cpu(), dh.double().cpu()
    total, gw, gb = grads_near(g64, h64, off, w.detach(), eps, dh64)
    dx, dr, dw, db = torch.autograd.grad((y, h), (x, r, w, b), (dy, dh), retain_graph=True)
    check_stored(dr, total)
    check_stored(dx, (total[0] * m, total[1] * m + 2 * U * (total[0] * m).abs()))
    check_stored(dw, gw)
    check_stored(db, gb)
    only_y, _, _ = grads_near(g64, h64, off, w.detach(), eps, None)
    check_stored(torch.autograd.grad(y, r, dy, retain_graph=True)[0], only_y)
    check_stored(torch.autograd.grad(y, w, dy, retain_graph=True)[0], gw)
    dx, dr = torch.autograd.grad(h, (x, r), dh, retain_graph=True)
    assert torch.equal(dr, dh)
    check_stored(dx, (dh64 * m, 2 * U * (dh64 * m).abs()))


def test_a_sum_past_the_largest_16_bit_value_keeps_its_gradients(on):  # noqa: F811
    """60,000 + 60,000 is infinite in fp16: y is finite, and so are the gradients of keep='inputs'."""
    x, r, w, b, dy, _ = join_case(on, (4, 40), F16, F32)
    with torch.no_grad():
        x[1], r[1] = 60000.0, 60000.0
        r[1, ::2] = 40000.0
    y, h = row_ops.dropout_add_layer_norm(x, r, w, b, keep='inputs', lib=on.lib)
    assert torch.isinf(h[1, 1]) and torch.isfinite(y).all()
    h64 = x.detach().double().cpu() + r.detach().double().cpu()
    total, gw, gb = grads_near(dy.double().cpu(), h64, 2 * U * h64.abs(), w.detach(), 1e-5, None)
    dx, dr, dw, db = torch.autograd.grad(y, (x, r, w, b), dy)
    check_stored(dx, total)
    check_stored(dr, total)
    check_stored(dw, gw)
    check_stored(db, gb)


def test_a_32_bit_stream_is_the_same_either_way(on):  # noqa: F811
    for dtype in (F32, BF16, F16):
        x, r = make((5, 70), dtype, on.device, 50).requires_grad_(), make((5, 70), F32, on.device, 51).requires_grad_()
        w, dy = make((70,), F32, on.device, 52, 0.2, 1.0).requires_grad_(), make((5, 70), dtype, on.device, 53)
        rng = row_ops.dropout_rng(9, on.device)
        got = []
        for keep in ('h', 'inputs'):
            y, h = row_ops.dropout_add_layer_norm(x, r, w, None, 0.4, rng, keep=keep, lib=on.lib)
            got.append([y, h, *torch.autograd.grad(y, (x, r, w), dy)])
        assert all(torch.equal(p, q) for p, q in zip(*got))


def test_what_is_kept_and_refused(sim):
    """keep='inputs' notices a changed input; other words and entry points without a 16-bit stream are refused."""
    x, r = torch.ones(3, 16, dtype=BF16).requires_grad_(), torch.ones(3, 16, dtype=BF16)
    z = x * 2.0
    y, h = row_ops.dropout_add_layer_norm(z, r, keep='inputs', lib=sim)
    h += 1.0                                                       # h is no longer what the backward pass reads
    torch.autograd.grad(y.float().sum(), x, retain_graph=True)
    z += 1.0
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.float().sum().backward()
    with pytest.raises(ValueError, match='keep'):
        row_ops.dropout_add_layer_norm(x, r, keep='x', lib=sim)
    p = torch.zeros(64).data_ptr()
    bwd = lambda x=p, res=p, t=1, x_ld=8: sim.check(sim.dll.fiery_dropout_add_layer_norm_bwd_unrounded(
        p, 8, None, 0, x, x_ld, res, 8, t, 2, 8, p, t, p, p, 0, None, 1, 0, p, 8, p, 8, None, None, None, 0, None))
    for kw in (dict(x=None), dict(res=None), dict(t=0), dict(t=3), dict(x_ld=-1)):
        with pytest.raises(native.NativeError):
            bwd(**kw)


@pytest.mark.parametrize('where', ['end', 'begin'])
def test_the_unrounded_kernels_stay_inside_their_operands(sim, where):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, os.path.join(root, 'tests', 'sim', 'guard_unrounded.py'), where], cwd=root, capture_output=True, text=True, timeout=900)
    assert res.returncode == 0 and f'ok unrounded {where} (' in res.stdout, res.stdout[-1500:] + res.stderr[-3000:]


# ---- means whose sums round ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('c', [1, 3, 8, 72, 300, 513, 1000, 2049, 8200])
@pytest.mark.parametrize('value', [0.1, -1000.1, 12345.678, 1e30, -1e36])
def test_a_constant_row_is_its_bias(on, c, value):  # noqa: F811
    """The sum of equal values is rounded, its mean is not: y is the bias exactly (v - v = 0), and dx is rstd (g - mean g) with
    rstd = 1 / sqrt(eps), as test_row_ops.norm_grads bounds it; neighbours of ordinary values are what they are without it."""
    skip_long(on, c > 2049)
    x = make((5, c), F32, on.device, 60, 2.0, 0.5)
    alone = x[[0, 4]].clone()
    x[1], x[3] = value, value
    leaf, w, b = x.clone().requires_grad_(), make((c,), F32, on.device, 61, 0.2, 1.0), make((c,), F32, on.device, 62)
    dy = make((5, c), F32, on.device, 63)
    y = row_ops.layer_norm(leaf, w, b, lib=on.lib)
    assert torch.equal(y[1], b) and torch.equal(y[3], b)
    assert torch.equal(y[[0, 4]], row_ops.layer_norm(alone, w, b, lib=on.lib))
    dx, = torch.autograd.grad(y, leaf, dy)
    g = dy[[1, 3]].double().cpu() * w.double().cpu()
    want = (g - g.mean(-1, keepdim=True)) / 1e-5 ** 0.5
    # xhat is 0: rstd's own error (3 u), the row mean's (DEPTH + 2) u, the products'
    tol = ((depth(c) + 2) * U * g.abs().mean(-1, keepdim=True) + 4 * U * g.abs()) / 1e-5 ** 0.5 + 8 * U * want.abs()
    check_stored(dx[[1, 3]], (want, tol))


@pytest.mark.parametrize('c', [24, 72, 1000])
@pytest.mark.parametrize('dtype,stream', [(F32, F32), (BF16, BF16), (F16, F16), (F16, F32)], ids=str)
def test_a_constant_sum_is_its_bias(on, c, dtype, stream):  # noqa: F811
    """The joined operator's statistics, both those of y and those that are kept: constant rows have xhat 0 in each."""
    value = 1000.1 if dtype is F32 else 12.3
    x, r = make((4, c), dtype, on.device, 64), make((4, c), stream, on.device, 65)
    x[2], r[2] = value, value / 3
    x, r, b = x.requires_grad_(), r.requires_grad_(), make((c,), dtype, on.device, 66)
    w = torch.ones(c, dtype=dtype, device=on.device, requires_grad=True)
    for keep in ('h', 'inputs'):
        y, h = row_ops.dropout_add_layer_norm(x, r, w, b, keep=keep, lib=on.lib)
        assert torch.equal(y[2], b)
        dy = torch.zeros(4, c, dtype=dtype, device=on.device)
        dy[2] = 1.0
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        assert not dw.any()                                        # dy xhat, xhat 0
        assert not dx[[0, 1, 3]].any()
        # (g - mean g) of equal g: the mean's rounding, (DEPTH + 2) u, over sqrt(eps); and its own rounding when it is stored
        assert float(dx[2].abs().max()) <= (depth(c) + 2) * U / 1e-5 ** 0.5 * 1.01


def test_a_mean_far_above_the_spread(on):  # noqa: F811
    """One value of c is a step (2^-10) above the others, 12345.678: the mean lies a c-th of a step above them and is rounded to them, so
    values are off by step / c, and the variance, (1 - 1/c) / c steps^2, by its c-th at most."""
    for c in (72, 513, 1000):
        x = torch.full((1, c), 12345.678, device=on.device)
        x[0, 5] += 2.0 ** -10
        y = row_ops.layer_norm(x, None, None, 1e-12, lib=on.lib).double().cpu()
        mean, rstd, xhat = norm64(x.double().cpu(), None, None, 1e-12)
        assert ((y - xhat).abs() <= 1.01 * (rstd * 2.0 ** -10 / c + xhat.abs() / c)).all(), c


# ---- calls that the operators do not provide are errors ------------------------------------------------------------------------
def _ops(lib, rng):
    """Each operator as a function of one tensor, its other operands plain."""
    return {'layer_norm': lambda t: row_ops.layer_norm(t, lib=lib), 'dropout': lambda t: row_ops.dropout(t, 0.5, rng, lib=lib),
            'joined': lambda t: row_ops.dropout_add_layer_norm(t, torch.ones_like(t), p=0.5, rng=rng, lib=lib)[0]}


@pytest.mark.parametrize('name', ['layer_norm', 'dropout', 'joined'])
def test_forward_mode_derivatives_are_refused(sim, name):
    """A tangent on any operand is an error, with and without a parameter that requires a gradient; it never comes out as zero."""
    import torch.autograd.forward_ad as fwd
    rng, x, w = row_ops.dropout_rng(0, 'cpu'), make((4, 16), F32, 'cpu', 70), make((16,), F32, 'cpu', 71)
    op = _ops(sim, rng)[name]
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        p, learnt = fwd.make_dual(w, torch.ones_like(w)), w.clone().requires_grad_()
        norm, drop, join = row_ops.layer_norm, row_ops.dropout, row_ops.dropout_add_layer_norm
        calls = [lambda: op(dual)] + {
            'layer_norm': [lambda: norm(x, p, w, lib=sim), lambda: norm(x, w, p, lib=sim), lambda: norm(dual, learnt, lib=sim)],
            'dropout': [lambda: drop(x, 0.5, rng, residual=dual, lib=sim), lambda: drop(dual, 0.5, rng, residual=x.clone().requires_grad_(), lib=sim)],
            'joined': [lambda: join(x, x, p, w, lib=sim), lambda: join(x, x, w, p, lib=sim), lambda: join(x, dual, lib=sim), lambda: join(x, dual, learnt, lib=sim)],
        }[name]
        for call in calls:
            with pytest.raises(RuntimeError, match='forward-mode'):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match='forward-mode'):
            op(dual)                                               # tangents live under no_grad too
        with fwd._set_fwd_grad_enabled(False):
            assert torch.equal(op(dual), op(x))                    # nobody asks for one
        assert torch.equal(op(fwd.unpack_dual(dual).primal), op(x))


@pytest.mark.parametrize('name', ['layer_norm', 'dropout', 'joined'])
def test_tracing_is_refused(sim, name):
    """A traced function would hold an allocation and no launch: torch.jit.trace, make_fx (before dispatch too) and torch.export are
    errors, in the backward pass as well.  Modes that only watch the calls are not tracing."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    op, x = _ops(sim, row_ops.dropout_rng(0, 'cpu'))[name], make((4, 16), F32, 'cpu', 72)

    class Module(torch.nn.Module):
        def forward(self, t):
            return op(t) + 1
    with pytest.raises(RuntimeError, match='tracing'):
        torch.jit.trace(lambda t: op(t) + 1, (x,), check_trace=False)
    for kw in ({}, dict(pre_dispatch=True)):
        with pytest.raises(RuntimeError, match='tracing'):
            make_fx(lambda t: op(t) + 1, **kw)(x)
    with pytest.raises(RuntimeError):                              # fake tensors have no memory, whoever notices first
        make_fx(lambda t: op(t) + 1, tracing_mode='fake')(x)
    with pytest.raises(Exception):
        torch.export.export(Module(), (x,), strict=False)
    leaf = x.clone().requires_grad_()
    y = op(leaf)
    with pytest.raises(RuntimeError, match='tracing'):
        make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True)[0])(x)
    with FlopCounterMode(display=False):
        assert torch.equal(op(x), y.detach())


def test_compiled_functions_break_around_the_operators(sim):
    x = make((4, 16), F32, 'cpu', 73)
    for op in _ops(sim, row_ops.dropout_rng(0, 'cpu')).values():
        assert torch.equal(torch.compile(lambda t: op(t * 2) + 1, backend='eager')(x), op(x * 2) + 1)


# ---- tensors whose memory is not their values ----------------------------------------------------------------------------------
def test_negative_views_are_read_as_their_values(on):  # noqa: F811
    """A tensor with the negative bit (the imaginary part of a conjugate) as each operand, the mask's numbers and an incoming gradient."""
    neg = lambda t: torch._neg_view(-t)                            # t's values over the memory of -t
    x, r, w, b = make((3, 5, 16), F32, on.device, 74), make((3, 5, 16), F32, on.device, 75), make((16,), F32, on.device, 76), make((16,), F32, on.device, 77)
    rng = row_ops.dropout_rng(6, on.device) + 3
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    norm, drop, join = row_ops.layer_norm, row_ops.dropout, row_ops.dropout_add_layer_norm
    want = norm(x, w, b, lib=on.lib)
    for args in ((neg(x), w, b), (x, neg(w), b), (x, w, neg(b))):
        assert torch.equal(norm(*args, lib=on.lib), want)
        leaf = args[0].detach().requires_grad_()
        assert torch.equal(norm(leaf, *args[1:], lib=on.lib), want)
    assert torch.equal(drop(neg(x), 0.0, lib=on.lib), x)
    want = drop(x, 0.5, rng, residual=r, lib=on.lib)
    for a, g, s in ((neg(x), rng, r), (x, neg(rng), r), (x, rng, neg(r))):
        assert torch.equal(drop(a, 0.5, g, residual=s, lib=on.lib), want)
    want = join(x, r, w, b, 0.5, rng, lib=on.lib)
    for a, s, p, q, g in ((neg(x), r, w, b, rng), (x, neg(r), w, b, rng), (x, r, neg(w), b, rng), (x, r, w, neg(b), rng), (x, r, w, b, neg(rng))):
        assert all(torch.equal(u, v) for u, v in zip(join(a, s, p, q, 0.5, g, lib=on.lib), want))
        got = join(a.detach().requires_grad_(), s, p, q, 0.5, g, lib=on.lib)
        assert all(torch.equal(u, v) for u, v in zip(got, want))
    one = make((7, 1), F32, on.device, 78)                         # (a column at any stride is read in place)
    assert torch.equal(drop(neg(one), 0.0, lib=on.lib), one)

    dy, dh = make((3, 5, 16), F32, on.device, 79), make((3, 5, 16), F32, on.device, 80)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y = norm(leaves[0], leaves[2], lib=on.lib)
    grads = lambda out, of, g: torch.autograd.grad(out, of, g, retain_graph=True)
    for out, of, g, n in ((y, (leaves[0], leaves[2]), (dy,), (neg(dy),)), (drop(leaves[0], 0.5, rng, residual=leaves[1], lib=on.lib), leaves[:2], (dy,), (neg(dy),)),
                          (join(*leaves, p=0.5, rng=rng, lib=on.lib), leaves, (dy, dh), (neg(dy), neg(dh))),
                          (join(*leaves, p=0.5, rng=rng, lib=on.lib)[1], leaves[:2], (dh,), (neg(dh),))):
        assert all(torch.equal(u, v) for u, v in zip(grads(out, of, g), grads(out, of, n)))


def test_tensors_without_memory_are_refused(sim):
    """Fake and zero tensors have no memory: an error, not an operand that is taken as absent (a residual that is not added, a weight of
    ones) nor an address handed to a kernel."""
    from torch._subclasses import FakeTensorMode
    fake = FakeTensorMode()
    x, w, rng = make((4, 16), F32, 'cpu', 81), make((16,), F32, 'cpu', 82), row_ops.dropout_rng(1, 'cpu')
    norm, drop, join = row_ops.layer_norm, row_ops.dropout, row_ops.dropout_add_layer_norm
    for empty in (lambda t: fake.from_tensor(t), lambda t: torch._efficientzerotensor(t.shape, dtype=t.dtype)):
        for call in (lambda: norm(empty(x), lib=sim), lambda: norm(x, empty(w), lib=sim), lambda: norm(x, w, empty(w), lib=sim), lambda: drop(empty(x), 0.0, lib=sim),
                     lambda: drop(x, 0.0, residual=empty(x), lib=sim), lambda: drop(x, 0.5, empty(rng), lib=sim), lambda: join(empty(x), x, lib=sim),
                     lambda: join(x, empty(x), lib=sim), lambda: join(x, x, empty(w), w, lib=sim), lambda: join(x, x, w, empty(w), lib=sim),
                     lambda: join(x, x, w, w, 0.5, empty(rng), lib=sim)):
            with pytest.raises(RuntimeError):
                call()
    assert norm(torch.zeros(0, 16), w, lib=sim).shape == (0, 16)   # no rows need no memory


# ---- columns that are none -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('c', [9, 16, 24, 35, 72, 520, 1032, 2049, 2056, 8200, 8201])
def test_gradients_of_far_rows_do_not_depend_on_the_width(on, c):  # noqa: F811
    """|mean| rstd past the largest fp32 value: what the lanes behind a row's last column hold stays out of its sums, whether the width
    fills its lanes (16) or not.  Rows of 1e33 with eps 1e-12 have xhat 0: dx = rstd (g - mean g), dweight takes nothing from them."""
    skip_long(on, c > 2056)
    x = make((4, c), F32, on.device, 83)
    x[1], x[2] = 1e33, -1e33
    leaf, w, dy = x.requires_grad_(), make((c,), F32, on.device, 84, 0.2, 1.0).requires_grad_(), make((4, c), F32, on.device, 85)
    y = row_ops.layer_norm(leaf, w, None, 1e-12, lib=on.lib)
    dx, dw = torch.autograd.grad(y, (leaf, w), dy)
    g = dy[1:3].double().cpu() * w.detach().double().cpu()
    want = (g - g.mean(-1, keepdim=True)) * 1e6
    check_stored(dx[1:3], (want, ((depth(c) + 2) * U * g.abs().mean(-1, keepdim=True) + 4 * U * g.abs()) * 1e6 + 8 * U * want.abs()))
    near = [0, 3]
    check_stored(dw, grads_near(dy[near].double().cpu(), x[near].detach().double().cpu(), torch.zeros(2, c, dtype=torch.float64), w.detach(), 1e-12, None)[1])
    if c <= 2049:
        r = torch.zeros(4, c, device=on.device)
        y, h = row_ops.dropout_add_layer_norm(leaf, r, w, eps=1e-12, lib=on.lib)
        assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], dx)


# ---- sizes at the ends of the stated range -------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_the_widest_parameters_gradient(hip):
    """2^26 + 13 columns: sixteen of them to a workgroup of 1024 work-items are more than the 2^32 that a launch may have.  The first
    and last columns are those of the definition over rows of two values (x = +-1 in turns: mean and spread known)."""
    c = (1 << 26) + 13
    sign = torch.ones(c, dtype=BF16, device='cuda')
    sign[1::2] = -1.0
    x = torch.stack((sign, -sign)).requires_grad_()
    w = torch.ones(c, dtype=BF16, device='cuda', requires_grad=True)
    b = torch.zeros(c, dtype=BF16, device='cuda', requires_grad=True)
    y = row_ops.layer_norm(x, w, b, 0.0)
    dy = torch.ones_like(y)
    dy[1] = 2.0
    dw, db = torch.autograd.grad(y, (w, b), dy)
    # mean = +-1 / c (an odd count) and rstd = 1: xhat = x to 2^-26; dweight = 1 x - 2 x = -x, dbias = 1 + 2
    assert torch.equal(dw, -sign) and torch.equal(db, torch.full_like(db, 3.0))


@pytest.mark.parametrize('per', ['element', 'channel', 'sample'])
@pytest.mark.parametrize('dtype,stream', [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)], ids=str)
def test_the_gradient_of_h_alone_at_the_entry_point(on, per, dtype, stream):  # noqa: F811
    """dy null: only h went on; dx is the dropout of dh, the mask that of the forward pass."""
    shape, lib = (3, 4, 21), native.get() if on.device == 'cuda' else on.lib
    rng, dh = row_ops.dropout_rng(5, on.device), make(shape, stream, on.device, 86)
    dx = torch.empty(shape, dtype=dtype, device=on.device)
    t, s, share = native.ROW_TYPES[dtype], native.ROW_TYPES[stream], 1 if per == 'element' else 4
    at = torch.cuda.current_stream().cuda_stream if on.device == 'cuda' else None
    call = lambda dy=None, dh=dh.data_ptr(), dres=None, dg=None: lib.check(lib.dll.fiery_dropout_add_layer_norm_bwd(
        dy, 21, dh, 21, None, 0, t, s, 12, 21, None, 0, None, None, 19661, rng.data_ptr(), share, per == 'sample', dx.data_ptr(), 21, dres, 21, dg, None, None, 0, at))
    call()
    want = dh.double().cpu() * kept(shape, 19661 / 65536, 5, 0, per)
    check_stored(dx, (want, 2 * U * want.abs()))
    if on.device == 'cpu':
        p = torch.zeros(300).data_ptr()
        for kw in (dict(dh=None), dict(dy=p), dict(dres=p), dict(dg=p)):
            with pytest.raises(native.NativeError):
                call(**kw)


@pytest.mark.gpu
def test_the_gradient_of_h_alone_past_two_billion_units(hip):
    """2^30 + 5 rows of nine columns are 2^31 + 10 units of eight: the forward pass takes them, and so does the gradient of h alone."""
    rows, c = (1 << 30) + 5, 9
    x = make((1, c), BF16, 'cuda', 87).expand(rows, c).requires_grad_()
    dh = make((1, c), BF16, 'cuda', 88).expand(rows, c)
    rng = row_ops.dropout_rng(13, 'cuda')
    y, h = row_ops.dropout_add_layer_norm(x, x.detach(), p=0.5, rng=rng)
    del y
    dx, = torch.autograd.grad(h, x, dh)
    for first in (0, (1 << 30) - 4, rows - 7):
        words = [[v >> 16 * k & 0xffff for unit in range(2) for v in philox([unit, first + i, 0, 0], [13, 0]) for k in range(2)][:c] for i in range(7)]
        keep = torch.tensor(words, device='cuda') >= 32768
        assert torch.equal(dx[first:first + 7], torch.where(keep, dh[:7] * 2, torch.zeros_like(dh[:7]))), first
    assert torch.equal(h[-7:], x.detach()[:7] + torch.where(keep, x.detach()[:7] * 2, torch.zeros_like(dh[:7])))


# ---- the two libraries ---------------------------------------------------------------------------------------------------------
def test_nodes_built_against_another_header_are_refused(sim, monkeypatch):
    """The nodes call the library by address with their own header's signatures: a stale build is an error, as a stale library is."""
    import types
    old = types.SimpleNamespace(abi_version=native.ABI_VERSION - 1, rows_of=None)
    monkeypatch.setattr(row_ops, '_nodes', None)
    monkeypatch.setitem(sys.modules, 'fiery_amd._row_autograd', old)
    monkeypatch.setattr('fiery_amd._row_autograd', old, raising=False)
    with pytest.raises(native.NativeError, match='ABI'):
        row_ops.layer_norm(torch.ones(2, 8), lib=sim)
    monkeypatch.setitem(sys.modules, 'fiery_amd._row_autograd', types.SimpleNamespace(rows_of=None))
    monkeypatch.delattr('fiery_amd._row_autograd', raising=False)
    with pytest.raises(native.NativeError, match='ABI'):           # from before the number was there
        row_ops.layer_norm(torch.ones(2, 8), lib=sim)


def test_a_graph_outlives_the_library_object_it_was_made_with(sim):
    """Nodes keep the address of the library's table of entry points: it stays, whatever becomes of the object that made it."""
    import gc
    import weakref
    lib = native.Lib(sim.path)
    x = make((4, 24), F32, 'cpu', 90).requires_grad_()
    dy = make((4, 24), F32, 'cpu', 91)
    y = row_ops.layer_norm(x, lib=lib)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    table, gone = weakref.ref(lib._row_entries), weakref.ref(lib)
    del lib
    gc.collect()
    assert gone() is None and table() is not None
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)


def _timed_step(lib, device):
    x, r = make((4, 24), F32, device, 92).requires_grad_(), make((4, 24), F32, device, 93).requires_grad_()
    w, rng = make((24,), F32, device, 94, 0.2, 1.0).requires_grad_(), row_ops.dropout_rng(3, device)
    y, h = row_ops.dropout_add_layer_norm(row_ops.layer_norm(x, w, lib=lib), row_ops.dropout(r, 0.3, rng, lib=lib), w, p=0.2, rng=rng, call=1, lib=lib)
    return [y, h, *torch.autograd.grad((y, h), (x, r, w), (make((4, 24), F32, device, 95), make((4, 24), F32, device, 96)))]


def test_the_call_table_sees_the_row_operators(on, monkeypatch):  # noqa: F811
    """native.CALL_SINK: forward and backward launches of the row operators are filed as the library's others are, and compute what they do
    without it; a graph that was made with the table open works when it is closed again."""
    if on.device == 'cpu':                                         # (no events there: stand-ins)
        class Event:
            def __init__(self, enable_timing):
                self.recorded = 0

            def record(self):
                self.recorded += 1
        monkeypatch.setattr(torch.cuda, 'is_available', lambda: True)
        monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
        monkeypatch.setattr(torch.cuda, 'Event', Event)
    want = _timed_step(on.lib, on.device)
    monkeypatch.setattr(native, 'CALL_SINK', [])
    got = _timed_step(on.lib, on.device)
    names = [name for name, _, _ in native.CALL_SINK]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert sorted(names) == sorted(['fiery_layer_norm_fwd', 'fiery_dropout', 'fiery_dropout_add_layer_norm_fwd', 'fiery_dropout_add_layer_norm_bwd',
                                    'fiery_layer_norm_bwd', 'fiery_dropout'])
    if on.device == 'cuda':
        torch.cuda.synchronize()
        assert all(start.elapsed_time(end) >= 0.0 for _, start, end in native.CALL_SINK)
    leaf = make((4, 24), F32, on.device, 97).requires_grad_()
    y = row_ops.layer_norm(leaf, lib=on.lib)
    monkeypatch.setattr(native, 'CALL_SINK', None)
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(dx, torch.autograd.grad(row_ops.layer_norm(leaf, lib=on.lib), leaf, torch.ones_like(y))[0])


@pytest.mark.gpu
def test_a_captured_step_at_the_unrounded_sum(hip):
    """keep='inputs' forward and backward in one hipGraph, rows of which some are constant (their squares are taken twice): every replay
    equals the eager step of its numbers bit for bit, with eager work in between."""
    for shape in ((60, 50, 64), (200, 2056), (30, 9000)):
        x, r, w, b, dy, dh = [t.detach() for t in join_case(type('On', (), dict(device='cuda')), shape, BF16, F32)]
        x[3], r[3] = 12.3, 4.1

        def step(rng):
            leaves = [t.detach().requires_grad_() for t in (x, r, w, b)]
            y, h = row_ops.dropout_add_layer_norm(*leaves, 0.3, rng, keep='inputs')
            grads = torch.autograd.grad((y, h), leaves, (dy, dh))
            rng[1:].add_(1)
            return [y.detach(), h.detach(), *grads]
        rng, eager = row_ops.dropout_rng(8, 'cuda'), row_ops.dropout_rng(8, 'cuda')
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(rng)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(rng)
        eager[1] += 1
        for _ in range(3):
            graph.replay()
            want = step(eager)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want)) and torch.equal(rng, eager)
