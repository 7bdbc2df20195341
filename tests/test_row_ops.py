"""Row operators (fiery_amd/row_ops.py) against plain implementations in 64 bits: the kernel sources on the CPU simulator, and the
same cases on the GPU.

Tolerances are first-order bounds, element by element, from the roundings that the formulas contain (u = 2^-24, half = half a
step of the stored type relative to the value):
  a sum of n terms in 32 bits, DEPTH additions deep, is off by at most DEPTH u sum |terms|;
  mean: DEPTH u mean|h|;  variance and rstd: (DEPTH + 4) u and half of it + 3 u, relative;
  xhat: |xhat| (DEPTH / 2 + 6) u + rstd (mean's error + what h itself is off).
Everything else is these carried through the products and sums of the formula."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from fiery_amd import native, row_ops

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: U, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}          # half of the smallest step, or a step


class Backend:
    def __init__(self, lib, device):
        self.lib, self.device = lib, device


@pytest.fixture(params=['sim', pytest.param('gpu', marks=pytest.mark.gpu)])
def on(request):
    if request.param == 'sim':
        return Backend(request.getfixturevalue('sim'), 'cpu')
    return Backend(request.getfixturevalue('hip'), 'cuda')


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 of one counter (four words) under one key (two words), in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xffffffff, (p >> 32) ^ c[3] ^ k[1], p & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def kept(shape, p, seed, call, per):
    """The mask of x (n, ..., C) as a float64 array of factors: 0 or 65536 / (65536 - threshold)."""
    c, rows = shape[-1], int(np.prod(shape[:-1]))
    share = 1 if per == 'element' else rows // max(1, shape[0])
    threshold = round(65536 * p)
    seed, call = seed % 2 ** 64, call % 2 ** 64
    out = np.zeros((rows, c))
    for mask_row in range((rows + share - 1) // share):
        line = []
        for unit in range((c + 7) // 8 if per != 'sample' else 1):
            w = philox([unit, mask_row, call & 0xffffffff, call >> 32], [seed & 0xffffffff, seed >> 32])
            line += [h for x in w for h in (x & 0xffff, x >> 16)]
        line = np.array(line[:c] if per != 'sample' else [line[0]] * c)
        out[mask_row * share:(mask_row + 1) * share] = (line >= threshold) * (65536.0 / max(1, 65536 - threshold))
    return torch.from_numpy(out).view(shape)


def norm64(h, weight, bias, eps):
    mean = h.mean(-1, keepdim=True)
    var = ((h - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    return mean, rstd, (h - mean) * rstd


def depth(c):
    """Additions in a row's sum, an upper bound: a lane's own columns, then 6 exchanges and up to 16 wavefronts."""
    return 8 * max(4, -(-c // 8192)) + 22


def xhat_error(h, mean, rstd, xhat, off):
    d = depth(h.shape[-1])
    return xhat.abs() * (d / 2 + 6) * U + rstd * (d * U * h.abs().mean(-1, keepdim=True) + U * mean.abs() + off + off.mean(-1, keepdim=True))


def check_norm_forward(y, h, weight, bias, eps, off=0.0):
    """y against the 64-bit norm of h; off: how far the h that the kernel normalised may be from this one."""
    off = off if isinstance(off, torch.Tensor) else torch.zeros_like(h)
    mean, rstd, xhat = norm64(h, weight, bias, eps)
    w = torch.ones(h.shape[-1], dtype=torch.float64) if weight is None else weight.double().cpu()
    b = torch.zeros(h.shape[-1], dtype=torch.float64) if bias is None else bias.double().cpu()
    want = xhat * w + b
    tol = w.abs() * xhat_error(h, mean, rstd, xhat, off) + 2 * U * ((xhat * w).abs() + b.abs()) + HALF[y.dtype] * want.abs() * 1.01 + TINY[y.dtype]
    check(y, want, tol)


def check(got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f'{int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol)[bad].max():.3g} of the bound, {(got - want).abs()[bad].max():.3g}'


def norm_grads(dy, h, weight, eps, dh=None):
    """64-bit gradients and their bounds: ((dh', tol), (dweight, tol), (dbias, tol)) before the rounding of what is stored."""
    mean, rstd, xhat = norm64(h, weight, None, eps)
    w = torch.ones(h.shape[-1], dtype=torch.float64) if weight is None else weight.double().cpu()
    d, ex = depth(h.shape[-1]), xhat_error(h, mean, rstd, xhat, torch.zeros_like(h))
    gg = dy * w
    m1, m2 = gg.mean(-1, keepdim=True), (gg * xhat).mean(-1, keepdim=True)
    e1 = (d + 2) * U * gg.abs().mean(-1, keepdim=True)
    e2 = (d + 3) * U * (gg * xhat).abs().mean(-1, keepdim=True) + (gg.abs() * ex).mean(-1, keepdim=True)
    norm = rstd * (gg - (m1 + xhat * m2))
    tol = rstd * (2 * U * gg.abs() + e1 + xhat.abs() * e2 + ex * m2.abs() + 4 * U * (m1.abs() + (xhat * m2).abs())) + (d / 2 + 8) * U * norm.abs()
    if dh is not None:
        norm = norm + dh
        tol = tol + 2 * U * (norm.abs() + dh.abs())
    lead = tuple(range(h.dim() - 1))
    rows = h.numel() // h.shape[-1]
    dw, db = (dy * xhat).sum(lead), dy.sum(lead)
    return ((norm, tol), (dw, (dy.abs() * ex).sum(lead) + (rows + 4) * U * (dy * xhat).abs().sum(lead)), (db, (rows + 4) * U * dy.abs().sum(lead)))


def check_stored(got, pair):
    want, tol = pair
    check(got, want, tol + HALF[got.dtype] * (want.abs() + tol) * 1.01 + TINY[got.dtype])


def make(shape, dtype, device, seed, spread=1.0, shift=0.0, pad=0):
    """Seeded values; pad > 0: a slice of wider rows whose other values are NaN."""
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(*shape, generator=g) * spread + shift).to(dtype)
    wide = torch.full((*shape[:-1], shape[-1] + pad), float('nan'), dtype=dtype)
    wide[..., :shape[-1]] = t
    return wide.to(device)[..., :shape[-1]]


def skip_long(on, long):
    if long and on.device == 'cpu':
        pytest.skip('long rows take seconds each on the simulator: a few there, all on the GPU')


# ---- layer norm ------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (4, 1), (3, 2), (5, 3), (9, 7), (1, 8), (70, 8), (3, 9), (2, 3, 35), (33, 64), (2, 5, 70), (4, 200), (3, 513), (2, 1000), (3, 1024),
          (2, 1025), (1, 2048), (3, 2056), (2, 4096), (2, 4101), (1, 8200), (2, 16384), (1, 16385), (1, 32768), (2, 32777)]


@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype,params', [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)], ids=str)
def test_layer_norm_and_its_gradients(on, shape, dtype, params):
    skip_long(on, shape[-1] > 8200 or shape[-1] > 4200 and dtype is not F32)
    x = make(shape, dtype, on.device, 1, 1.5, 0.4).requires_grad_()
    w, b = make(shape[-1:], params, on.device, 2, 0.3, 1.0).requires_grad_(), make(shape[-1:], params, on.device, 3, 0.3).requires_grad_()
    dy = make(shape, dtype, on.device, 4)
    y = row_ops.layer_norm(x, w, b, 1e-5, lib=on.lib)
    assert y.dtype is dtype and y.is_contiguous()
    h = x.detach().double().cpu()
    check_norm_forward(y, h, w.detach(), b.detach(), 1e-5)
    with torch.no_grad():
        assert torch.equal(row_ops.layer_norm(x, w, b, 1e-5, lib=on.lib), y)                  # the serving form: no statistics kept
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    gx, gw, gb = norm_grads(dy.double().cpu(), h, w.detach(), 1e-5)
    for got, like, want in ((dx, x, gx), (dw, w, gw), (db, b, gb)):
        assert got.dtype is like.dtype
        check_stored(got, want)


@pytest.mark.parametrize('rows,c', [(9000, 8), (1000, 8), (257, 40), (131, 1024), (37, 2048), (35, 3000), (50, 16400)])
def test_layer_norm_sums_over_many_rows(on, rows, c):
    """More rows than one pass of the workgroups: partial rows of the parameters' gradients and their sum; the same bits twice."""
    skip_long(on, c > 16000)
    x, dy = make((rows, c), F32, on.device, 5, 2.0, -1.0).requires_grad_(), make((rows, c), F32, on.device, 6)
    w, b = make((c,), F32, on.device, 7, 0.2, 1.0).requires_grad_(), make((c,), F32, on.device, 8).requires_grad_()
    got = torch.autograd.grad(row_ops.layer_norm(x, w, b, lib=on.lib), (x, w, b), dy)
    h = x.detach().double().cpu()
    for g, want in zip(got, norm_grads(dy.double().cpu(), h, w.detach(), 1e-5)):
        check_stored(g, want)
    again = torch.autograd.grad(row_ops.layer_norm(x, w, b, lib=on.lib), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize('which', ['none', 'weight', 'bias'])
def test_layer_norm_without_some_parameters_and_gradients(on, which):
    shape = (6, 50)
    x, dy = make(shape, F32, on.device, 9, shift=3.0).requires_grad_(), make(shape, F32, on.device, 10)
    w = make((50,), F32, on.device, 11, 0.2, 1.0).requires_grad_() if which == 'weight' else None
    b = make((50,), F32, on.device, 12).requires_grad_() if which == 'bias' else None
    y = row_ops.layer_norm(x, w, b, lib=on.lib)
    h = x.detach().double().cpu()
    check_norm_forward(y, h, None if w is None else w.detach(), None if b is None else b.detach(), 1e-5)
    gx, gw, gb = norm_grads(dy.double().cpu(), h, None if w is None else w.detach(), 1e-5)
    for leaf, want in ((x, gx), (w, gw), (b, gb)):
        if leaf is not None:                                                                 # one at a time: the others are not computed
            check_stored(torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], want)


@pytest.mark.parametrize('pad', [1, 5, 8])
def test_rows_inside_wider_rows(on, pad):
    """Channel slices of wider rows are read in place: their neighbours (NaN here) neither enter nor change."""
    shape = (3, 4, 37)
    x, dy = make(shape, F32, on.device, 13, pad=pad), make(shape, F32, on.device, 14, pad=pad)
    assert row_ops._rows(x)[0] is x and row_ops._rows(x)[1] == 37 + pad
    leaf = x.detach().requires_grad_()
    y = row_ops.layer_norm(leaf, lib=on.lib)
    check_norm_forward(y, x.double().cpu(), None, None, 1e-5)
    dx, = torch.autograd.grad(y, leaf, dy)
    check_stored(dx, norm_grads(dy.double().cpu(), x.double().cpu(), None, 1e-5)[0])


def test_other_layouts_give_the_same_values(on):
    """An expanded row (stride 0), a transposed tensor (copied), a channels-last image batch and an odd storage offset."""
    base = make((5, 6, 24), F32, on.device, 15)
    want = row_ops.layer_norm(base, lib=on.lib)
    assert torch.equal(row_ops.layer_norm(base.transpose(0, 1), lib=on.lib), want.transpose(0, 1))
    one = base[2, 3].expand(7, 24)
    assert row_ops._rows(one)[1] == 0
    assert torch.equal(row_ops.layer_norm(one, lib=on.lib), want[2, 3].expand(7, 24))
    images = base.view(5, 2, 3, 24).permute(0, 3, 1, 2)                                      # (N, C, H, W), channels last
    assert torch.equal(row_ops.layer_norm(images.permute(0, 2, 3, 1), lib=on.lib), want.view(5, 2, 3, 24))
    flat = torch.zeros(1 + base.numel(), dtype=F32, device=on.device)
    flat[1:] = base.reshape(-1)
    assert torch.equal(row_ops.layer_norm(flat[1:].view(5, 6, 24), lib=on.lib), want)
    x = base.detach().requires_grad_()
    dx, = torch.autograd.grad(row_ops.layer_norm(x, lib=on.lib).sum(), x)                     # an expanded gradient
    check_stored(dx, norm_grads(torch.ones(5, 6, 24).double(), base.double().cpu(), None, 1e-5)[0])


def test_layer_norm_keeps_far_means_and_bad_rows_apart(on):
    """A mean of a thousand deviations loses no more than its bound; rows with NaN or infinity stay by themselves; a constant row is
    its bias."""
    x = make((6, 72), F32, on.device, 16, 1.0, 1000.0)
    x[1, 3], x[2, 5], x[3] = float('nan'), float('inf'), 7.0
    b = make((72,), F32, on.device, 17)
    y = row_ops.layer_norm(x, None, b, lib=on.lib)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    assert torch.equal(y[3], b)
    for r in (0, 4, 5):
        check_norm_forward(y[r:r + 1], x[r:r + 1].double().cpu(), None, b, 1e-5)


def test_no_rows(on):
    x = torch.zeros(0, 4, 16, device=on.device, requires_grad=True)
    w, b = torch.ones(16, device=on.device, requires_grad=True), torch.ones(16, device=on.device, requires_grad=True)
    y = row_ops.layer_norm(x, w, b, lib=on.lib)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == dx.shape == x.shape and not dw.any() and not db.any()
    rng = row_ops.dropout_rng(1, on.device)
    for per in ('element', 'channel', 'sample'):
        assert row_ops.dropout(x, 0.5, rng, per=per, residual=x, lib=on.lib).shape == x.shape
        y, h = row_ops.dropout_add_layer_norm(x, x, w, b, 0.5, rng, per=per, lib=on.lib)
        grads = torch.autograd.grad((y, h), (x, w, b), (torch.zeros_like(y), torch.zeros_like(h)))
        assert grads[0].shape == x.shape and not grads[1].any() and not grads[2].any()


# ---- dropout -----------------------------------------------------------------------------------------------------------------------
def test_generator_has_the_published_answers():
    """The known answers of Philox4x32-10 that its authors publish."""
    assert philox([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert philox([0xffffffff] * 4, [0xffffffff] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert philox([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


@pytest.mark.parametrize('per', ['element', 'channel', 'sample'])
@pytest.mark.parametrize('shape', [(1, 1), (3, 7), (2, 5, 8), (4, 3, 35), (2, 300), (7, 1, 64), (2, 2, 2, 19)], ids=str)
@pytest.mark.parametrize('dtype,stream', [(F32, F32), (BF16, BF16), (F16, F32), (F16, F16), (BF16, F32)], ids=str)
def test_dropout_and_its_gradients(on, per, shape, dtype, stream):
    seed, start, call, p = -(1 << 62) + 12345, (1 << 40) + 9, 5, 0.37
    rng = row_ops.dropout_rng(seed, on.device)
    rng[1] = start
    x, r = make(shape, dtype, on.device, 20).requires_grad_(), make(shape, stream, on.device, 21).requires_grad_()
    dy = make(shape, stream, on.device, 22)
    m = kept(shape, p, seed, start + call, per)
    y = row_ops.dropout(x, p, rng, call=call, per=per, residual=r, lib=on.lib)
    assert y.dtype is stream
    want = x.detach().double().cpu() * m + r.detach().double().cpu()
    check_stored(y, (want, 3 * U * ((x.detach().double().cpu() * m).abs() + want.abs())))
    rng[1] += 1000                                               # the backward pass has its own copy of what was used
    dx, dr = torch.autograd.grad(y, (x, r), dy)
    assert dx.dtype is dtype and torch.equal(dr, dy)
    want = dy.double().cpu() * m
    check_stored(dx, (want, 2 * U * want.abs()))
    assert torch.equal(dx == 0, (want == 0).to(dx.device))
    rng[1] -= 1000
    plain = row_ops.dropout(x.detach(), p, rng, call=call, per=per, lib=on.lib)
    assert plain.dtype is dtype
    want = x.detach().double().cpu() * m
    check_stored(plain, (want, 2 * U * want.abs()))


@pytest.mark.parametrize('p', [0.0, 1.0, 0.25, 1e-6])
def test_dropout_at_the_ends_of_p(on, p):
    """p = 1 drops all, infinities and NaN too; p = 0 and a p that rounds to 0 of 65536 change nothing, and p = 0 needs no rng."""
    x = make((6, 40), F32, on.device, 23)
    x[0, 0], x[1, 1], x[2, 2] = float('nan'), float('inf'), -float('inf')
    rng = None if p == 0.0 else row_ops.dropout_rng(3, on.device)
    y = row_ops.dropout(x, p, rng, lib=on.lib)
    if p == 1.0:
        assert not y.any()
    elif p == 0.25:
        m = kept((6, 40), p, 3, 0, 'element').to(on.device)
        assert not y[m == 0].any()
        assert torch.equal(torch.isfinite(y), torch.isfinite(x) | (m == 0))
    else:
        assert torch.equal(torch.nan_to_num(y, nan=9.0), torch.nan_to_num(x, nan=9.0))


def test_masks_do_not_depend_on_layout_stride_or_type(on):
    rng = row_ops.dropout_rng(77, on.device)
    ones = torch.ones(4, 9, 21, device=on.device)
    want = row_ops.dropout(ones, 0.5, rng, lib=on.lib)
    wide = torch.ones(4, 9, 30, device=on.device)[..., 3:24]
    assert torch.equal(row_ops.dropout(wide, 0.5, rng, lib=on.lib), want)
    assert torch.equal(row_ops.dropout(ones.view(36, 21), 0.5, rng, lib=on.lib), want.view(36, 21))
    assert torch.equal(row_ops.dropout(ones.transpose(0, 1).contiguous().transpose(0, 1), 0.5, rng, lib=on.lib), want)
    for t in (BF16, F16):
        assert torch.equal(row_ops.dropout(ones.to(t), 0.5, rng, lib=on.lib).float(), want)
    assert not torch.equal(row_ops.dropout(ones, 0.5, rng, call=1, lib=on.lib), want)
    advanced = rng.clone()
    advanced[1] += 1
    assert torch.equal(row_ops.dropout(ones, 0.5, advanced, lib=on.lib), row_ops.dropout(ones, 0.5, rng, call=1, lib=on.lib))
    y, h = row_ops.dropout_add_layer_norm(ones, torch.zeros_like(ones), None, None, 0.5, rng, lib=on.lib)
    assert torch.equal(h, want)                                   # the joined operator draws the same mask
    flat = row_ops.dropout(torch.ones(5003, device=on.device), 0.5, rng, lib=on.lib)        # one long row
    assert torch.equal(flat.cpu().double(), kept((1, 5003), 0.5, 77, 0, 'element').view(-1))


def test_share_of_what_is_dropped(on):
    """4096 masks at p: the count is binomial, 6 deviations are allowed (2e-9 by chance; the seed is fixed)."""
    ones = torch.ones(64, 64, device=on.device)
    for p in (0.1, 0.5, 0.9):
        n = int((row_ops.dropout(ones, p, row_ops.dropout_rng(5, on.device), lib=on.lib) == 0).sum())
        assert abs(n - 4096 * p) <= 6 * (4096 * p * (1 - p)) ** 0.5


# ---- residual + dropout + layer norm -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('per', ['element', 'channel', 'sample'])
@pytest.mark.parametrize('shape', [(1, 1), (3, 7), (4, 5, 35), (9, 64), (2, 3, 200), (2, 1000), (3, 2049), (1, 8201), (2, 16400), (1, 32777)], ids=str)
@pytest.mark.parametrize('dtype,stream,params', [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16)], ids=str)
def test_dropout_add_layer_norm_and_its_gradients(on, per, shape, dtype, stream, params):
    skip_long(on, shape[-1] > 8201 or shape[-1] > 2000 and (per != 'element' or (dtype, stream) != (BF16, BF16)))
    seed, p, eps = 1 << 50, 0.3, 1e-3
    rng = row_ops.dropout_rng(seed, on.device)
    x, r = make(shape, dtype, on.device, 30, 1.5).requires_grad_(), make(shape, stream, on.device, 31, 1.0, 0.5).requires_grad_()
    w, b = make(shape[-1:], params, on.device, 32, 0.3, 1.0).requires_grad_(), make(shape[-1:], params, on.device, 33, 0.3).requires_grad_()
    dy, dh = make(shape, dtype, on.device, 34), make(shape, stream, on.device, 35)
    m = kept(shape, p, seed, 3, per)
    y, h = row_ops.dropout_add_layer_norm(x, r, w, b, p, rng, call=3, per=per, eps=eps, lib=on.lib)
    assert y.dtype is dtype and h.dtype is stream
    dropped = x.detach().double().cpu() * m
    h64 = dropped + r.detach().double().cpu()
    off = 3 * U * (dropped.abs() + h64.abs())
    check_stored(h, (h64, off))
    check_norm_forward(y, h64, w.detach(), b.detach(), eps, off)
    with torch.no_grad():
        again = row_ops.dropout_add_layer_norm(x, r, w, b, p, rng, call=3, per=per, eps=eps, lib=on.lib)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)
    rng[1] += 17
    stored = h.detach().double().cpu()                            # the gradients are the norm's at the h that is stored
    g64, dh64 = dy.double().cpu(), dh.double().cpu()
    total, gw, gb = norm_grads(g64, stored, w.detach(), eps, dh64)
    dx, dr, dw, db = torch.autograd.grad((y, h), (x, r, w, b), (dy, dh), retain_graph=True)
    check_stored(dr, total)
    check_stored(dx, (total[0] * m, total[1] * m + 2 * U * (total[0] * m).abs()))
    check_stored(dw, gw)
    check_stored(db, gb)
    # one of the two outputs alone
    only_y, _, _ = norm_grads(g64, stored, w.detach(), eps)
    check_stored(torch.autograd.grad(y, r, dy, retain_graph=True)[0], only_y)
    dx, dr, dw, db = torch.autograd.grad(h, (x, r, w, b), dh, retain_graph=True, allow_unused=True)
    assert torch.equal(dr, dh) and not dw.any() and not db.any()
    check_stored(dx, (dh64 * m, 2 * U * (dh64 * m).abs()))


def test_join_with_nothing_dropped_is_the_sum_and_its_norm(on):
    x, r = make((5, 48), F32, on.device, 36), make((5, 48), F32, on.device, 37)
    y, h = row_ops.dropout_add_layer_norm(x, r, lib=on.lib)
    assert torch.equal(h, x + r)
    assert torch.equal(y, row_ops.layer_norm(h, lib=on.lib))


def test_gradients_against_differences(on):
    """Central differences of a scalar through all three operators, in float32 with steps of 1/64: the second-order error of the
    difference is measured by halving the step (Richardson), the rounding of the two sums is 2 * 64 * 2^-23 * |sum| of terms."""
    shape = (3, 4, 20)
    rng = row_ops.dropout_rng(11, on.device)
    x, r = make(shape, F32, on.device, 40).requires_grad_(), make(shape, F32, on.device, 41).requires_grad_()
    w, b = make((20,), F32, on.device, 42, 0.2, 1.0).requires_grad_(), make((20,), F32, on.device, 43).requires_grad_()
    probe = make(shape, F32, on.device, 44).double()

    def value(x, r, w, b):
        skip = row_ops.dropout(x, 0.2, rng, call=0, per='channel', residual=r, lib=on.lib)
        y, h = row_ops.dropout_add_layer_norm(row_ops.layer_norm(skip, w, b, lib=on.lib), skip, w, b, 0.3, rng, call=1, lib=on.lib)
        return (y.double() * probe + 0.5 * (h.double() * probe) ** 2).sum()
    grads = torch.autograd.grad(value(x, r, w, b), (x, r, w, b))
    for i, leaf in enumerate((x, r, w, b)):
        d = make(tuple(leaf.shape), F32, on.device, 45 + i)
        slope = float((grads[i].double() * d.double()).sum())

        def difference(step):
            args = [t.detach() for t in (x, r, w, b)]
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + step * d, args[i] - step * d
            return float(value(*up) - value(*down)) / (2 * step)
        coarse, fine = difference(1 / 32), difference(1 / 64)
        size = float((probe.abs() * 3 + (probe * 3) ** 2).sum())
        assert abs(slope - fine) <= abs(coarse - fine) + 64 * size * 2 ** -23, (i, slope, coarse, fine)


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------
def test_refusals(sim):
    x, w = torch.zeros(4, 3, 16), torch.ones(16)
    rng = row_ops.dropout_rng(0, 'cpu')
    norm = lambda *a, **k: row_ops.layer_norm(*a, lib=sim, **k)
    drop = lambda *a, **k: row_ops.dropout(*a, lib=sim, **k)
    join = lambda *a, **k: row_ops.dropout_add_layer_norm(*a, lib=sim, **k)
    for call in (lambda: norm(x.double()), lambda: norm(x.long()), lambda: norm([1.0]), lambda: norm(torch.zeros(3, 0)), lambda: norm(torch.tensor(1.0)),
                 lambda: norm(x, torch.ones(15)), lambda: norm(x, w, torch.ones(1, 16)), lambda: norm(x, w.bfloat16()), lambda: norm(x.bfloat16(), w.half()),
                 lambda: norm(x.bfloat16(), w, w.bfloat16()),
                 lambda: drop(x, -0.1, rng), lambda: drop(x, 1.5, rng), lambda: drop(x, float('nan'), rng), lambda: drop(x, 0.5), lambda: drop(x, 0.5, rng.int()),
                 lambda: drop(x, 0.5, torch.zeros(3, dtype=torch.int64)), lambda: drop(x, 0.5, torch.zeros(4, dtype=torch.int64)[::2]),
                 lambda: drop(x, 0.5, rng, per='pixel'), lambda: drop(x[0, 0], 0.5, rng, per='sample'), lambda: drop(x, 0.5, rng, call=1 << 63),
                 lambda: drop(x, 0.5, rng, residual=x[:1]), lambda: drop(x, 0.5, rng, residual=x.half()), lambda: drop(x.half(), 0.5, rng, residual=x.bfloat16()),
                 lambda: join(x, x[..., :8], None, None), lambda: join(x, x, w, None, 0.5), lambda: join(x, x.double(), w, None)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError, match='GPU'):
        row_ops.layer_norm(x)                                      # host tensors without a library of their own
    product = type('Lib', (), dict(launches_on_gpu=True))()
    for call in (lambda: row_ops.layer_norm(x, lib=product), lambda: row_ops.dropout(x, 0.5, rng, lib=product),
                 lambda: row_ops.dropout_add_layer_norm(x, x, p=0.5, rng=rng, lib=product)):
        with pytest.raises(ValueError, match='GPU'):                # host addresses never reach the GPU's library
            call()
    huge = torch.zeros(1, dtype=torch.float16)
    for shape in ((1, (1 << 32) + 5), (1 << 31, 2)):                # (a width that a 32-bit argument would cut to 5)
        for call in (norm, lambda t: drop(t, 0.5, rng), lambda t: join(t, t)):
            with pytest.raises(ValueError, match='columns'):
                call(huge.expand(shape))


def test_gradients_of_gradients_are_refused(on):
    """With create_graph the gradients come out as ever; what would go through them once more is an error, not a wrong number."""
    rng = row_ops.dropout_rng(0, on.device)
    for op in (lambda t: row_ops.layer_norm(t, lib=on.lib), lambda t: row_ops.dropout(t, 0.5, rng, lib=on.lib),
               lambda t: row_ops.dropout_add_layer_norm(t, t, p=0.5, rng=rng, lib=on.lib)[0]):
        x = make((4, 16), F32, on.device, 100).requires_grad_()
        want, = torch.autograd.grad((op(x) ** 2).sum(), x)
        got, = torch.autograd.grad((op(x) ** 2).sum(), x, create_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match='gradients of gradients'):
            torch.autograd.grad(got.sum() + x.sum(), x)


def test_a_norm_of_a_constant_gradient_is_refused_too(on):
    """dx depends on x even where the incoming gradient depends on nothing."""
    x = make((4, 16), F32, on.device, 102).requires_grad_()
    got, = torch.autograd.grad(row_ops.layer_norm(x, lib=on.lib)[..., 0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='gradients of gradients'):
        torch.autograd.grad((got ** 2).sum(), x)


def test_a_changed_input_is_noticed(on):
    """Autograd's version check: an input of the backward pass that was written in between is an error."""
    x = make((4, 16), F32, on.device, 101).requires_grad_()
    z = x * 1.0
    y = row_ops.layer_norm(z, lib=on.lib)
    z += 1.0
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    y, h = row_ops.dropout_add_layer_norm(x, x, lib=on.lib)
    h += 1.0
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_entry_points_refuse(sim):
    """The C entry points answer with an error, not with a launch."""
    d, p = sim.dll, torch.zeros(64).data_ptr()
    bad = native.NativeError
    fwd = lambda x=p, ld=8, t=0, rows=2, c=8, pt=0, y=p, y_ld=8, mean=None, rstd=None: sim.check(
        d.fiery_layer_norm_fwd(x, ld, t, rows, c, p, p, pt, 1e-5, y, y_ld, mean, rstd, None))
    for kw in (dict(x=None), dict(y=None), dict(mean=p), dict(t=3), dict(rows=0), dict(rows=1 << 31), dict(c=0), dict(pt=1), dict(ld=-1), dict(y_ld=7)):
        with pytest.raises(bad):
            fwd(**kw)
    bwd = lambda ws=p, n=1 << 20, dx=p, dg=p, x_ld=8: sim.check(
        d.fiery_layer_norm_bwd(p, 8, p, x_ld, 0, 1 << 20, 8, p, 0, p, p, dx, 8, dg, dg, ws, n, None))
    for kw in (dict(ws=None), dict(n=0), dict(dx=None, dg=None), dict(x_ld=-8)):
        with pytest.raises(bad):
            bwd(**kw)
    drop = lambda x_type=0, y_type=0, rows=2, c=8, t=1, rng=p, share=1, y_ld=8: sim.check(
        d.fiery_dropout(p, 8, x_type, None, 0, rows, c, t, rng, 0, share, 0, None, p, y_ld, y_type, None))
    for kw in (dict(x_type=1, y_type=2), dict(x_type=9), dict(rows=0), dict(rows=1 << 30, c=17), dict(t=-1), dict(t=65537), dict(rng=None), dict(share=0),
               dict(y_ld=7)):
        with pytest.raises(bad):
            drop(**kw)
    join = lambda res=p, st=0, xt=0, t=0, h=p: sim.check(
        d.fiery_dropout_add_layer_norm_fwd(p, 8, xt, res, 8, st, 2, 8, p, p, 0, 1e-5, t, None, 0, 1, 0, None, p, 8, h, 8, None, None, None))
    for kw in (dict(res=None), dict(h=None), dict(st=1), dict(xt=1, st=2), dict(t=5)):
        with pytest.raises(bad):
            join(**kw)
    assert d.fiery_layer_norm_bwd_workspace_floats(0, 8) == 0 == d.fiery_layer_norm_bwd_workspace_floats(8, 0)


@pytest.mark.parametrize('where', ['end', 'begin'])
@pytest.mark.parametrize('case', ['norm', 'dropout', 'join'])
def test_row_kernels_stay_inside_their_operands(sim, case, where):
    """Operands, outputs and workspaces that end (or begin) at an inaccessible page, in a process of its own."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, os.path.join(root, 'tests', 'sim', 'guard_rows.py'), case, where], cwd=root, capture_output=True, text=True,
                         timeout=900)
    assert res.returncode == 0 and f'ok {case} {where} (' in res.stdout, res.stdout[-1500:] + res.stderr[-3000:]


# ---- together, captured, on other streams, past 32 bits ------------------------------------------------------------------------------------
def _block(x, w1, b1, w2, b2, rng, lib=None):
    """A residual block as a model uses the operators: norm, branch, channel dropout + skip, then the joined norm of a second branch."""
    branch = torch.relu(row_ops.layer_norm(x, w1, b1, lib=lib))
    skip = row_ops.dropout(branch, 0.2, rng, call=0, per='channel', residual=x, lib=lib)
    return row_ops.dropout_add_layer_norm(torch.tanh(skip), skip, w2, b2, 0.3, rng, call=1, lib=lib)


def _block_leaves(device, shape, seed=50):
    c = shape[-1]
    return [make(shape, F32, device, seed).requires_grad_()] + [make((c,), F32, device, seed + 1 + i, 0.2, 1.0 if i % 2 == 0 else 0.0).requires_grad_() for i in range(4)]


def test_operators_together_against_64_bit_autograd(on):
    """Outputs and gradients of the chain against torch's autograd of its 64-bit definition.  Errors of single operators stay below
    40 u of a row's largest value here (rows of 24: DEPTH / 2 + 6 is 33); four in a row with factors up to 3 each (norms of
    spread 1, weights up to 1.6, scales up to 1.43): 4 * 40 * 3^3 u = 2.6e-4 of the tensor's largest value."""
    shape = (3, 5, 24)
    leaves, rng = _block_leaves(on.device, shape), row_ops.dropout_rng(31, on.device)
    y, h = _block(*leaves, rng, lib=on.lib)
    gy, gh = make(shape, F32, on.device, 60), make(shape, F32, on.device, 61)
    got = [y, h, *torch.autograd.grad((y, h), leaves, (gy, gh))]
    x, w1, b1, w2, b2 = ref = [t.detach().double().cpu().requires_grad_() for t in leaves]
    m1, m2 = kept(shape, 0.2, 31, 0, 'channel'), kept(shape, 0.3, 31, 1, 'element')
    norm = lambda t, w, b: norm64(t, None, None, 1e-5)[2] * w + b
    skip = x + torch.relu(norm(x, w1, b1)) * m1
    h64 = skip + torch.tanh(skip) * m2
    y64 = norm(h64, w2, b2)
    want = [y64, h64, *torch.autograd.grad((y64, h64), ref, (gy.double().cpu(), gh.double().cpu()))]
    for g, t in zip(got, want):
        assert (g.detach().double().cpu() - t.detach()).abs().max() <= 4 * 40 * 27 * U * t.abs().max()


@pytest.mark.gpu
def test_captured_step_draws_new_masks_at_every_replay(hip):
    """Forward, backward and the advance of the numbers in one hipGraph; every replay equals the eager step of its numbers bit for
    bit, with eager work of the same operators in between."""
    shape = (4, 300, 64)
    x0 = make(shape, F32, 'cuda', 70)
    gy = make(shape, F32, 'cuda', 71)

    def step(x, params, rng):
        leaves = [x.detach().requires_grad_()] + [p.detach().requires_grad_() for p in params]
        y, h = _block(*leaves, rng)
        grads = torch.autograd.grad((y, h), leaves, (gy, gy))
        rng[1:].add_(2)
        return [y.detach(), h.detach(), *grads]
    params = [t.detach() for t in _block_leaves('cuda', shape)[1:]]
    rng, eager = row_ops.dropout_rng(8, 'cuda'), row_ops.dropout_rng(8, 'cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x0, params, rng)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x0, params, rng)
    eager[1] += 4
    assert torch.equal(rng, eager)                       # the warm-up's two steps; the capture itself ran nothing
    first = None
    for k in range(3):
        graph.replay()
        want = step(x0, params, eager)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k
        assert torch.equal(rng, eager)
        if first is None:
            first = out[0].clone()
    assert not torch.equal(first, out[0])


@pytest.mark.gpu
def test_two_streams_at_once(hip):
    """The same step on two side streams without a wait between them: nothing is shared (workspaces are allocated per call)."""
    shape = (6, 700, 200)
    want, streams, got = [], [torch.cuda.Stream() for _ in range(2)], []
    leaves = [_block_leaves('cuda', shape, 80 + 10 * i) for i in range(2)]
    rng = row_ops.dropout_rng(2, 'cuda')
    gy = make(shape, F32, 'cuda', 99)
    for i in range(2):
        y, h = _block(*leaves[i], rng)
        want.append([y, h, *torch.autograd.grad((y, h), leaves[i], (gy, gy))])
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y, h = _block(*leaves[i], rng)
            got.append([y, h, *torch.autograd.grad((y, h), leaves[i], (gy, gy))])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_offsets_past_32_bits(hip):
    """Over 2^31 elements, and rows 1.2e9 elements apart: the rows at the far end are those of a small call."""
    c, rows = 4104, (1 << 31) // 4104 + 7
    x = torch.empty(rows, c, dtype=BF16, device='cuda').normal_(generator=torch.Generator(device='cuda').manual_seed(1)).requires_grad_()
    w = make((c,), F32, 'cuda', 90, 0.2, 1.0).requires_grad_()
    y = row_ops.layer_norm(x, w)
    assert torch.equal(y[-9:], row_ops.layer_norm(x[-9:], w)) and torch.equal(y[:9], row_ops.layer_norm(x[:9], w))
    dx, = torch.autograd.grad(y, x, x.detach())
    tail = x.detach()[-9:].requires_grad_()
    assert torch.equal(dx[-9:], torch.autograd.grad(row_ops.layer_norm(tail, w), tail, tail.detach())[0])
    del y, dx
    rng = row_ops.dropout_rng(4, 'cuda')
    d = row_ops.dropout(x.detach(), 0.5, rng)
    words = [h for unit in range(c // 8) for v in philox([unit, rows - 1, 0, 0], [4, 0]) for h in (v & 0xffff, v >> 16)]
    keep = torch.tensor(words, device='cuda') >= 32768
    assert torch.equal(d[-1], torch.where(keep, x.detach()[-1] * 2, torch.zeros_like(d[-1])))
    del d, x
    far = torch.zeros(2 * 1_200_000_000 + 40, dtype=F16, device='cuda').as_strided((3, 40), (1_200_000_000, 1))
    far.copy_(make((3, 40), F16, 'cuda', 91))
    assert row_ops._rows(far)[1] == 1_200_000_000
    assert torch.equal(row_ops.layer_norm(far), row_ops.layer_norm(far.contiguous()))
    assert torch.equal(row_ops.dropout(far, 0.3, rng, residual=far), row_ops.dropout(far.contiguous(), 0.3, rng, residual=far.contiguous()))


def test_errors_of_the_library_and_of_the_build_are_told(sim, monkeypatch):
    """A refusal of an entry point comes out with its text, in the forward and in the backward pass; a missing build says what to do."""
    import ctypes
    table = (ctypes.c_void_p * len(native.ROW_ENTRIES))(*sim._row_entries)
    answer = {'rc': 0}
    signature = ctypes.CFUNCTYPE(*[native._SIGNATURES['fiery_dropout'][0], *native._SIGNATURES['fiery_dropout'][1]])
    refuse = signature(lambda *args: answer['rc'])
    table[native.ROW_ENTRIES.index('fiery_dropout')] = ctypes.cast(refuse, ctypes.c_void_p).value
    lib = type('Lib', (), dict(launches_on_gpu=False, row_entries=ctypes.addressof(table)))()
    sim.dll.fiery_dropout(None, 0, 0, None, 0, 1, 1, 0, None, 0, 1, 0, None, None, 0, 0, None)           # leaves 'dropout: null pointer'
    x = torch.ones(2, 8, requires_grad=True)
    rng = row_ops.dropout_rng(0, 'cpu')
    y = row_ops.dropout(x, 0.5, rng, lib=lib)
    answer['rc'] = -22
    with pytest.raises(RuntimeError, match='error -22: dropout: null pointer'):
        row_ops.dropout(x, 0.5, rng, lib=lib)
    with pytest.raises(RuntimeError, match='error -22'):
        y.sum().backward()
    monkeypatch.setattr(row_ops, '_nodes', None)
    monkeypatch.setitem(sys.modules, 'fiery_amd._row_autograd', None)
    monkeypatch.delattr('fiery_amd._row_autograd', raising=False)
    with pytest.raises(native.NativeError, match='build it first'):
        row_ops.layer_norm(x, lib=sim)


def test_activation_checkpointing_draws_the_same_masks(on):
    """The forward pass run again inside the backward pass: the same numbers, as long as rng stays."""
    from torch.utils.checkpoint import checkpoint
    x = make((4, 24), F32, on.device, 110).requires_grad_()
    rng = row_ops.dropout_rng(12, on.device)

    def block(t):
        y, h = row_ops.dropout_add_layer_norm(torch.tanh(t), t, p=0.4, rng=rng, lib=on.lib)
        return row_ops.dropout(y, 0.3, rng, call=1, residual=h, lib=on.lib)
    want, = torch.autograd.grad(block(x).square().sum(), x)
    got, = torch.autograd.grad(checkpoint(block, x, use_reentrant=False).square().sum(), x)
    assert torch.equal(got, want)


def test_widest_and_narrowest_parameters(on):
    """Parameters that are views: strided, and one value expanded over the columns (its gradient is the sum)."""
    x, dy = make((9, 40), F32, on.device, 111), make((9, 40), F32, on.device, 112)
    wide = make((80,), F32, on.device, 113, 0.2, 1.0).requires_grad_()
    one = make((1,), F32, on.device, 114).requires_grad_()
    y = row_ops.layer_norm(x, wide[::2], one.expand(40), lib=on.lib)
    check_norm_forward(y, x.double().cpu(), wide.detach()[::2], one.detach().expand(40), 1e-5)
    dw, db = torch.autograd.grad(y, (wide, one), dy)
    _, gw, gb = norm_grads(dy.double().cpu(), x.double().cpu(), wide.detach()[::2], 1e-5)
    check_stored(dw[::2], gw)
    assert not dw[1::2].any()
    check_stored(db, (gb[0].sum(0, keepdim=True), gb[1].sum(0, keepdim=True) + 40 * U * gb[0].abs().sum(0, keepdim=True)))
