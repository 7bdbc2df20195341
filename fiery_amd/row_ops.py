"""Row operators for training and serving: layer norm, dropout whose mask is never stored, and residual + dropout + layer norm
in one pass - the normalisation and regularisation beside the training graph's BatchNorm (`train_graph.HipBatchNormAct`).

    y    = layer_norm(x, weight, bias)
    y    = dropout(x, p, rng, per='channel', residual=skip)               # nn.Dropout2d + the skip of a Bottleneck
    y, h = dropout_add_layer_norm(x, residual, weight, bias, p, rng)      # h = residual + dropout(x), y = layer_norm(h)

All are differentiable, capturable into a hipGraph (nothing synchronises; the workspace of the backward pass is allocated per call)
and deterministic.  They work on ROWS: the last axis of `x` is normalised or masked, so a pixel-major image batch goes in as
`x.permute(0, 2, 3, 1)` of a channels-last (N, C, H, W) tensor, and a channel slice of wider rows is read in place.  `x` is float32,
bfloat16 or float16; sums and statistics are kept in float32 whatever it is.

The dropout mask is a function of (seed, call, row, column) - Philox4x32-10 (Salmon et al. 2011), 16 bits per value:
p is drawn as round(65536 p) / 65536 and what is kept is scaled by the inverse of exactly that.  `rng` is a device tensor
int64 [seed, call] (`dropout_rng`); `call=` is added to its second number.  Give every dropout of a step its own number and
advance the tensor between steps (`rng[1] += calls_per_step`, also inside a captured graph: replays then draw new masks).  The
forward pass keeps the two numbers it used, so the backward pass draws the same mask whatever happens to `rng` in between.

Only `p = 0` works without an `rng`.  Gradients of gradients are not provided."""
import torch
from torch.autograd.function import once_differentiable

from . import native

_TYPES = native.ROW_TYPES
_MASKS = ('element', 'channel', 'sample')


def dropout_rng(seed, device='cuda'):
    """The state of the dropout masks on `device`: int64 [seed, call], call 0.  `seed`: any integer, taken modulo 2^64."""
    seed = int(seed) % (1 << 64)
    return torch.tensor([seed - (1 << 64) if seed >> 63 else seed, 0], dtype=torch.int64, device=device)


# ---- rows -----------------------------------------------------------------------------------------------------------------
def _rows(t):
    """(tensor, elements between rows): `t` itself where its rows lie at one stride with their values side by side, else a copy."""
    if t.is_contiguous():
        return t, t.shape[-1]
    shape, stride = t.shape, t.stride()
    if stride[-1] == 1 or shape[-1] == 1:
        ld = None
        for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
            if n == 1:
                continue
            if ld is None:
                ld, expect = s, s * n
            elif s == expect:
                expect = s * n
            else:
                break
        else:
            return t, shape[-1] if ld is None else ld
    return t.contiguous(), shape[-1]


def _sizes(x):
    c = x.shape[-1]
    return (x.numel() // c if c else 0), c


def _lib_for(lib, x):
    if not x.is_cuda and (lib is None or lib.launches_on_gpu):   # (a host address in a GPU kernel faults)
        raise ValueError('row operators run on the GPU: x is on ' + str(x.device))
    return native.get() if lib is None else lib


def _launch(lib, x, entry, *args):
    """`entry(*args, stream)` on x's device and its current stream."""
    dev = x.get_device()
    if dev < 0:                                                  # the simulator's library, on host tensors
        rc = entry(*args, None)
    elif dev == torch._C._cuda_getDevice():
        rc = entry(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = entry(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        lib.check(rc)


def _new(t, dtype=None):
    """A dense tensor of t's shape, uninitialised."""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- arguments ------------------------------------------------------------------------------------------------------------
def _check_x(x, what):
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES:
        raise ValueError(f'{what}: x is a float32, bfloat16 or float16 tensor, got {getattr(x, "dtype", type(x).__name__)}')
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f'{what}: the last axis of x has no values: shape {tuple(x.shape)}')
    if x.shape[-1] > 1 << 30 or x.numel() // x.shape[-1] >= 1 << 31:
        raise ValueError(f'{what}: at most 2^30 columns and 2^31 - 1 rows, got shape {tuple(x.shape)}')


def _check_params(x, weight, bias, what):
    kind = None
    for name, t in (('weight', weight), ('bias', bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError(f'{what}: {name} has one value for each of the {x.shape[-1]} columns, got shape {tuple(t.shape)}')
        if t.dtype is not torch.float32 and t.dtype is not x.dtype:
            raise ValueError(f'{what}: {name} is float32 or {x.dtype} as x is, got {t.dtype}')
        if kind is not None and t.dtype is not kind:
            raise ValueError(f'{what}: weight is {kind}, bias {t.dtype}')
        if t.device != x.device:
            raise ValueError(f'{what}: {name} is on {t.device}, x on {x.device}')
        kind = t.dtype


def _check_residual(x, residual, what):
    if residual.shape != x.shape:
        raise ValueError(f'{what}: the residual has the shape of x, {tuple(x.shape)}, got {tuple(residual.shape)}')
    if residual.dtype is not torch.float32 and residual.dtype is not x.dtype:
        raise ValueError(f'{what}: the residual is float32 or {x.dtype} as x is, got {residual.dtype}')
    if residual.device != x.device:
        raise ValueError(f'{what}: the residual is on {residual.device}, x on {x.device}')


def _mask_args(x, p, rng, call, per, what):
    """-> (threshold, rows that share a mask row, one column for all)."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f'{what}: p is a probability, got {p}')
    if per not in _MASKS:
        raise ValueError(f'{what}: per is one of {_MASKS}, got {per!r}')
    if per != 'element' and x.dim() < 2:
        raise ValueError(f'{what}: per={per!r} needs a first axis of samples beside the channels: shape {tuple(x.shape)}')
    threshold = round(65536 * float(p))
    if threshold:
        if not isinstance(rng, torch.Tensor) or rng.dtype is not torch.int64 or rng.shape != (2,) or not rng.is_contiguous():
            raise ValueError(f'{what}: rng is an int64 tensor [seed, call] (dropout_rng)')
        if rng.device != x.device:
            raise ValueError(f'{what}: rng is on {rng.device}, x on {x.device}')
        if not -(1 << 63) <= call < 1 << 63:
            raise ValueError(f'{what}: call is a 64-bit integer, got {call}')
    if per == 'element':
        return threshold, 1, 0
    rows, _ = _sizes(x)
    return threshold, max(1, rows // max(1, x.shape[0])), int(per == 'sample')



def _once(grads, ctx, *args):
    """The gradients, refusing gradients of gradients; the check costs nothing where no graph of the backward pass is made."""
    return once_differentiable(grads)(ctx, *args) if torch.is_grad_enabled() else grads(ctx, *args)


# ---- layer norm -----------------------------------------------------------------------------------------------------------
def _norm_fwd(lib, x, weight, bias, eps, keep):
    rows, c = _sizes(x)
    xr, ld = _rows(x)
    y = _new(x)
    stats = mean = rstd = None
    if keep:
        stats = torch.empty(2 * rows, dtype=torch.float32, device=x.device)        # mean, then rstd
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    if rows:
        params = weight if weight is not None else bias
        _launch(lib, x, lib.dll.fiery_layer_norm_fwd, xr.data_ptr(), ld, _TYPES[x.dtype], rows, c, _ptr(weight), _ptr(bias),
                0 if params is None else _TYPES[params.dtype], eps, y.data_ptr(), c, mean, rstd)
    return y, xr, (rows, c, ld), stats


def _param_grads(lib, weight, bias, want_w, want_b, rows, c, device):
    """Buffers for the parameters' gradients where they are wanted, and the workspace of their sums: (dweight, dbias, their
    FIERY_TYPE, workspace, its floats).  bias: its type or None.  The workspace is allocated per call: calls on other streams and
    captured graphs share none."""
    dw = _new(weight) if want_w else None
    db = torch.empty(c, dtype=bias, device=device) if want_b else None
    kind = weight.dtype if weight is not None else bias
    n = lib.dll.fiery_layer_norm_bwd_workspace_floats(rows, c) if want_w or want_b else 0
    return dw, db, 0 if kind is None else _TYPES[kind], torch.empty(n, dtype=torch.float32, device=device) if n else None, n


class HipLayerNorm(torch.autograd.Function):
    """`fiery_layer_norm_fwd / _bwd`; x (..., C)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, lib):
        y, xr, sizes, stats = _norm_fwd(lib, x, weight, bias, eps, True)
        ctx.save_for_backward(xr, weight, stats)
        ctx.meta = (sizes, None if bias is None else bias.dtype, lib)
        return y

    @staticmethod
    def backward(ctx, dy):
        return _once(HipLayerNorm._grads, ctx, dy)

    @staticmethod
    def _grads(ctx, dy):
        xr, weight, stats = ctx.saved_tensors
        (rows, c, ld), bias, lib = ctx.meta
        want_x, want_w, want_b, _, _ = ctx.needs_input_grad
        dx = _new(xr) if want_x else None
        dw, db, kind, ws, n = _param_grads(lib, weight, bias, want_w, want_b, rows, c, xr.device)
        if rows:
            dr, dy_ld = _rows(dy)
            mean = stats.data_ptr()
            _launch(lib, xr, lib.dll.fiery_layer_norm_bwd, dr.data_ptr(), dy_ld, xr.data_ptr(), ld, _TYPES[xr.dtype], rows, c, _ptr(weight), kind,
                    mean, mean + 4 * rows, _ptr(dx), c, _ptr(dw), _ptr(db), _ptr(ws), n)
        else:
            _zero(dw, db)
        return dx, dw, db, None, None


def _zero(*tensors):
    for t in tensors:
        if t is not None:
            t.zero_()


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, lib=None):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (..., C); weight and bias (C,) in float32 or x's type,
    either may be None.  Returns x's shape and type, dense.  `lib`: the loaded library (the product's by default)."""
    _check_x(x, 'layer_norm')
    _check_params(x, weight, bias, 'layer_norm')
    lib = _lib_for(lib, x)
    weight, bias = _dense(weight), _dense(bias)
    if torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad or bias is not None and bias.requires_grad):
        return HipLayerNorm.apply(x, weight, bias, eps, lib)
    return _norm_fwd(lib, x, weight, bias, eps, False)[0]


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


# ---- dropout --------------------------------------------------------------------------------------------------------------
def _dropout(lib, x, residual, out_type, mask, rng, call, used):
    rows, c = _sizes(x)
    y = _new(x, out_type)
    if rows:
        xr, ld = _rows(x)
        rr, r_ld = (None, 0) if residual is None else _rows(residual)
        threshold, share, one = mask
        _launch(lib, x, lib.dll.fiery_dropout, xr.data_ptr(), ld, _TYPES[x.dtype], _ptr(rr), r_ld, rows, c, threshold,
                _ptr(rng) if threshold else None, call, share, one, _ptr(used), y.data_ptr(), c, _TYPES[out_type])
    return y


class HipDropout(torch.autograd.Function):
    """`fiery_dropout` in both directions; the gradient of the residual is the gradient that comes in."""

    @staticmethod
    def forward(ctx, x, residual, mask, rng, call, lib):
        used = torch.empty(2, dtype=torch.int64, device=x.device) if mask[0] else None
        y = _dropout(lib, x, residual, x.dtype if residual is None else residual.dtype, mask, rng, call, used)
        ctx.save_for_backward(used)
        ctx.meta = (x.dtype, mask, lib)
        return y

    @staticmethod
    def backward(ctx, dy):
        return _once(HipDropout._grads, ctx, dy)

    @staticmethod
    def _grads(ctx, dy):
        used, = ctx.saved_tensors
        dtype, mask, lib = ctx.meta
        dx = _dropout(lib, dy, None, dtype, mask, used, 0, None) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x, p, rng=None, *, call=0, per='element', residual=None, lib=None):
    """[residual +] (kept ? x / (1 - p) : 0) for x (..., C).

    per: 'element' - every value its own mask; 'channel' - one per (first-axis index, column), what nn.Dropout2d drops of a batch
    of pixel-major images; 'sample' - one per first-axis index, drop-connect / stochastic depth.  residual: x's shape, float32 or
    x's type, which is then the type of the result.  A dropped infinity or NaN leaves a zero.  rng, call: see the module's text."""
    _check_x(x, 'dropout')
    if residual is not None:
        _check_residual(x, residual, 'dropout')
    mask = _mask_args(x, p, rng, call, per, 'dropout')
    lib = _lib_for(lib, x)
    if torch.is_grad_enabled() and (x.requires_grad or residual is not None and residual.requires_grad):
        return HipDropout.apply(x, residual, mask, rng, call, lib)
    return _dropout(lib, x, residual, x.dtype if residual is None else residual.dtype, mask, rng, call, None)


# ---- residual + dropout + layer norm ----------------------------------------------------------------------------------------
def _join_fwd(lib, x, residual, weight, bias, mask, rng, call, eps, keep):
    rows, c = _sizes(x)
    y, h = _new(x), _new(x, residual.dtype)
    threshold, share, one = mask
    stats = used = mean = rstd = None
    if keep:
        stats = torch.empty(2 * rows, dtype=torch.float32, device=x.device)        # mean, then rstd
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
        if threshold:
            used = torch.empty(2, dtype=torch.int64, device=x.device)
    if rows:
        xr, ld = _rows(x)
        rr, r_ld = _rows(residual)
        params = weight if weight is not None else bias
        _launch(lib, x, lib.dll.fiery_dropout_add_layer_norm_fwd, xr.data_ptr(), ld, _TYPES[x.dtype], rr.data_ptr(), r_ld, _TYPES[residual.dtype],
                rows, c, _ptr(weight), _ptr(bias), 0 if params is None else _TYPES[params.dtype], eps, threshold, _ptr(rng) if threshold else None,
                call, share, one, _ptr(used), y.data_ptr(), c, h.data_ptr(), c, mean, rstd)
    return y, h, (rows, c), stats, used


class HipDropoutAddLayerNorm(torch.autograd.Function):
    """`fiery_dropout_add_layer_norm_fwd / _bwd`: (y, h)."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, mask, rng, call, eps, lib):
        y, h, sizes, stats, used = _join_fwd(lib, x, residual, weight, bias, mask, rng, call, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, weight, stats, used)
        ctx.meta = (sizes, x.dtype, None if bias is None else bias.dtype, mask, lib)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        return _once(HipDropoutAddLayerNorm._grads, ctx, dy, dh)

    @staticmethod
    def _grads(ctx, dy, dh):
        h, weight, stats, used = ctx.saved_tensors
        (rows, c), dtype, bias, mask, lib = ctx.meta
        threshold, share, one = mask
        want_x, want_r, want_w, want_b = ctx.needs_input_grad[:4]
        if dy is None:                                           # only h went on: there is no norm to differentiate
            dw, db, _, _, _ = _param_grads(lib, weight, bias, want_w, want_b, 0, c, h.device)
            _zero(dw, db)
            dx = _dropout(lib, dh, None, dtype, mask, used, 0, None) if want_x and dh is not None else None
            return dx, dh if want_r else None, dw, db, None, None, None, None, None
        dx, dr = _new(h, dtype) if want_x else None, _new(h) if want_r else None
        dw, db, kind, ws, n = _param_grads(lib, weight, bias, want_w, want_b, rows, c, h.device)
        if rows:
            gr, dy_ld = _rows(dy)
            hg, dh_ld = (None, 0) if dh is None else _rows(dh)
            mean = stats.data_ptr()
            _launch(lib, h, lib.dll.fiery_dropout_add_layer_norm_bwd, gr.data_ptr(), dy_ld, _ptr(hg), dh_ld, h.data_ptr(), c, _TYPES[dtype],
                    _TYPES[h.dtype], rows, c, _ptr(weight), kind, mean, mean + 4 * rows, threshold, _ptr(used), share, one, _ptr(dx), c, _ptr(dr), c,
                    _ptr(dw), _ptr(db), _ptr(ws), n)
        else:
            _zero(dw, db)
        return dx, dr, dw, db, None, None, None, None, None


def dropout_add_layer_norm(x, residual, weight=None, bias=None, p=0.0, rng=None, *, call=0, per='element', eps=1e-5, lib=None):
    """h = residual + dropout(x, p), y = layer_norm(h, weight, bias) in one pass each way -> (y, h): y in x's type, h in the residual's
    (float32 or x's type).  y comes from h before it is rounded to that type; the gradients are the norm's at the h that is returned."""
    _check_x(x, 'dropout_add_layer_norm')
    _check_residual(x, residual, 'dropout_add_layer_norm')
    _check_params(x, weight, bias, 'dropout_add_layer_norm')
    mask = _mask_args(x, p, rng, call, per, 'dropout_add_layer_norm')
    lib = _lib_for(lib, x)
    weight, bias = _dense(weight), _dense(bias)
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight is not None and weight.requires_grad or
                                    bias is not None and bias.requires_grad):
        return HipDropoutAddLayerNorm.apply(x, residual, weight, bias, mask, rng, call, eps, lib)
    return _join_fwd(lib, x, residual, weight, bias, mask, rng, call, eps, False)[:2]
