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
forward pass keeps the two numbers it used, so the backward pass draws the same mask whatever happens to `rng` in between (activation
checkpointing runs the forward pass again: advance `rng` after the backward pass there; the training graph sees to it by itself).

Only `p = 0` works without an `rng`.  Gradients of gradients, forward-mode derivatives and tracing (torch.jit.trace, make_fx) are not
provided: an error; torch.compile breaks its graph around a call.  The autograd nodes are csrc/row_autograd.cpp; here are
the arguments and their checks."""
import torch

from . import native

_TYPES = native.ROW_TYPES
_MASKS = ('element', 'channel', 'sample')
_nodes = None


def _autograd():
    global _nodes
    if _nodes is None:
        try:
            from . import _row_autograd
        except ImportError as e:
            raise native.NativeError(f'fiery_amd/_row_autograd.so does not load ({e}): build it first (`python -m fiery_amd.build`)') from e
        got = getattr(_row_autograd, 'abi_version', None)
        if got != native.ABI_VERSION:
            raise native.NativeError(f'fiery_amd/_row_autograd.so: ABI version {got}, bindings expect {native.ABI_VERSION}; rebuild')
        _nodes = _row_autograd
    return _nodes


def dropout_rng(seed, device='cuda'):
    """The state of the dropout masks on `device`: int64 [seed, call], call 0.  `seed`: any integer, taken modulo 2^64."""
    seed = int(seed) % (1 << 64)
    return torch.tensor([seed - (1 << 64) if seed >> 63 else seed, 0], dtype=torch.int64, device=device)


def _rows(t):
    """(tensor, elements between rows) as the operators read t: `t` itself where its rows lie at one stride with their values side
    by side, else a copy."""
    return _autograd().rows_of(t)


def _to(lib, x):
    """Where a call on x goes: the addresses of the library's entry points and the current stream of x's device."""
    dev = x.get_device()
    if dev < 0 and (lib is None or lib.launches_on_gpu):         # (a host address in a GPU kernel faults)
        raise ValueError('row operators run on the GPU: x is on ' + str(x.device))
    return (native.get() if lib is None else lib).row_entries, 0 if dev < 0 else torch._C._cuda_getCurrentRawStream(dev)


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
    return threshold, max(1, x.numel() // (x.shape[-1] * max(1, x.shape[0]))), int(per == 'sample')



# ---- the operators --------------------------------------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps=1e-5, *, lib=None):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (..., C); weight and bias (C,) in float32 or x's type,
    either may be None.  Returns x's shape and type, dense.  `lib`: the loaded library (the product's by default)."""
    _check_x(x, 'layer_norm')
    _check_params(x, weight, bias, 'layer_norm')
    entries, stream = _to(lib, x)
    return _autograd().layer_norm(x, weight, bias, eps, entries, stream)


def dropout(x, p, rng=None, *, call=0, per='element', residual=None, lib=None):
    """[residual +] (kept ? x / (1 - p) : 0) for x (..., C).

    per: 'element' - every value its own mask; 'channel' - one per (first-axis index, column), what nn.Dropout2d drops of a batch
    of pixel-major images; 'sample' - one per first-axis index, drop-connect / stochastic depth.  residual: x's shape, float32 or
    x's type, which is then the type of the result.  A dropped infinity or NaN leaves a zero.  rng, call: see the module's text."""
    _check_x(x, 'dropout')
    if residual is not None:
        _check_residual(x, residual, 'dropout')
    mask = _mask_args(x, p, rng, call, per, 'dropout')
    entries, stream = _to(lib, x)
    return _autograd().dropout(x, residual, rng if mask[0] else None, mask, call, entries, stream)


def dropout_add_layer_norm(x, residual, weight=None, bias=None, p=0.0, rng=None, *, call=0, per='element', eps=1e-5, keep='h', lib=None):
    """h = residual + dropout(x, p), y = layer_norm(h, weight, bias) in one pass each way -> (y, h): y in x's type, h in the residual's
    (float32 or x's type).  y comes from h before it is rounded to that type.

    keep: what the backward pass reads where h has 16 bits.  'h' - the h that is returned: the gradients are the norm's at that h, and the
    weight's carries its rounding (more of it the larger a row's mean is beside its spread; no finite gradient where h overflows fp16).
    'inputs' - x and residual, which autograd then keeps: h is made again before its rounding, the gradients are as exact as beside an h
    of 32 bits, and the pass reads one tensor more.  An h of 32 bits is not rounded: the two are the same there."""
    if keep not in ('h', 'inputs'):
        raise ValueError(f"dropout_add_layer_norm: keep is 'h' or 'inputs', got {keep!r}")
    _check_x(x, 'dropout_add_layer_norm')
    _check_residual(x, residual, 'dropout_add_layer_norm')
    _check_params(x, weight, bias, 'dropout_add_layer_norm')
    mask = _mask_args(x, p, rng, call, per, 'dropout_add_layer_norm')
    entries, stream = _to(lib, x)
    return _autograd().dropout_add_layer_norm(x, residual, weight, bias, rng if mask[0] else None, mask, call, eps, keep == 'inputs', entries, stream)
